// Internal launch API of the attention over shared tokens.
#pragma once
#include "kv_attention.h"
#include "kv_shared.cuh"

namespace bfvgpu {
namespace kv {

struct SharedPlan {
  int32_t warps = 0, dim_padded = 128;
  int64_t places[2] = {}, slots = 0;  // units over shared and over own keys; partial results
  uint64_t scratch_floats() const;
};
SharedPlan plan_shared(const View& kv, const Batch& bt, const SharedQuery& q, int sms);
cudaError_t launch_shared(const View& kv, const Batch& bt, const SharedQuery& q, int dtype, const SharedPlan& plan, float* scratch,
                          cudaStream_t st, int* launches);

}  // namespace kv
}  // namespace bfvgpu
