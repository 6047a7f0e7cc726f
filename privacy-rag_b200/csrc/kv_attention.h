// Internal launch API of the attention kernels over the paged cache.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "kv_common.cuh"

namespace bfvgpu {
namespace kv {

// Largest group and rows of a block: x / group = (x group_inverse) >> 21 for x < kMaxGroup + kMaxRows
// (x group_inverse < 2^32, and x (group group_inverse - 2^21) < 1280 x 1024 < 2^21).
constexpr int kMaxGroup = 1024, kMaxRows = 256, kGroupShift = 21;

// Queries and results.  Row R of a (sequence, key head) is query head (key head * group + R % group)
// of the sequence's new token R / group: all rows of one key head read the same keys.
struct Query {
  const uint16_t* q = nullptr;
  int64_t token_stride = 0, head_stride = 0;  // elements (of an axis of one element: the dims)
  uint16_t* out = nullptr;                    // [tokens][heads * group][dim]
  int32_t tokens = 0;                         // new tokens of the batch
  int32_t group = 1;                          // query heads per key head (at most kMaxGroup)
  uint32_t group_inverse = 0;                 // ceil(2^21 / group)
  int32_t window = 0, sinks = 0;              // window 0: every earlier key
  float scale_log2 = 0;                       // scale * log2(e)
};

// Split of one launch of the row kernel.
struct RowSplit {
  int32_t cluster = 1;     // blocks that share a unit and join in shared memory
  int32_t parts = 1;       // clusters per unit, joined by a second kernel
  int64_t blocks16 = 0;    // units: (16-row block, key head)
  uint64_t scratch_floats() const;
  int32_t dim_padded = 128;
};
RowSplit plan_rows(const View& kv, const Batch& bt, const Query& q, int device);  // device: current, or -1
cudaError_t launch_rows(const View& kv, const Batch& bt, const Query& q, int dtype, const RowSplit& split,
                        float* scratch, cudaStream_t st, int* launches);


// Launch of the prompt kernel: units of 256 rows of one key head, each in so many parts of its keys.
struct PromptSplit {
  int64_t units = 0;
  int32_t parts = 1, dim_padded = 128;
  bool ranked = false;  // the units of all sequences in the order of their keys
  uint64_t scratch_floats() const;
};
// Whether the queries' strides suit the prompt kernel's loads (no broadcast, no reversed axis).
bool prompt_strides(const Query& q);
PromptSplit plan_prompt(const View& kv, const Batch& bt, const Query& q, int sms);
cudaError_t launch_prompt(const View& kv, const Batch& bt, const Query& q, int dtype, const PromptSplit& split,
                          float* scratch, cudaStream_t st, int* launches);

}  // namespace kv
}  // namespace bfvgpu
