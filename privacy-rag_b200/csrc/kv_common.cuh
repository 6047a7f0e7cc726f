// Paged key-value cache: device view of one layer's pages and the helpers its kernels share.
//
// K and V are [pages][heads][page tokens][dim] in any order of the three outer axes (strides in
// elements, dim innermost), 16-bit floating point.  A sequence's tokens lie in the pages that its
// row of the table names: token j in page table[row][j / page_tokens], at row j % page_tokens.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace bfvgpu {
namespace kv {

// Error bits in the context's word (bfvgpu_ctx_check): 1 and 2 belong to the product kernels.
constexpr uint32_t kErrTable = 4;  // a page number, row, length or start outside its range; the access was skipped
constexpr uint32_t kErrWait = 8;   // a bounded wait of the prompt kernel expired

struct View {
  uint16_t* k = nullptr;
  uint16_t* v = nullptr;
  int64_t page_stride = 0, head_stride = 0, token_stride = 0;  // elements
  int32_t pages = 0, heads = 0, dim = 0;
  int32_t page_log = 0;  // log2(tokens per page)
};

// Tables and lengths of a batch.
struct Batch {
  const int32_t* table = nullptr;    // [seqs][width]
  const int32_t* lengths = nullptr;  // [seqs], the new tokens included
  const int32_t* starts = nullptr;   // [seqs + 1] first new token of each sequence; null: one each
  int32_t seqs = 0, width = 0;
  uint32_t* err = nullptr;
};

struct Bf16 {
  static constexpr int kind = 0;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
  }
};
struct Fp16 {
  static constexpr int kind = 1;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
  }
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// 2^x, to 2^-22 of the result; 2^-inf = 0, 2^NaN = NaN, results below the normal range are 0.
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// A launch that may begin while the kernel before it on the stream ends: its kernel calls
// cudaGridDependencySynchronize before it touches memory, so that only the start of its blocks, and what they do
// before that, runs under the other's last blocks (calls back to back, 64 new tokens
// appended: 3.5 -> 3.1 us, eight prompts of 512 tokens: 24.0 -> 23.2).
template <class... P, class... A>
cudaError_t launch_next(void (*kernel)(P...), dim3 grid, int threads, size_t shared, cudaStream_t st, int cluster, A... args) {
  cudaLaunchAttribute at[2]{};
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = cluster;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = shared;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

__device__ __forceinline__ void flag_error(uint32_t* err, uint32_t bit) { atomicOr(err, bit); }

// A sequence's length, held to what its row of the table can name.
__device__ __forceinline__ int32_t checked_length(const Batch& bt, const View& kv, int32_t n) {
  const int64_t most = (int64_t)bt.width << kv.page_log;
  if (n < 0 || n > most) {
    flag_error(bt.err, kErrTable);
    n = n < 0 ? 0 : (int32_t)most;
  }
  return n;
}

// The sequence of new token t: the number of i in [1, seqs] with starts[i] <= t.  One warp; the
// loads of all steps are independent, so the search costs about one round trip.
__device__ __forceinline__ int32_t sequence_of_token(const Batch& bt, int32_t t) {
  const int lane = threadIdx.x & 31;
  int32_t n = 0;
  for (int32_t i = 1 + lane; i - lane <= bt.seqs; i += 32)
    n += __popc(__ballot_sync(0xffffffffu, i <= bt.seqs && bt.starts[i] <= t));
  return n < bt.seqs ? n : bt.seqs - 1;
}

}  // namespace kv
}  // namespace bfvgpu
