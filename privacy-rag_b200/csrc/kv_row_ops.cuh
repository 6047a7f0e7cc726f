// What the kernels of few query rows share: 16 rows as the rows of mma.m16n8k16, keys in stages of 16 in a warp's ring.
#pragma once
#include "kv_attention.h"

namespace bfvgpu {
namespace kv {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kKeys = 16;   // keys per stage
constexpr int kRows = 16;   // query rows per unit

template <int DP>
struct Ring {
  static constexpr int kStages = 3;
  static constexpr int kRowBytes = DP * 2;
  static constexpr int kTile = kKeys * kRowBytes;       // K or V of one stage
  static constexpr int kWarpBytes = kStages * 2 * kTile;
  static constexpr int kBytes = kWarps * kWarpBytes;
  // after the loop the same memory holds the warps' results, then the block's
  static constexpr int kMergeFloats = kWarps * kRows * (DP + 2) + kRows * (DP + 2);
  static_assert(kMergeFloats * 4 <= kBytes, "results fit the ring");
};

__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool take) {
  const uint32_t n = take ? 16 : 0;  // 0: the 16 bytes are filled with zeros and nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(n) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
template <class T>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (T::kind == 0)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// What p loses in 16 bits, as a second pair: hi + lo holds p to about 16 bits more.
template <class T>
__device__ __forceinline__ uint32_t pack_rest(float x, float y, uint32_t hi) {
  const float2 h = T::unpack(hi);
  return T::pack(x - h.x, y - h.y);
}

// One stage of 16 keys: scores, exponents, running maximum, sum and result of the warp's 16 rows.  seen(h, i): whether the
// thread's row h (lane / 4 + 8 h) sees the stage's key i.
// PAIR: at most 8 rows.  The upper 8 rows of the products then carry what p loses in 16 bits (p = hi
// + lo), so o keeps about 16 bits of p at no cost; with more rows a second product does the same.
template <class T, int DP, bool PAIR, int NK, class Seen>
__device__ __forceinline__ void row_stage(uint32_t kt, uint32_t vt, const uint32_t (&qa)[NK][4], float scale_log2, float (&m)[2],
                                          float (&l)[2], float (&o)[NK * 2][4], Seen&& seen) {
  using R = Ring<DP>;
  const int lane = threadIdx.x & 31, pair = (lane & 3) * 2;
  float c[2][4];
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) c[t][i] = 0;
  const int mat = lane >> 3, r8 = lane & 7;
#pragma unroll
  for (int ks = 0; ks < NK; ++ks) {
    uint32_t b[4];
    ldsm4(b, kt + ((mat >> 1) * 8 + r8) * R::kRowBytes + (((ks * 2 + (mat & 1)) ^ r8) << 4));
    mma<T>(c[0], qa[ks], b[0], b[1]);
    mma<T>(c[1], qa[ks], b[2], b[3]);
  }
  // exponents; keys past the visible ones and, with several tokens, those a row does not see: -inf
  float x[2][4], top[2] = {-INFINITY, -INFINITY};
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (PAIR && i >= 2) continue;
      const int h = i >> 1;
      x[t][i] = seen(h, t * 8 + pair + (i & 1)) ? c[t][i] * scale_log2 : -INFINITY;
      top[h] = fmaxf(top[h], x[t][i]);
    }
#pragma unroll
  for (int h = 0; h < (PAIR ? 1 : 2); ++h) {
    top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
    top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
  }
  float use[2];
  bool grew = false;
#pragma unroll
  for (int h = 0; h < (PAIR ? 1 : 2); ++h) {
    grew |= top[h] > m[h];
    top[h] = fmaxf(m[h], top[h]);
    use[h] = top[h] == -INFINITY ? 0.f : top[h];  // nothing seen yet: every p is 0
  }
  if (__any_sync(0xffffffffu, grew)) {
    float f[2];
#pragma unroll
    for (int h = 0; h < (PAIR ? 1 : 2); ++h) {
      f[h] = exp2_fast(m[h] - use[h]);
      l[h] *= f[h];
      m[h] = top[h];
    }
    if (PAIR) f[1] = f[0];
#pragma unroll
    for (int i = 0; i < NK * 2; ++i) {
      o[i][0] *= f[0];
      o[i][1] *= f[0];
      o[i][2] *= f[1];
      o[i][3] *= f[1];
    }
  }
  uint32_t hi[4], lo[4];
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int h = 0; h < (PAIR ? 1 : 2); ++h) {
      const float p0 = exp2_fast(x[t][2 * h] - use[h]), p1 = exp2_fast(x[t][2 * h + 1] - use[h]);
      l[h] += p0 + p1;
      hi[2 * t + h] = T::pack(p0, p1);
      lo[2 * t + h] = pack_rest<T>(p0, p1, hi[2 * t + h]);
      if (PAIR) hi[2 * t + 1] = lo[2 * t];
    }
#pragma unroll
  for (int ks = 0; ks < NK; ++ks) {
    uint32_t b[4];
    ldsm4t(b, vt + ((mat & 1) * 8 + r8) * R::kRowBytes + (((ks * 2 + (mat >> 1)) ^ r8) << 4));
    mma<T>(o[2 * ks], hi, b[0], b[1]);
    mma<T>(o[2 * ks + 1], hi, b[2], b[3]);
    if (!PAIR) {
      mma<T>(o[2 * ks], lo, b[0], b[1]);
      mma<T>(o[2 * ks + 1], lo, b[2], b[3]);
    }
  }
}

}  // namespace
}  // namespace kv
}  // namespace bfvgpu
