// Attention of a few query rows per key head over the paged cache: the single-token form, and the
// form for prompts of few tokens.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c (q.k_j) - m),  c = scale log2(e),
// in one pass over the visible keys: a block keeps the running maximum m of the exponents, the
// running sum and the running o, and rescales the last two when m grows.  Partial results (m, sum, o)
// of disjoint key sets join by the same rule.
//
// Bound by HBM: per visible key and key head 4 dim bytes are read for 4 dim group operations (group
// query heads per key head), about one byte per operation at group 1.  So the layout serves the
// loads.  A warp owns its own ring of 16-key stages in shared memory, filled by 16-byte asynchronous
// copies that follow the page table row by row, and no block-wide barrier stands in the loop.  The
// rows of a key head share each key, as the 16 rows of mma.m16n8k16 (K and V fragments by ldmatrix
// from a ring swizzled by 16-byte chunks): two m16n8k16 products per key and 128 dims, a fifth of
// the time that the key's bytes take to arrive, so the wide tensor path, whose smallest tile is 64
// rows and which would need the keys of all warps in one tile, has nothing to give here.
//
// The length is split: the blocks of a thread-block cluster take equal runs of the visible keys and
// join through distributed shared memory in rank order, which needs no workspace, no atomics and no
// second launch, and adapts to the lengths on the device.  Only where units x 8 blocks cannot fill
// the GPU (few sequences and key heads, long context) does a unit take several clusters, whose
// partial results a second kernel joins, in order too: results do not depend on timing.
//
// Measured: 64 sequences of up to 4096 tokens, 8 key heads of 128: 102 us, 5.6 TB/s, of a copy's 6.5; 256 of 2048:
// 6.4 TB/s; one of 131071 tokens, 4 key heads, 8 query heads each: 49 us, 5.5 TB/s; 96 windows of 1024 keys, 2 key
// heads of 64: 14.5 us, 3.4 TB/s; one of 513 tokens: 5.9 us.  The short ones spend their time in the chain of
// launch, length, table, keys and join, whose 5 to 6 us no split makes shorter.
//
// Keys that no row sees (before the window, past the length) are never read: the loop runs over the
// visible keys, counted through: first tokens, then the window.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "kv_attention.h"
#include "kv_units.cuh"

namespace cg = cooperative_groups;

namespace bfvgpu {
namespace kv {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kKeys = 16;   // keys per stage
constexpr int kRows = 16;   // query rows per unit
constexpr int kMaxCluster = 8;

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

// NK: 16-dim steps of the products, of a ring whose rows have DP dims (256 sequences of 2048 tokens of 72 and 96 dims:
// 157 and 155 us with the eight steps of 128, 140 both with six).
// PAIR: at most 8 rows.  The upper 8 rows of the products then carry what p loses in 16 bits (p = hi
// + lo), so o keeps about 16 bits of p at no cost; with more rows a second product does the same.
template <class T, int DP, bool PAIR, int NK>
__global__ void __launch_bounds__(kThreads)
    k_kv_rows(View kv, Batch bt, Query q, int32_t cluster, int32_t parts, float* scratch) {
  using R = Ring<DP>;
  extern __shared__ __align__(1024) uint8_t ring[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t at_part = blockIdx.x / (uint32_t)cluster, u = at_part / (uint32_t)parts;
  const int32_t rank = (int32_t)(blockIdx.x - at_part * cluster), part = (int32_t)(at_part - u * parts);
  cudaGridDependencySynchronize();
  const Unit un = find_unit<kRows>(kv, bt, q, u);
  const int32_t quad = lane >> 2, pair = (lane & 3) * 2;

  // stages of the unit -> this block's run of them
  const int32_t stages = (un.n + kKeys - 1) / kKeys;
  const int32_t shares = cluster * parts, share = part * cluster + rank;
  const int32_t per = stages / shares, more = stages - per * shares;
  const int32_t s0 = share * per + min(share, more), s1 = s0 + per + (share < more);

  // query fragments (rows past the unit's and dims past the head's are 0)
  uint32_t qa[NK][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const bool in = quad + 8 * h < un.rows;
    const uint16_t* p = un.query(q, quad + 8 * h);
#pragma unroll
    for (int ks = 0; ks < NK; ++ks)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int32_t d = ks * 16 + c * 8 + pair;
        qa[ks][h + 2 * c] = in && d < kv.dim ? __ldg(reinterpret_cast<const uint32_t*>(p + d)) : 0;
      }
  }

  const uint32_t base = smem_addr(ring) + warp * R::kWarpBytes;

  // lane l looks up the page of key l % 16 of a stage, one stage ahead of its copies
  const int32_t* row_of_table = bt.table + (int64_t)un.b * bt.width;
  const int32_t page_mask = (1 << kv.page_log) - 1;
  const int64_t head_at = un.g * kv.head_stride;
  auto entry_of = [&](int32_t s) {
    const int32_t i = s * kKeys + (lane & 15);
    return s < s1 && i < un.n ? __ldg(row_of_table + (un.token(i) >> kv.page_log)) : 0;
  };
  int32_t entry = entry_of(s0 + warp);
  auto issue = [&](int32_t s, int32_t slot) {
    if (s < s1) {
      const int32_t i = s * kKeys + (lane & 15);
      const bool in = i < un.n, good = (uint32_t)entry < (uint32_t)kv.pages;
      if (in && !good) flag_error(bt.err, kErrTable);
      const int64_t off = in && good ? entry * kv.page_stride + head_at + (int64_t)(un.token(i) & page_mask) * kv.token_stride : -1;
      entry = entry_of(s + kWarps);
      constexpr int kChunks = DP / 8, kPer = 32 / kChunks;  // chunks a row, rows an access
      const int chunk = lane % kChunks;
      const uint32_t to = base + slot * 2 * R::kTile;
#pragma unroll
      for (int it = 0; it < kKeys / kPer; ++it) {
        const int r = it * kPer + lane / kChunks;
        const int64_t o = __shfl_sync(0xffffffffu, off, r);
        const uint32_t dst = to + r * R::kRowBytes + ((chunk ^ (r & 7)) << 4);
        if (chunk * 8 < kv.dim) {
          const bool take = o >= 0;
          const int64_t from = take ? o + chunk * 8 : 0;
          copy16(dst, kv.k + from, take);
          copy16(dst + R::kTile, kv.v + from, take);
        }
      }
    }
    copies_commit();
  };

  float o[NK * 2][4];
#pragma unroll
  for (int i = 0; i < NK * 2; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) o[i][c] = 0;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0, 0};
  // positions of this thread's two rows
  int32_t pos[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) pos[h] = un.position(q, quad + 8 * h);
  const bool one_token = un.token_of(q, un.rows - 1) == 0;

#pragma unroll
  for (int i = 0; i < R::kStages - 1; ++i) issue(s0 + warp + i * kWarps, i);
  if (kv.dim != NK * 16) {  // the chunks past the head's dims are never copied: zeros, while the first copies are on their way
    for (int r = lane; r < R::kStages * 2 * kKeys; r += 32)
      for (int c = kv.dim / 8; c < NK * 2; ++c)
        *reinterpret_cast<uint4*>(ring + warp * R::kWarpBytes + r * R::kRowBytes + ((c ^ (r & 7)) << 4)) = make_uint4(0, 0, 0, 0);
  }
  int slot = 0;
  for (int32_t s = s0 + warp; s < s1; s += kWarps) {
    // the slot filled next was read in the last step
    issue(s + (R::kStages - 1) * kWarps, slot == 0 ? R::kStages - 1 : slot - 1);
    copies_wait<R::kStages - 1>();
    __syncwarp();
    const uint32_t kt = base + slot * 2 * R::kTile, vt = kt + R::kTile;
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
        const int32_t key = s * kKeys + t * 8 + pair + (i & 1);
        bool seen = key < un.n;
        if (!one_token) {
          const int32_t tok = un.token(key);
          seen = seen && tok <= pos[h] && (!q.window || tok > pos[h] - q.window || tok < q.sinks);
        }
        x[t][i] = seen ? c[t][i] * q.scale_log2 : -INFINITY;
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
    __syncwarp();
    slot = slot + 1 == R::kStages ? 0 : slot + 1;
  }
  copies_wait<0>();
  __syncthreads();

  // ---- join: the block's warps, then the cluster's blocks, each in a fixed order ----
  float* res = reinterpret_cast<float*>(ring);             // [warp][row][DP], then [warp][row][m, l]
  float* ml = res + kWarps * kRows * DP;
  float* own = ml + kWarps * kRows * 2;                    // the block's [row][DP], [row][m, l]
  float* own_ml = own + kRows * DP;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (PAIR && h) break;
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    const int row = quad + 8 * h;
    float* to = res + (warp * kRows + row) * DP;
#pragma unroll
    for (int i = 0; i < NK * 2; ++i) {
      const float a = PAIR ? o[i][0] + o[i][2] : o[i][2 * h], b = PAIR ? o[i][1] + o[i][3] : o[i][2 * h + 1];
      *reinterpret_cast<float2*>(to + i * 8 + pair) = make_float2(a, b);
    }
    if (pair == 0) {
      ml[(warp * kRows + row) * 2] = m[h];
      ml[(warp * kRows + row) * 2 + 1] = l[h];
    }
  }
  __syncthreads();
  const int32_t live = un.rows * DP;
  for (int32_t e = threadIdx.x; e < live; e += kThreads) {
    const int32_t row = e / DP;
    float top = -INFINITY, sum = 0, val = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ml[(w * kRows + row) * 2]);
    const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = exp2_fast(ml[(w * kRows + row) * 2] - ref);
      sum += f * ml[(w * kRows + row) * 2 + 1];
      val += f * res[w * kRows * DP + e];
    }
    own[e] = val;
    if (e % DP == 0) {
      own_ml[row * 2] = top;
      own_ml[row * 2 + 1] = sum;
    }
  }
  cg::cluster_group cl = cg::this_cluster();
  if (cluster > 1) cl.sync();
  else __syncthreads();
  for (int32_t e = (rank * kThreads + threadIdx.x) * 2; e < live; e += cluster * kThreads * 2) {
    const int32_t row = e / DP, d = e % DP;
    if (d >= kv.dim) continue;  // padding: nobody reads it
    // all blocks' numbers asked for together: each is a round trip to another processor
    float2 mlc[kMaxCluster], vc[kMaxCluster];
#pragma unroll
    for (int32_t c = 0; c < kMaxCluster; ++c) {
      if (c >= cluster) break;
      const float* other = cluster > 1 ? cl.map_shared_rank(own, c) : own;
      mlc[c] = *reinterpret_cast<const float2*>(other + kRows * DP + row * 2);
      vc[c] = *reinterpret_cast<const float2*>(other + e);
    }
    float top = -INFINITY, sum = 0, v0 = 0, v1 = 0;
#pragma unroll
    for (int32_t c = 0; c < kMaxCluster; ++c)
      if (c < cluster) top = fmaxf(top, mlc[c].x);
    const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int32_t c = 0; c < kMaxCluster; ++c) {
      if (c >= cluster) break;
      const float f = exp2_fast(mlc[c].x - ref);
      sum += f * mlc[c].y;
      v0 += f * vc[c].x;
      v1 += f * vc[c].y;
    }
    if (parts == 1) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;  // no key seen: zeros
      *reinterpret_cast<uint32_t*>(un.result(kv, q, row) + d) = T::pack(v0 * inv, v1 * inv);
    } else {
      float* to = scratch + ((int64_t)u * parts + part) * (kRows * (DP + 2));
      *reinterpret_cast<float2*>(to + e) = make_float2(v0, v1);
      if (d == 0) *reinterpret_cast<float2*>(to + kRows * DP + row * 2) = make_float2(top, sum);
    }
  }
  // No block leaves while another reads its shared memory: every read is released by this arrival.  (A relaxed arrival,
  // which orders no read, saved 0.25 us: one of 513 tokens 5.7 us against 5.95, 64 of up to 4096 101 against 102.)
  if (cluster > 1) cl.sync();
}

// Joins the parts of a unit's rows, in order: a warp per row, four rows a block.
template <class T, int DP>
__global__ void __launch_bounds__(kThreads)
    k_kv_rows_join(View kv, Batch bt, Query q, int32_t parts, const float* scratch) {
  cudaGridDependencySynchronize();
  constexpr int kPer = DP / 32;  // dims a lane
  const uint32_t u = blockIdx.x / (kRows / kWarps);
  const int32_t row = (blockIdx.x % (kRows / kWarps)) * kWarps + (threadIdx.x >> 5), d = (threadIdx.x & 31) * kPer;
  const Unit un = find_unit<kRows>(kv, bt, q, u);
  if (row >= un.rows || d >= kv.dim) return;
  const float* from = scratch + (int64_t)u * parts * (kRows * (DP + 2));
  float top = -INFINITY, sum = 0, v[kPer] = {};
  constexpr int kTogether = 8;  // parts whose numbers are asked for together
  for (int32_t c0 = 0; c0 < parts; c0 += kTogether) {
    float2 mlc[kTogether];
    float vc[kTogether][kPer];
#pragma unroll
    for (int c = 0; c < kTogether; ++c) {
      const float* other = from + (int64_t)(c0 + c) * (kRows * (DP + 2));
      mlc[c] = make_float2(-INFINITY, 0.f);
      if (c0 + c < parts) mlc[c] = *reinterpret_cast<const float2*>(other + kRows * DP + row * 2);
#pragma unroll
      for (int e = 0; e < kPer; e += 2) {
        float2 x = make_float2(0.f, 0.f);
        if (c0 + c < parts) x = *reinterpret_cast<const float2*>(other + row * DP + d + e);
        vc[c][e] = x.x;
        vc[c][e + 1] = x.y;
      }
    }
    float now = top;
#pragma unroll
    for (int c = 0; c < kTogether; ++c) now = fmaxf(now, mlc[c].x);
    const float ref = now == -INFINITY ? 0.f : now, fo = exp2_fast(top - ref);
    sum *= fo;
#pragma unroll
    for (int e = 0; e < kPer; ++e) v[e] *= fo;
#pragma unroll
    for (int c = 0; c < kTogether; ++c) {
      const float f = exp2_fast(mlc[c].x - ref);
      sum += f * mlc[c].y;
#pragma unroll
      for (int e = 0; e < kPer; ++e) v[e] += f * vc[c][e];
    }
    top = now;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint16_t* out = un.result(kv, q, row) + d;
#pragma unroll
  for (int e = 0; e < kPer; e += 2) *reinterpret_cast<uint32_t*>(out + e) = T::pack(v[e] * inv, v[e + 1] * inv);
}

constexpr int kDevices = 64;

// The shared-memory limit is an attribute of the function on a device.
template <class T, int DP, bool PAIR, int NK>
cudaError_t allow_ring(int device) {
  static std::atomic<uint64_t> allowed{0};
  if (device < kDevices && (allowed.load() >> device & 1)) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(k_kv_rows<T, DP, PAIR, NK>, cudaFuncAttributeMaxDynamicSharedMemorySize, Ring<DP>::kBytes);
  if (e == cudaSuccess && device < kDevices) allowed.fetch_or(uint64_t(1) << device);
  return e;
}

template <int DP>
void configure(cudaLaunchConfig_t* cfg, cudaLaunchAttribute* at, int64_t blocks, int cluster, cudaStream_t st) {
  cfg->gridDim = dim3((unsigned)blocks);
  cfg->blockDim = dim3(kThreads);
  cfg->dynamicSmemBytes = Ring<DP>::kBytes;
  cfg->stream = st;
  at->id = cudaLaunchAttributeClusterDimension;
  at->val.clusterDim.x = cluster;
  at->val.clusterDim.y = at->val.clusterDim.z = 1;
  cfg->attrs = at;
  cfg->numAttrs = 1;
}

template <class T, int DP, bool PAIR, int NK>
cudaError_t launch(const View& kv, const Batch& bt, const Query& q, const RowSplit& sp, float* scratch, cudaStream_t st,
                   int* launches) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess) e = allow_ring<T, DP, PAIR, NK>(device);
  if (e != cudaSuccess) return e;
  e = launch_next(k_kv_rows<T, DP, PAIR, NK>, dim3((unsigned)(sp.blocks16 * sp.parts * sp.cluster)), kThreads, Ring<DP>::kBytes, st,
                  sp.cluster, kv, bt, q, sp.cluster, sp.parts, scratch);
  if (e != cudaSuccess) return e;
  *launches += 1;
  if (sp.parts > 1) {
    e = launch_next(k_kv_rows_join<T, DP>, dim3((unsigned)(sp.blocks16 * (kRows / kWarps))), kThreads, 0, st, 1, kv, bt, q, sp.parts,
                    scratch);
    if (e != cudaSuccess) return e;
    *launches += 1;
  }
  return cudaGetLastError();
}

// How many clusters of 2^log blocks a device holds at once (a cluster lies within one of its processor
// groups, so that large ones leave processors idle); without a device, what this GPU gives.
template <int DP>
int64_t resident_clusters(int device, int log) {
  constexpr int kPerSm = DP == 64 ? 4 : 2;
  static const int given[4] = {148 * kPerSm, 74 * kPerSm, DP == 64 ? 142 : 71, DP == 64 ? 71 : 33};
  static std::atomic<int> known[kDevices][4];
  if (device < 0 || device >= kDevices) return given[log];
  int n = known[device][log].load();
  if (!n) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at{};
    configure<DP>(&cfg, &at, 1 << log, 1 << log, nullptr);
    if (allow_ring<Bf16, DP, true, DP / 16>(device) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, k_kv_rows<Bf16, DP, true, DP / 16>, &cfg) != cudaSuccess || n < 1) {
      cudaGetLastError();
      n = given[log];
    }
    known[device][log].store(n);
  }
  return n;
}

template <class T>
cudaError_t launch_typed(const View& kv, const Batch& bt, const Query& q, const RowSplit& sp, float* scratch,
                         cudaStream_t st, int* launches) {
  const bool pair = !bt.starts && q.group <= 8;
  if (sp.dim_padded == 64)
    return pair ? launch<T, 64, true, 4>(kv, bt, q, sp, scratch, st, launches)
                : launch<T, 64, false, 4>(kv, bt, q, sp, scratch, st, launches);
  if (kv.dim <= 96)
    return pair ? launch<T, 128, true, 6>(kv, bt, q, sp, scratch, st, launches)
                : launch<T, 128, false, 6>(kv, bt, q, sp, scratch, st, launches);
  return pair ? launch<T, 128, true, 8>(kv, bt, q, sp, scratch, st, launches)
              : launch<T, 128, false, 8>(kv, bt, q, sp, scratch, st, launches);
}

}  // namespace

uint64_t RowSplit::scratch_floats() const {
  return parts > 1 ? (uint64_t)blocks16 * parts * kRows * (dim_padded + 2) : 0;
}

// Shares of the keys, by an estimate in keys that one block streams while all are busy: a block costs its
// share plus kStart (start, first loads, joins: 6 us against 23 ns a key, measured with 2048 units of
// 2048 keys in 1 to 8 shares: 167, 195, 269, 444 us), and blocks run in waves of what is resident
// (up to two waves they mix in part, after that wholly: lengths differ, and where they do not the blocks of a part-filled
// wave are the faster for it; 12 sequences of up to 16000 keys, 4 key heads: 68 us in 4 shares, one wave, 46 in 8; 119 of up
// to 8670, one key head: 74 in 2, 61 in 4).  One unit's further parts cost a second kernel, kJoin.
// 16 sequences of 1024 keys and 8 key heads: 20, 17, 22 us in 1, 2, 4 shares; 131071 keys and 4 key heads:
// 55 us in 8 x 8 shares, which are resident together, 82 us in 8 x 9, which are not.
RowSplit plan_rows(const View& kv, const Batch& bt, const Query& q, int device) {
  constexpr double kStart = 270, kJoin = 170;
  RowSplit sp;
  sp.dim_padded = kv.dim <= 64 ? 64 : 128;
  const int64_t per = (q.group + kRows - 1) / kRows;
  // at most ceil(rows / 16) blocks per sequence
  const int64_t row_blocks = bt.starts ? (int64_t)q.tokens * q.group / kRows + bt.seqs : bt.seqs * per;
  sp.blocks16 = row_blocks * kv.heads;
  // what a unit can have to read, from the width of the table
  int64_t keys = (int64_t)bt.width << kv.page_log;
  if (q.window) keys = std::min<int64_t>(keys, (int64_t)q.window + q.sinks + kRows);
  auto resident = [&](int log) {
    return sp.dim_padded == 64 ? resident_clusters<64>(device, log) : resident_clusters<128>(device, log);
  };
  double best = 0;
  for (int log = 0; 1 << log <= kMaxCluster; ++log) {
    const double fill = (double)sp.blocks16 / resident(log);
    const double time = (fill > 1 && fill < 2 ? (fill + 2) / 2 : std::max(fill, 1.0)) * ((double)keys / (1 << log) + kStart);
    if (log && time >= best) continue;
    best = time;
    sp.cluster = 1 << log;
  }
  if (sp.cluster == kMaxCluster) {
    const int64_t most = std::min<int64_t>(resident(3) / std::max<int64_t>(1, sp.blocks16), keys / (kKeys * kWarps * kMaxCluster));
    if (most > 1 && (double)keys / kMaxCluster * (1 - 1.0 / most) > kJoin) sp.parts = (int32_t)most;
  }
  return sp;
}

cudaError_t launch_rows(const View& kv, const Batch& bt, const Query& q, int dtype, const RowSplit& sp, float* scratch,
                        cudaStream_t st, int* launches) {
  return dtype == 0 ? launch_typed<Bf16>(kv, bt, q, sp, scratch, st, launches)
                    : launch_typed<Fp16>(kv, bt, q, sp, scratch, st, launches);
}

}  // namespace kv
}  // namespace bfvgpu
