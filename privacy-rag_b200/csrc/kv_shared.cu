// Attention over tokens that groups of sequences share: the shared keys are read once for all rows of a group.
//
//   o = (f_s o_s + f_o o_o) / (f_s l_s + f_o l_o),  f_x = 2^(m_x - max(m_s, m_o)),
// from the maxima m, sums l and weighted values o that the rows have over their shared and over their own keys.
//
// What a call's host side cannot know, because lengths and groups are numbers on the device, is how long either part is:
// a table may be wide, the shared part nearly all of it or nothing.  So the work is cut on the device.  The stages of 16
// keys of all units (16 rows of a group, or of a sequence, and one key head) lie in a row; each warp takes an equal run
// of them, finds its first unit by a scan over the groups and sequences, and leaves m, l and o of the units that it had a
// part of in slots of its own; a second kernel joins them in order.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "kv_row_ops.cuh"
#include "kv_shared.cuh"
#include "kv_shared.h"

namespace bfvgpu {
namespace kv {
namespace {

constexpr int kRunStages = 4;  // a warp has at least, where the row has them
#ifndef TRS
#define TRS 64
#endif
#ifndef TRO
#define TRO 64
#endif
constexpr int kTileRowsShared = TRS, kTileRowsOwn = TRO;

template <int DP>
constexpr int64_t kSlotFloats = kRows * (DP + 2);
static_assert(kRows == kSharedRows);

template <class T, int DP, int NK>
__global__ void __launch_bounds__(kThreads) k_kv_shared_rows(View kv, Batch bt, SharedQuery q, Slots sl) {
  using R = Ring<DP>;
  extern __shared__ __align__(1024) uint8_t ring[];
  const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int32_t me = blockIdx.x * kWarps + warp;
  cudaGridDependencySynchronize();
  if (me == 0) record_uncovered(bt, q);
  Runs<kRows, kKeys> runs;
  runs.start(kv, bt, q, sl, me, kRunStages);
  if (me >= runs.runs) return;

  const uint32_t base = smem_addr(ring) + warp * R::kWarpBytes;
  if (kv.dim != NK * 16) {  // the chunks past the head's dims are never copied
    for (int r = lane; r < R::kStages * 2 * kKeys; r += 32)
      for (int c = kv.dim / 8; c < NK * 2; ++c)
        *reinterpret_cast<uint4*>(ring + warp * R::kWarpBytes + r * R::kRowBytes + ((c ^ (r & 7)) << 4)) = make_uint4(0, 0, 0, 0);
  }
  const int32_t quad = lane >> 2, pair = (lane & 3) * 2, page_mask = (1 << kv.page_log) - 1;

  for (Piece p; runs.next(kv, bt, q, sl, &p);) {
    const Unit& un = p.un;
    const int32_t s0 = p.from, s1 = p.to;
    const bool flat = p.list == 0;
    uint32_t qa[NK][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool some = quad + 8 * h < un.rows;
      const uint16_t* p = un.query(q, quad + 8 * h);
#pragma unroll
      for (int ks = 0; ks < NK; ++ks)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int32_t d = ks * 16 + c * 8 + pair;
          qa[ks][h + 2 * c] = some && d < kv.dim ? __ldg(reinterpret_cast<const uint32_t*>(p + d)) : 0;
        }
    }
    // lane l looks up the page of key l % 16 of a stage, one stage ahead of its copies
    const int32_t* row_of_table = bt.table + (int64_t)un.b * bt.width;
    const int64_t head_at = un.g * kv.head_stride;
    auto entry_of = [&](int32_t s) {
      const int32_t i = s * kKeys + (lane & 15);
      return s < s1 && i < un.n ? __ldg(row_of_table + (un.token(i) >> kv.page_log)) : 0;
    };
    int32_t entry = entry_of(s0);
    auto issue = [&](int32_t s, int32_t place) {
      if (s < s1) {
        const int32_t i = s * kKeys + (lane & 15);
        const bool some = i < un.n, good = (uint32_t)entry < (uint32_t)kv.pages;
        if (some && !good) flag_error(bt.err, kErrTable);
        const int64_t off = some && good ? entry * kv.page_stride + head_at + (int64_t)(un.token(i) & page_mask) * kv.token_stride : -1;
        entry = entry_of(s + 1);
        constexpr int kChunks = DP / 8, kPer = 32 / kChunks;  // chunks a row, rows an access
        const int chunk = lane % kChunks;
        const uint32_t to = base + place * 2 * R::kTile;
#pragma unroll
        for (int it = 0; it < kKeys / kPer; ++it) {
          const int r = it * kPer + lane / kChunks;
          const int64_t o = __shfl_sync(0xffffffffu, off, r);
          const uint32_t dst = to + r * R::kRowBytes + ((chunk ^ (r & 7)) << 4);
          if (chunk * 8 < kv.dim) {
            const bool take = o >= 0;
            const int64_t at = take ? o + chunk * 8 : 0;
            copy16(dst, kv.k + at, take);
            copy16(dst + R::kTile, kv.v + at, take);
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
    int32_t pos[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) pos[h] = flat ? un.pos0 : un.pos0 + un.token_of(q, quad + 8 * h);
    const bool all = flat || un.token_of(q, un.rows - 1) == 0;
#pragma unroll
    for (int i = 0; i < R::kStages - 1; ++i) issue(s0 + i, i);
    int place = 0;
    for (int32_t s = s0; s < s1; ++s) {
      issue(s + R::kStages - 1, place == 0 ? R::kStages - 1 : place - 1);
      copies_wait<R::kStages - 1>();
      __syncwarp();
      const uint32_t kt = base + place * 2 * R::kTile;
      row_stage<T, DP, false, NK>(kt, kt + R::kTile, qa, q.scale_log2, m, l, o, [&](int h, int i) {
        const int32_t key = s * kKeys + i;
        return key < un.n && (all || un.token(key) <= pos[h]);
      });
      __syncwarp();
      place = place + 1 == R::kStages ? 0 : place + 1;
    }
    copies_wait<0>();
    __syncwarp();
    float* to = sl.floats + (int64_t)p.slot * kSlotFloats<DP>;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      const int r = quad + 8 * h;
      if (r >= un.rows) continue;
#pragma unroll
      for (int i = 0; i < NK * 2; ++i)
        *reinterpret_cast<float2*>(to + r * DP + i * 8 + pair) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
      if (pair == 0) *reinterpret_cast<float2*>(to + kRows * DP + r * 2) = make_float2(m[h], l[h]);
    }
  }
}

// Where the two lists' partial results are.
struct Sources {
  Slots slots[2];
  bool tiles[2];
};

// A warp a row (query head of a token): its parts over shared keys, then those over its own, in order.
template <class T, int DP>
__global__ void __launch_bounds__(kThreads) k_kv_shared_join(View kv, Batch bt, SharedQuery q, Sources src) {
  cudaGridDependencySynchronize();
  constexpr int kPer = DP / 32;  // dims a lane
  const int lane = threadIdx.x & 31, d = lane * kPer;
  const int32_t heads = kv.heads * q.group;
  const int64_t rows = (int64_t)q.tokens * heads, row = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int32_t t = (int32_t)(row / heads), head = (int32_t)(row - (int64_t)t * heads), g = head / q.group, in_group = head - g * q.group;
  const int32_t s = bt.starts ? sequence_of_token(bt, t) : t;
  int32_t group;
  const Element own = own_element(kv, bt, q, s, &group);
  if (t < own.first || t >= own.first + own.tokens) {  // of no sequence
    if (lane == 0) flag_error(bt.err, kErrTable);
    return;
  }
  float top = -INFINITY, sum = 0, v[kPer] = {};
#pragma unroll
  for (int list = 0; list < 2; ++list) {
    if (list == 0 && group < 0) continue;
    const Element el = list == 0 ? shared_element(kv, bt, q, group) : own;
    if (el.end <= el.begin || t < el.first || t >= el.first + el.tokens) continue;
    const Slots& sl = src.slots[list];
    const int32_t r = (t - el.first) * q.group + in_group, of = list == 0 ? group : s;
    const int32_t unit_rows = src.tiles[list] ? kSharedTileRows : kSharedRows, block = r / unit_rows, in = r - block * unit_rows;
    const int64_t place = src.tiles[list] ? place_of<kSharedTileRows>(kv, q, el, of, block, g) : place_of<kSharedRows>(kv, q, el, of, block, g);
    const int2 parts = sl.index[list][place];
    if (parts.x < 0 || parts.y < 0 || parts.y > sl.most - parts.x) {  // sequences that overlap
      if (lane == 0) flag_error(bt.err, kErrTable);
      continue;
    }
    const int64_t slot_floats = (int64_t)unit_rows * (DP + 2);
    const float* from = sl.floats + parts.x * slot_floats + in * DP;
    const int64_t to_ml = (int64_t)unit_rows * DP + in * 2 - in * DP;
    constexpr int kTogether = 8;  // parts whose numbers are asked for together
    for (int32_t c0 = 0; c0 < parts.y; c0 += kTogether) {
      float2 mlc[kTogether];
      float vc[kTogether][kPer];
#pragma unroll
      for (int c = 0; c < kTogether; ++c) {
        const float* other = from + (c0 + c) * slot_floats;
        mlc[c] = make_float2(-INFINITY, 0.f);
        if (c0 + c < parts.y) mlc[c] = *reinterpret_cast<const float2*>(other + to_ml);
#pragma unroll
        for (int i = 0; i < kPer; i += 2) {
          float2 y = make_float2(0.f, 0.f);
          if (c0 + c < parts.y) y = *reinterpret_cast<const float2*>(other + d + i);
          vc[c][i] = y.x;
          vc[c][i + 1] = y.y;
        }
      }
      float now = top;
#pragma unroll
      for (int c = 0; c < kTogether; ++c) now = fmaxf(now, mlc[c].x);
      const float ref = now == -INFINITY ? 0.f : now, fo = exp2_fast(top - ref);
      sum *= fo;
#pragma unroll
      for (int i = 0; i < kPer; ++i) v[i] *= fo;
#pragma unroll
      for (int c = 0; c < kTogether; ++c) {
        const bool some = mlc[c].x != -INFINITY || mlc[c].y != 0.f;  // else nothing was seen, and values may not be there
        const float f = some ? exp2_fast(mlc[c].x - ref) : 0.f;
        sum += f * mlc[c].y;
#pragma unroll
        for (int i = 0; i < kPer; ++i) v[i] += some ? f * vc[c][i] : 0.f;
      }
      top = now;
    }
  }
  if (d >= kv.dim) return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;  // no key seen: zeros
  uint16_t* out = q.out + row * kv.dim + d;
#pragma unroll
  for (int i = 0; i < kPer; i += 2) *reinterpret_cast<uint32_t*>(out + i) = T::pack(v[i] * inv, v[i + 1] * inv);
}

template <class T, int DP, int NK>
cudaError_t launch_rows_of(const View& kv, const Batch& bt, const SharedQuery& q, const Slots& sl, cudaStream_t st) {
  static std::atomic<uint64_t> allowed{0};
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  if (device >= 64 || !(allowed.load() >> device & 1)) {
    e = cudaFuncSetAttribute(k_kv_shared_rows<T, DP, NK>, cudaFuncAttributeMaxDynamicSharedMemorySize, Ring<DP>::kBytes);
    if (e != cudaSuccess) return e;
    if (device < 64) allowed.fetch_or(uint64_t(1) << device);
  }
  return launch_next(k_kv_shared_rows<T, DP, NK>, dim3((unsigned)(sl.workers / kWarps)), kThreads, Ring<DP>::kBytes, st, 1, kv, bt, q, sl);
}

template <class T>
cudaError_t launch_rows_typed(const View& kv, const Batch& bt, const SharedQuery& q, const Slots& sl, cudaStream_t st) {
  if (kv.dim <= 64) return launch_rows_of<T, 64, 4>(kv, bt, q, sl, st);
  if (kv.dim <= 96) return launch_rows_of<T, 128, 6>(kv, bt, q, sl, st);
  return launch_rows_of<T, 128, 8>(kv, bt, q, sl, st);
}

template <class T>
cudaError_t launch_join(const View& kv, const Batch& bt, const SharedQuery& q, const Sources& src, cudaStream_t st) {
  const int64_t rows = (int64_t)q.tokens * kv.heads * q.group;
  return launch_next(kv.dim <= 64 ? k_kv_shared_join<T, 64> : k_kv_shared_join<T, 128>, dim3((unsigned)((rows + kWarps - 1) / kWarps)),
                     kThreads, 0, st, 1, kv, bt, q, src);
}

}  // namespace

SharedPlan plan_shared(const View& kv, const Batch& bt, const SharedQuery& q, int sms, bool tiles) {
  SharedPlan p;
  const bool narrow = kv.dim <= 64;
  p.dim_padded = narrow ? 64 : 128;
  const int64_t rows = (int64_t)q.tokens * q.group;
  p.tiles[0] = tiles && rows >= (int64_t)kTileRowsShared * q.count;
  p.tiles[1] = tiles && rows >= (int64_t)kTileRowsOwn * bt.seqs;
  const int32_t elements[2] = {q.count, bt.seqs};
  p.workers[0] = sms * (narrow ? 3 : 2) * kWarps;
  p.workers[1] = sms;
  for (int list = 0; list < 2; ++list) {
    p.places[list] = places(kv, q, elements[list], p.tiles[list] ? kSharedTileRows : kSharedRows);
    p.slots[p.tiles[list]] += p.places[list];
  }
  for (int kernel = 0; kernel < 2; ++kernel)
    if (p.slots[kernel]) p.slots[kernel] += p.workers[kernel];
  return p;
}

// [first slots and parts of the units][slots of few rows][slots of tiles], each 32-byte aligned
uint64_t SharedPlan::scratch_floats() const {
  auto up = [](int64_t n) { return (n + 7) & ~int64_t(7); };
  return up(2 * (places[0] + places[1])) + up(slots[0] * kSharedRows * (dim_padded + 2)) + slots[1] * kSharedTileRows * (dim_padded + 2);
}

cudaError_t launch_shared(const View& kv, const Batch& bt, const SharedQuery& q, int dtype, const SharedPlan& p, float* scratch,
                          cudaStream_t st, int* launches) {
  auto up = [](int64_t n) { return (n + 7) & ~int64_t(7); };
  Slots kernel[2];
  float* at = scratch + up(2 * (p.places[0] + p.places[1]));
  for (int k = 0; k < 2; ++k) {
    kernel[k].index[0] = reinterpret_cast<int2*>(scratch);
    kernel[k].index[1] = kernel[k].index[0] + p.places[0];
    kernel[k].floats = at;
    kernel[k].most = (int32_t)p.slots[k];
    kernel[k].workers = p.workers[k];
    for (int list = 0; list < 2; ++list) kernel[k].has[list] = p.tiles[list] == (k == 1);
    at += up(p.slots[k] * (k ? kSharedTileRows : kSharedRows) * (p.dim_padded + 2));
  }
  Sources src;
  for (int list = 0; list < 2; ++list) {
    src.tiles[list] = p.tiles[list];
    src.slots[list] = kernel[p.tiles[list]];
  }
  cudaError_t e = cudaSuccess;
  if (p.slots[1]) {
    e = launch_shared_tiles(kv, bt, q, dtype, kernel[1], st);
    if (e != cudaSuccess) return e;
    *launches += 1;
  }
  if (p.slots[0]) {
    e = dtype == 0 ? launch_rows_typed<Bf16>(kv, bt, q, kernel[0], st) : launch_rows_typed<Fp16>(kv, bt, q, kernel[0], st);
    if (e != cudaSuccess) return e;
    *launches += 1;
  }
  e = dtype == 0 ? launch_join<Bf16>(kv, bt, q, src, st) : launch_join<Fp16>(kv, bt, q, src, st);
  if (e != cudaSuccess) return e;
  *launches += 1;
  return cudaGetLastError();
}

}  // namespace kv
}  // namespace bfvgpu
