// Attention over tokens that groups of sequences share: the shared keys are read once for all rows of a group.
//
//   o = (f_s o_s + f_o o_o) / (f_s l_s + f_o l_o),  f_x = 2^(m_x - max(m_s, m_o)),
// from the maxima m, sums l and weighted values o that the rows have over their shared and over their own keys.
//
// What a call's host side cannot know, because lengths and groups are numbers on the device, is how long either part is:
// a table may be wide, the shared part nearly all of it or nothing.  So the work is cut on the device.  The stages of 16
// keys of all units (16 rows of a group, or of a sequence, and one key head) lie in a row; each warp takes an equal run
// of them, finds its first unit by a scan over the groups and sequences, and leaves m, l and o of the units that it had a
// part of in slots of its own; a second kernel joins them in order.  A unit's parts lie side by side: the slot of warp w
// and unit u is w + u, which rises from part to part in the order of the row.
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

struct Slots {
  int2* index[2] = {};          // of the units over shared and over own keys: first slot, slots
  float* slots = nullptr;
  int32_t most = 0;             // slots
  int32_t warps = 0;
  bool has[2] = {true, true};   // which keys
};
template <int DP>
constexpr int64_t kSlotFloats = kRows * (DP + 2);

struct Row {
  int64_t total = 0;      // stages
  int32_t runs = 0;       // warps that have some
  __device__ __forceinline__ int64_t begin_of(int32_t w) const { return total * w / runs; }
  __device__ __forceinline__ int32_t warp_of(int64_t stage) const { return (int32_t)(((stage + 1) * runs - 1) / total); }
};

template <class T, int DP, int NK>
__global__ void __launch_bounds__(kThreads) k_kv_shared_rows(View kv, Batch bt, SharedQuery q, Slots sl) {
  using R = Ring<DP>;
  extern __shared__ __align__(1024) uint8_t ring[];
  const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int32_t me = blockIdx.x * kWarps + warp;
  cudaGridDependencySynchronize();
  if (me == 0) record_uncovered(bt, q);
  // 32 elements of a list (0 shared keys, 1 own keys), a lane each: what they are, their units and stages a unit
  Element el;
  int32_t units = 0, stages = 0;
  auto load = [&](int list, int32_t e0) {
    int32_t group;
    el = list == 0 ? shared_element(kv, bt, q, e0 + lane) : own_element(kv, bt, q, e0 + lane, &group);
    stages = (max(0, el.end - el.begin) + kKeys - 1) / kKeys;
    units = stages ? (int32_t)(((uint32_t)el.tokens * q.group + kRows - 1) / kRows) * kv.heads : 0;
  };
  const int32_t length[2] = {sl.has[0] ? q.count : 0, sl.has[1] ? bt.seqs : 0};
  Row row;
  for (int list = 0; list < 2; ++list)
    for (int32_t e0 = 0; e0 < length[list]; e0 += 32) {
      load(list, e0);
      row.total += (int64_t)units * stages;
    }
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) row.total += __shfl_xor_sync(0xffffffffu, row.total, d);
  row.runs = (int32_t)max((int64_t)1, min((int64_t)sl.warps, row.total / kRunStages));
  if (me >= row.runs) return;
  int64_t x = row.begin_of(me);
  const int64_t x1 = row.begin_of(me + 1);

  const uint32_t base = smem_addr(ring) + warp * R::kWarpBytes;
  if (kv.dim != NK * 16) {  // the chunks past the head's dims are never copied
    for (int r = lane; r < R::kStages * 2 * kKeys; r += 32)
      for (int c = kv.dim / 8; c < NK * 2; ++c)
        *reinterpret_cast<uint4*>(ring + warp * R::kWarpBytes + r * R::kRowBytes + ((c ^ (r & 7)) << 4)) = make_uint4(0, 0, 0, 0);
  }
  const int32_t quad = lane >> 2, pair = (lane & 3) * 2, page_mask = (1 << kv.page_log) - 1;

  int list = 0;
  int32_t e0 = -32, units_before = 0, units_upto = 0;  // of the 32 elements; up to a lane's
  int64_t before = 0, upto = 0;                        // stages
  bool loaded = false;
  while (x < x1) {
    const uint32_t hit = loaded ? __ballot_sync(0xffffffffu, x < upto) : 0;
    if (!hit) {  // the next 32 elements
      before = loaded ? __shfl_sync(0xffffffffu, upto, 31) : 0;
      units_before = loaded ? __shfl_sync(0xffffffffu, units_upto, 31) : 0;
      e0 += 32;
      while (list < 2 && e0 >= length[list]) ++list, e0 = 0;
      if (list == 2) return;
      load(list, e0);
      loaded = true;
      upto = (int64_t)units * stages;
      units_upto = units;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int64_t a = __shfl_up_sync(0xffffffffu, upto, d);
        const int32_t b = __shfl_up_sync(0xffffffffu, units_upto, d);
        if (lane >= d) upto += a, units_upto += b;
      }
      upto += before;
      units_upto += units_before;
      continue;
    }
    const int from = __ffs(hit) - 1;
    Element e;
    e.row = __shfl_sync(0xffffffffu, el.row, from);
    e.first = __shfl_sync(0xffffffffu, el.first, from);
    e.tokens = __shfl_sync(0xffffffffu, el.tokens, from);
    e.begin = __shfl_sync(0xffffffffu, el.begin, from);
    e.end = __shfl_sync(0xffffffffu, el.end, from);
    const int32_t per = __shfl_sync(0xffffffffu, stages, from);
    const int64_t first_stage = __shfl_sync(0xffffffffu, upto - (int64_t)units * stages, from);
    const int32_t first_unit = __shfl_sync(0xffffffffu, units_upto - units, from);
    const int32_t in = (int32_t)((uint64_t)(x - first_stage) / (uint32_t)per);
    const int64_t unit_stage = first_stage + (int64_t)in * per;
    const int32_t s0 = (int32_t)(x - unit_stage), s1 = (int32_t)min((int64_t)per, s0 + (x1 - x));
    const int32_t block = in / kv.heads, g = in - block * kv.heads;
    const bool flat = list == 0;
    Unit un = element_unit<kRows>(q, e, block, g, flat);
    un.n = e.end - e.begin;  // (whichever of its rows see them)
    const int32_t slot = me + first_unit + in;
    if (slot >= sl.most) {  // sequences that overlap have more units than there are
      if (lane == 0) flag_error(bt.err, kErrTable);
      return;
    }
    if (s0 == 0 && lane == 0) {
      const int32_t last = row.warp_of(unit_stage + per - 1);
      sl.index[list][place_of<kRows>(kv, q, e, e0 + from, block, g)] = make_int2(slot, last - me + 1);
    }
    x += s1 - s0;

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
    float* to = sl.slots + (int64_t)slot * kSlotFloats<DP>;
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

// A warp a row (query head of a token): its parts over shared keys, then those over its own, in order.
template <class T, int DP>
__global__ void __launch_bounds__(kThreads) k_kv_shared_join(View kv, Batch bt, SharedQuery q, Slots sl) {
  cudaGridDependencySynchronize();
  constexpr int kPer = DP / 32;  // dims a lane
  const int lane = threadIdx.x & 31, d = lane * kPer;
  const int32_t heads = kv.heads * q.group;
  const int64_t rows = (int64_t)q.tokens * heads, row = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int32_t t = (int32_t)(row / heads), head = (int32_t)(row - (int64_t)t * heads), g = head / q.group, in_group = head - g * q.group;
  const int32_t s = bt.starts ? sequence_of_token(bt, t) : t;
  Element e[2];
  int32_t number[2];
  number[1] = s;
  e[1] = own_element(kv, bt, q, s, &number[0]);
  if (t < e[1].first || t >= e[1].first + e[1].tokens) {  // of no sequence
    if (lane == 0) flag_error(bt.err, kErrTable);
    return;
  }
  if (number[0] >= 0) e[0] = shared_element(kv, bt, q, number[0]);
  float top = -INFINITY, sum = 0, v[kPer] = {};
#pragma unroll
  for (int list = 0; list < 2; ++list) {
    const Element& el = e[list];
    if (el.end <= el.begin || t < el.first || t >= el.first + el.tokens) continue;
    const int32_t r = (t - el.first) * q.group + in_group, block = r / kRows, in = r - block * kRows;
    const int2 parts = sl.index[list][place_of<kRows>(kv, q, el, number[list], block, g)];
    if (parts.x < 0 || parts.y < 0 || parts.y > sl.most - parts.x) {  // sequences that overlap
      if (lane == 0) flag_error(bt.err, kErrTable);
      continue;
    }
    const float* from = sl.slots + (int64_t)parts.x * kSlotFloats<DP>;
    constexpr int kTogether = 8;  // parts whose numbers are asked for together
    for (int32_t c0 = 0; c0 < parts.y; c0 += kTogether) {
      float2 mlc[kTogether];
      float vc[kTogether][kPer];
#pragma unroll
      for (int c = 0; c < kTogether; ++c) {
        const float* other = from + (c0 + c) * kSlotFloats<DP>;
        mlc[c] = make_float2(-INFINITY, 0.f);
        if (c0 + c < parts.y) mlc[c] = *reinterpret_cast<const float2*>(other + kRows * DP + in * 2);
#pragma unroll
        for (int i = 0; i < kPer; i += 2) {
          float2 y = make_float2(0.f, 0.f);
          if (c0 + c < parts.y) y = *reinterpret_cast<const float2*>(other + in * DP + d + i);
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
        const float f = exp2_fast(mlc[c].x - ref);
        sum += f * mlc[c].y;
#pragma unroll
        for (int i = 0; i < kPer; ++i) v[i] += f * vc[c][i];
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
cudaError_t launch(const View& kv, const Batch& bt, const SharedQuery& q, const Slots& sl, cudaStream_t st, int* launches) {
  static std::atomic<uint64_t> allowed{0};
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  if (device >= 64 || !(allowed.load() >> device & 1)) {
    e = cudaFuncSetAttribute(k_kv_shared_rows<T, DP, NK>, cudaFuncAttributeMaxDynamicSharedMemorySize, Ring<DP>::kBytes);
    if (e != cudaSuccess) return e;
    if (device < 64) allowed.fetch_or(uint64_t(1) << device);
  }
  e = launch_next(k_kv_shared_rows<T, DP, NK>, dim3((unsigned)(sl.warps / kWarps)), kThreads, Ring<DP>::kBytes, st, 1, kv, bt, q, sl);
  if (e != cudaSuccess) return e;
  *launches += 1;
  const int64_t rows = (int64_t)q.tokens * kv.heads * q.group;
  e = launch_next(k_kv_shared_join<T, DP>, dim3((unsigned)((rows + kWarps - 1) / kWarps)), kThreads, 0, st, 1, kv, bt, q, sl);
  if (e != cudaSuccess) return e;
  *launches += 1;
  return cudaGetLastError();
}

template <class T>
cudaError_t launch_typed(const View& kv, const Batch& bt, const SharedQuery& q, const Slots& sl, cudaStream_t st, int* launches) {
  if (kv.dim <= 64) return launch<T, 64, 4>(kv, bt, q, sl, st, launches);
  if (kv.dim <= 96) return launch<T, 128, 6>(kv, bt, q, sl, st, launches);
  return launch<T, 128, 8>(kv, bt, q, sl, st, launches);
}

}  // namespace

SharedPlan plan_shared(const View& kv, const Batch& bt, const SharedQuery& q, int sms) {
  SharedPlan p;
  const bool narrow = kv.dim <= 64;
  p.dim_padded = narrow ? 64 : 128;
  p.warps = sms * (narrow ? 4 : 2) * kWarps;
  p.places[0] = places(kv, q, q.count, kRows);
  p.places[1] = places(kv, q, bt.seqs, kRows);
  p.slots = p.warps + p.places[0] + p.places[1];
  return p;
}

uint64_t SharedPlan::scratch_floats() const {
  return (uint64_t)2 * (places[0] + places[1]) + 4 + (uint64_t)slots * kRows * (dim_padded + 2);
}

cudaError_t launch_shared(const View& kv, const Batch& bt, const SharedQuery& q, int dtype, const SharedPlan& p, float* scratch,
                          cudaStream_t st, int* launches) {
  Slots sl;
  sl.index[0] = reinterpret_cast<int2*>(scratch);
  sl.index[1] = sl.index[0] + p.places[0];
  // (16-byte aligned)
  sl.slots = scratch + ((2 * (p.places[0] + p.places[1]) + 3) & ~int64_t(3));
  sl.most = (int32_t)p.slots;
  sl.warps = p.warps;
  return dtype == 0 ? launch_typed<Bf16>(kv, bt, q, sl, st, launches) : launch_typed<Fp16>(kv, bt, q, sl, st, launches);
}

}  // namespace kv
}  // namespace bfvgpu
