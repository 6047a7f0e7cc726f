// Groups of sequences that share their first tokens: which rows and keys the attention kernels have of them.
//
// The keys of a token's query are those that its sequence shares with its group, read through the table's row of the
// group's first sequence, and the sequence's own.  The rows of all tokens of a group see the same shared keys, all of
// them: together they are the rows of one list of keys, as the rows of a sequence are for its own.  An element is such a
// list with its rows: one for each group (shared keys), one for each sequence (own keys).
#pragma once
#include "kv_units.cuh"

namespace bfvgpu {
namespace kv {

struct SharedQuery : Query {
  const int32_t* groups = nullptr;  // [count + 1] first sequence of each group
  const int32_t* shared = nullptr;  // [count] tokens that the sequences of a group share
  int32_t count = 0;
};

struct Element {
  int32_t row = 0;                // of the table
  int32_t first = 0, tokens = 0;  // the tokens whose rows see the keys
  int32_t begin = 0, end = 0;     // keys
};

__device__ __forceinline__ int32_t start_of(const Batch& bt, int32_t s) { return bt.starts ? bt.starts[s] : s; }

// The number of ends[0 .. count - 1], which rise, that are at most x, for each lane's x.  Whole warps.
__device__ __forceinline__ int32_t ends_up_to(const int32_t* ends, int32_t count, int32_t x) {
  const int lane = threadIdx.x & 31;
  int32_t n = 0;
  for (int32_t i0 = 0; i0 < count; i0 += 32) {
    const int32_t end = i0 + lane < count ? ends[i0 + lane] : 0x7fffffff;
    int32_t c = 0;
#pragma unroll
    for (int d = 16; d; d >>= 1)
      if (__shfl_sync(0xffffffffu, end, c + d - 1) <= x) c += d;
    n += c + (__shfl_sync(0xffffffffu, end, c) <= x);
  }
  return n;
}

__device__ __forceinline__ int32_t checked_shared(const View& kv, const Batch& bt, int32_t n) {
  return checked_length(bt, kv, n);
}

// The shared keys of group j (a lane each; none: from q.count on, or numbers outside their range, which are recorded).
__device__ __forceinline__ Element shared_element(const View& kv, const Batch& bt, const SharedQuery& q, int32_t j) {
  Element e;
  if (j >= q.count) return e;
  const int32_t a = q.groups[j], b = q.groups[j + 1], n = q.shared[j];
  if (a < 0 || b < a || b > bt.seqs) {
    flag_error(bt.err, kErrTable);
    return e;
  }
  if (a == b) return e;
  const int32_t s = start_of(bt, a), t = start_of(bt, b);
  if (s < 0 || t < s || t > q.tokens) {
    flag_error(bt.err, kErrTable);
    return e;
  }
  e.row = a;
  e.first = s;
  e.tokens = t - s;
  e.end = checked_shared(kv, bt, n);
  return e;
}

// The own keys of sequence s (a lane each; whole warps), and its group (-1: it is in none, which is recorded).
__device__ __forceinline__ Element own_element(const View& kv, const Batch& bt, const SharedQuery& q, int32_t s, int32_t* group) {
  Element e;
  int32_t j = ends_up_to(q.groups + 1, q.count, s);
  *group = -1;
  if (s >= bt.seqs) return e;
  const int32_t first = start_of(bt, s), next = start_of(bt, s + 1), length = bt.lengths[s];
  if (j < q.count && q.groups[j] <= s) {
    e.begin = checked_shared(kv, bt, q.shared[j]);
    *group = j;
  } else {
    flag_error(bt.err, kErrTable);
  }
  if (first < 0 || next < first || next > q.tokens) {
    flag_error(bt.err, kErrTable);
    return Element{};
  }
  e.row = s;
  e.first = first;
  e.tokens = next - first;
  e.end = checked_length(bt, kv, length);
  // every new token sees all that is shared
  if (e.tokens && e.begin > max(0, e.end - e.tokens + 1)) flag_error(bt.err, kErrTable);
  return e;
}

// All sequences are in groups, and all tokens in sequences; one warp records it where they are not.
__device__ __forceinline__ void record_uncovered(const Batch& bt, const SharedQuery& q) {
  if ((threadIdx.x & 31) != 0) return;
  if (q.groups[0] != 0 || q.groups[q.count] != bt.seqs ||
      (bt.starts && (bt.starts[0] != 0 || bt.starts[bt.seqs] != q.tokens)))
    flag_error(bt.err, kErrTable);
}

// A unit (ROWS rows of an element's tokens and one key head) has a place in a table of all units that needs no sum over
// the elements before it: the element's first unit of rows is at (first row) / ROWS + its number, which leaves room for
// each element's last, partly filled one.
template <int ROWS>
__device__ __forceinline__ int64_t place_of(const View& kv, const Query& q, const Element& e, int32_t number, int32_t block, int32_t g) {
  return ((int64_t)((uint32_t)e.first * (uint32_t)q.group / ROWS) + number + block) * kv.heads + g;
}
inline int64_t places(const View& kv, const Query& q, int32_t elements, int rows) {
  return ((int64_t)q.tokens * q.group / rows + elements) * kv.heads;
}

// Block `block` of ROWS rows of an element, and key head g.  FLAT: shared keys, which every row sees.
template <int ROWS>
__device__ __forceinline__ Unit element_unit(const Query& q, const Element& e, int32_t block, int32_t g, bool flat) {
  Unit un;
  un.b = e.row;
  un.g = g;
  const uint32_t all = (uint32_t)e.tokens * q.group, row0 = (uint32_t)block * ROWS;
  un.rows = (int32_t)min(all - row0, (uint32_t)ROWS);
  const int32_t before = (int32_t)(row0 / (uint32_t)q.group);
  un.head0 = (int32_t)(row0 - (uint32_t)before * q.group);
  un.token0 = e.first + before;
  un.flat = flat;
  un.pos0 = flat ? e.end - 1 : e.end - e.tokens + before;
  un.begin = e.begin;
  const int32_t hi = flat ? un.pos0 : un.pos0 + un.token_of(q, un.rows - 1);
  un.n = max(0, hi + 1 - e.begin);
  return un;
}

// What all workers leave: a unit's parts lie side by side in slots.  The slot of worker w and unit u (counted through the
// row of all units) is w + u, which rises from part to part in the order of the row.
struct Slots {
  int2* index[2] = {};  // at the places of the units over shared and over own keys: first slot, parts
  float* floats = nullptr;
  int32_t most = 0;     // slots
  int32_t workers = 0;
  bool has[2] = {};     // which keys
};

// A worker's part of a unit: its tiles of KEYS keys [from, to) of n.
struct Piece {
  Unit un;
  int list = 0;
  int32_t from = 0, to = 0, n = 0;
  int32_t slot = 0;
};

// The work of all units in a row, cut into one equal run for each worker.  A unit's work is its number of key tiles, for
// own keys as if it rose evenly from block to block of its element's rows: ROWS / KEYS tiles each `group` blocks, so that
// sums have a closed form.  Work counts in 1 / group of a tile.  Whole warps; the elements are 32 at a time, a lane each.
template <int ROWS, int KEYS>
struct Runs {
  static constexpr int32_t kRise = ROWS / KEYS;
  Element el;
  int32_t blocks = 0, rise = 0;               // of the lane's element: blocks of rows; rise of the units' work from block to block
  int64_t base = 0;                           // and work of the first block's units
  int64_t upto = 0;                           // work up to and with the lane's element
  int32_t units_upto = 0;
  int64_t total = 0, x = 0, end = 0;          // work; the worker's run
  int32_t runs = 0, worker = 0, list = 0, e0 = -32;

  __device__ __forceinline__ static int32_t tiles(int32_t begin, int32_t end) {
    if (end <= begin) return 0;
    return KEYS == 16 ? (end - begin + KEYS - 1) / KEYS : (end - 1) / KEYS - begin / KEYS + 1;
  }
  __device__ __forceinline__ int64_t before(int32_t b, int64_t of_base, int32_t of_rise) const {  // work of b blocks of one key head
    return b * of_base + (int64_t)b * (b - 1) / 2 * of_rise;
  }
  __device__ __forceinline__ int64_t load(const View& kv, const Batch& bt, const SharedQuery& q, int of, int32_t at) {
    const int lane = threadIdx.x & 31;
    int32_t group;
    el = of == 0 ? shared_element(kv, bt, q, at + lane) : own_element(kv, bt, q, at + lane, &group);
    const uint32_t rows = (uint32_t)el.tokens * q.group;
    blocks = el.end > el.begin ? (int32_t)((rows + ROWS - 1) / ROWS) : 0;
    // the last key of the first block's rows
    const int32_t seen = of == 0 ? el.end : el.end - el.tokens + (int32_t)((min(rows, (uint32_t)ROWS) - 1) / (uint32_t)q.group) + 1;
    base = (int64_t)max(1, tiles(el.begin, min(seen, el.end))) * q.group;
    rise = of == 0 ? 0 : kRise;
    return before(blocks, base, rise) * kv.heads;
  }
  __device__ __forceinline__ int32_t length(const Batch& bt, const SharedQuery& q, const Slots& sl, int of) const {
    return sl.has[of] ? (of == 0 ? q.count : bt.seqs) : 0;
  }
  __device__ __forceinline__ int64_t cut(int32_t w) const { return total * w / runs; }
  // least: tiles that a run has at least
  __device__ __forceinline__ void start(const View& kv, const Batch& bt, const SharedQuery& q, const Slots& sl, int32_t me, int32_t least) {
#pragma unroll 1
    for (int of = 0; of < 2; ++of)
#pragma unroll 1
      for (int32_t at = 0; at < length(bt, q, sl, of); at += 32) total += load(kv, bt, q, of, at);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
    runs = (int32_t)max((int64_t)1, min((int64_t)sl.workers, total / ((int64_t)least * q.group)));
    worker = me;
    if (me < runs) {
      x = cut(me);
      end = cut(me + 1);
    }
  }
  // The next piece of the run; false: none is left.
  __device__ __forceinline__ bool next(const View& kv, const Batch& bt, const SharedQuery& q, const Slots& sl, Piece* piece) {
    const int lane = threadIdx.x & 31;
    if (x >= end) return false;
    uint32_t hit;
#pragma unroll 1
    while (!(hit = __ballot_sync(0xffffffffu, x < upto))) {  // the next 32 elements
      const int64_t so_far = __shfl_sync(0xffffffffu, upto, 31);
      const int32_t units_so_far = __shfl_sync(0xffffffffu, units_upto, 31);
      e0 += 32;
      while (list < 2 && e0 >= length(bt, q, sl, list)) ++list, e0 = 0;
      if (list == 2) return false;
      upto = load(kv, bt, q, list, e0);
      units_upto = blocks * kv.heads;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int64_t a = __shfl_up_sync(0xffffffffu, upto, d);
        const int32_t b = __shfl_up_sync(0xffffffffu, units_upto, d);
        if (lane >= d) upto += a, units_upto += b;
      }
      upto += so_far;
      units_upto += units_so_far;
    }
    const int at = __ffs(hit) - 1;
    Element e;
    e.row = __shfl_sync(0xffffffffu, el.row, at);
    e.first = __shfl_sync(0xffffffffu, el.first, at);
    e.tokens = __shfl_sync(0xffffffffu, el.tokens, at);
    e.begin = __shfl_sync(0xffffffffu, el.begin, at);
    e.end = __shfl_sync(0xffffffffu, el.end, at);
    const int64_t of_base = __shfl_sync(0xffffffffu, base, at);
    const int32_t of_rise = __shfl_sync(0xffffffffu, rise, at), of_blocks = __shfl_sync(0xffffffffu, blocks, at);
    const int64_t first = __shfl_sync(0xffffffffu, upto, at) - before(of_blocks, of_base, of_rise) * kv.heads;
    const int32_t first_unit = __shfl_sync(0xffffffffu, units_upto, at) - of_blocks * kv.heads;
    // the block: the last that begins at or before x
    int32_t low = 0, high = of_blocks;
    while (high - low > 1) {
      const int32_t mid = low + (high - low) / 2;
      if (first + before(mid, of_base, of_rise) * kv.heads <= x) low = mid;
      else high = mid;
    }
    const int64_t work = of_base + (int64_t)low * of_rise, into = x - first - before(low, of_base, of_rise) * kv.heads;
    const int32_t g = (int32_t)(into / work);
    const int64_t unit_x = x - (into - g * work), to = min(end, unit_x + work);
    piece->list = list;
    piece->un = element_unit<ROWS>(q, e, low, g, list == 0);
    piece->n = tiles(e.begin, e.begin + piece->un.n);
    piece->from = (int32_t)((x - unit_x) * piece->n / work);
    piece->to = (int32_t)((to - unit_x) * piece->n / work);
    piece->slot = worker + first_unit + low * kv.heads + g;
    if (piece->slot >= sl.most) {  // sequences that overlap have more units than there are
      if (lane == 0) flag_error(bt.err, kErrTable);
      x = end;
      return false;
    }
    if (x == unit_x && lane == 0) {
      const int32_t last = (int32_t)(((unit_x + work) * runs - 1) / total);  // the worker of the unit's last work
      sl.index[list][place_of<ROWS>(kv, q, e, e0 + at, low, g)] = make_int2(piece->slot, last - worker + 1);
    }
    x = to;
    return true;
  }
};

}  // namespace kv
}  // namespace bfvgpu
