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

// The same where each sequence is worked on by itself, its shared keys read through the row of its group's first.
struct EachQuery : SharedQuery {};

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
#pragma unroll 1
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

// The shared keys of group `index` (OWN false), or the own keys of sequence `index`: an index a lane, whole warps; below
// 0, or past the last: none.  What is outside its range is recorded, and has no rows.
__device__ __forceinline__ Element element_at(const View& kv, const Batch& bt, const SharedQuery& q, int32_t index, bool own) {
  Element e;
  const bool some = index >= 0 && index < (own ? bt.seqs : q.count);
  // what needs no other number is asked for first, in one round trip
  const int32_t at = some ? index : 0;
  const int32_t* one = own ? bt.starts : q.groups;
  int32_t x = own && !one ? at : one[at], y = own && !one ? at + 1 : one[at + 1], n = own ? bt.lengths[at] : q.shared[at];
  int32_t a = x, b = y, shared = n;
  bool good = true;
  if (__any_sync(0xffffffffu, some && own)) {
    const int32_t j = ends_up_to(q.groups + 1, q.count, own ? index : -1);
    if (own) {
      good = j < q.count;
      a = q.groups[good ? j : 0];
      b = q.groups[good ? j + 1 : 0];
      shared = q.shared[good ? j : 0];
    }
  }
  if (!some) return e;
  good = good && a >= 0 && b >= a && b <= bt.seqs && (!own || a <= index);
  e.row = own ? index : good ? min(a, bt.seqs - 1) : 0;
  if (!own) {
    x = start_of(bt, good ? a : 0);
    y = start_of(bt, good ? b : 0);
  }
  const int32_t most = bt.width << kv.page_log;
  good = good && x >= 0 && y >= x && y <= q.tokens && shared >= 0 && shared <= most && n >= 0 && n <= most;
  // every new token sees all that is shared
  good = good && !(own && y > x && shared > max(0, n - (y - x) + 1));
  if (!good) {
    flag_error(bt.err, kErrTable);
    return e;
  }
  e.first = x;
  e.tokens = y - x;
  e.begin = own ? shared : 0;
  e.end = n;
  return e;
}

// All sequences are in groups, and all tokens in sequences; one warp records it where they are not.
__device__ __forceinline__ void record_uncovered(const Batch& bt, const SharedQuery& q) {
  if ((threadIdx.x & 31) != 0) return;
  if (q.groups[0] != 0 || q.groups[q.count] != bt.seqs ||
      (bt.starts && (bt.starts[0] != 0 || bt.starts[bt.seqs] != q.tokens)))
    flag_error(bt.err, kErrTable);
}

struct SharedUnit : Unit {
  bool flat = false;  // every row stands at pos0, behind all of the keys
};

// Block `block` of ROWS rows of an element, and key head g.  FLAT: shared keys, which every row sees.
template <int ROWS>
__device__ __forceinline__ SharedUnit element_unit(const Query& q, const Element& e, int32_t block, int32_t g, bool flat) {
  SharedUnit un;
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

// What sequence s shares (0: nothing, or numbers outside their range, which are recorded), and the row of the table
// that it is read through.  first: the position of the sequence's first new token, or a later one.  Whole warps, s the same.
struct Prefix {
  int32_t tokens = 0, row = 0;
};
__device__ __forceinline__ Prefix prefix_of(const View& kv, const Batch& bt, const SharedQuery& q, int32_t s, int32_t first) {
  Prefix p;
  const int32_t j = ends_up_to(q.groups + 1, q.count, s), at = j < q.count ? j : 0;
  const int32_t a = q.groups[at], b = q.groups[at + 1], n = q.shared[at];
  if (j < q.count && a >= 0 && a <= s && b <= bt.seqs && n >= 0 && n <= bt.width << kv.page_log && n <= max(0, first + 1)) {
    p.tokens = n;
    p.row = a;
  } else {
    flag_error(bt.err, kErrTable);
  }
  return p;
}

// What all workers leave.  A unit's parts lie side by side in slots: the slot of worker w and unit u (counted through the
// row of all units) is w + u, which rises from part to part in the order of the row.
struct Slots {
  int2* parts[2] = {};      // [tokens][query heads] of the rows' shared and own keys: first slot times its rows + row, parts
  float* values = nullptr;  // [slots][rows of a unit][padded dims]
  float2* sums = nullptr;   // [slots][rows of a unit] maximum and sum
  int32_t most = 0;         // slots
  int32_t workers = 0;
  int32_t coarse = 0;       // log2 of the tiles that work is counted in, for sums in 32 bits
  bool has[2] = {};         // which keys
};

// A worker's part of a unit: its tiles of KEYS keys [from, to).
struct Piece {
  SharedUnit un;
  int32_t from = 0, to = 0;
  int32_t slot = 0;
};

// The work of all units in a row, cut into one equal run for each worker.  Work is counted in key tiles, and a unit's start
// as LEAD of them, so that runs of many short units are not longer than others; a run that ends in a unit's start leaves
// it to the next.  Of an element's blocks of rows the later ones see more own keys, so they are taken in pairs, the last with the first and so
// on, which have much the same work.  Whole warps; the elements are 32 at a time, a lane each.  Small code, in 32 bits: it
// runs once, and its instructions come from memory (in 64 bits, with divisions for each unit, it took 20 us).
template <int ROWS, int KEYS, int LEAD>
struct Runs {
  Element el;
  int32_t pairs = 0;                        // of the lane's element and one key head
  uint32_t work = 0, upto = 0;              // of a pair, and up to and with the lane's element
  int32_t units_upto = 0;
  uint32_t total = 0, length = 1, x = 0, end = 0;  // work; a run's, the worker's
  int32_t worker = 0, e0 = -32;

  __device__ __forceinline__ static int32_t tiles(int32_t begin, int32_t end) {
    if (end <= begin) return 0;
    return KEYS == 16 ? (end - begin + KEYS - 1) / KEYS : (end - 1) / KEYS - begin / KEYS + 1;
  }
  // tiles of block b, and the work they are counted as
  __device__ __forceinline__ static int32_t tiles_of(const SharedQuery& q, const Element& e, bool own, int32_t b) {
    const uint32_t rows = min((uint32_t)e.tokens * q.group, (uint32_t)(b + 1) * ROWS);
    const int32_t end = own ? e.end - e.tokens + (int32_t)((rows - 1) / (uint32_t)q.group) + 1 : e.end;
    return tiles(e.begin, end);
  }
  __device__ __forceinline__ static uint32_t lead(const Slots& sl) { return LEAD >> sl.coarse; }
  __device__ __forceinline__ static uint32_t counted(const Slots& sl, int32_t tiles) {
    return max(1u, ((uint32_t)tiles + (1u << sl.coarse) - 1) >> sl.coarse) + lead(sl);
  }
  __device__ __forceinline__ static int32_t blocks_of(const SharedQuery& q, const Element& e) {
    return e.end > e.begin ? (int32_t)(((uint32_t)e.tokens * q.group + ROWS - 1) / ROWS) : 0;
  }
  // units of a pair, or of a block by itself
  __device__ __forceinline__ static int32_t units_of(bool own, int32_t blocks) { return own && blocks > 1 ? 2 : 1; }
  __device__ __forceinline__ void load(const View& kv, const Batch& bt, const SharedQuery& q, const Slots& sl) {
    const int32_t e = e0 + (threadIdx.x & 31), groups = sl.has[0] ? q.count : 0;
    const bool own = e >= groups;
    el = element_at(kv, bt, q, own && !sl.has[1] ? -1 : own ? e - groups : e, own);
    const int32_t blocks = blocks_of(q, el);
    // own keys of several blocks in pairs, else one by one
    const bool paired = own && blocks > 1;
    pairs = paired ? (blocks + 1) / 2 : blocks;
    work = blocks ? counted(sl, tiles_of(q, el, own, blocks - 1)) + (paired ? counted(sl, tiles_of(q, el, own, 0)) : 0) : 0;
  }
  __device__ __forceinline__ int32_t elements(const Batch& bt, const SharedQuery& q, const Slots& sl) const {
    return (sl.has[0] ? q.count : 0) + (sl.has[1] ? bt.seqs : 0);
  }
  // The next 32 elements.
  __device__ __forceinline__ void advance(const View& kv, const Batch& bt, const SharedQuery& q, const Slots& sl) {
    const int lane = threadIdx.x & 31;
    const uint32_t so_far = __shfl_sync(0xffffffffu, upto, 31);
    const int32_t units_so_far = __shfl_sync(0xffffffffu, units_upto, 31);
    e0 += 32;
    load(kv, bt, q, sl);
    upto = (uint32_t)(pairs * kv.heads) * work;
    units_upto = pairs * kv.heads * units_of(e0 + lane >= (sl.has[0] ? q.count : 0), blocks_of(q, el));
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t a = __shfl_up_sync(0xffffffffu, upto, d);
      const int32_t b = __shfl_up_sync(0xffffffffu, units_upto, d);
      if (lane >= d) upto += a, units_upto += b;
    }
    upto += so_far;
    units_upto += units_so_far;
  }
  // Elements without keys have no units: their rows have no parts.
  __device__ __forceinline__ void record_none(const View& kv, const SharedQuery& q, const Slots& sl) const {
    const int32_t e = e0 + (threadIdx.x & 31), list = e >= (sl.has[0] ? q.count : 0);
    const int32_t heads = kv.heads * q.group;
    for (uint32_t left = __ballot_sync(0xffffffffu, el.tokens && !pairs); left; left &= left - 1) {
      const int from = __ffs(left) - 1;
      const int64_t first = (int64_t)__shfl_sync(0xffffffffu, el.first, from) * heads;
      const int64_t rows = (int64_t)__shfl_sync(0xffffffffu, el.tokens, from) * heads;
      int2* to = sl.parts[__shfl_sync(0xffffffffu, list, from)] + first;
      for (int64_t r = threadIdx.x & 31; r < rows; r += 32) to[r] = make_int2(0, 0);
    }
  }
  // least: tiles that a run has at least
  __device__ __forceinline__ void start(const View& kv, const Batch& bt, const SharedQuery& q, const Slots& sl, int32_t me, uint32_t least) {
    const int32_t count = elements(bt, q, sl);
#pragma unroll 1
    do {
      advance(kv, bt, q, sl);
      if (me == 0) record_none(kv, q, sl);
    } while (e0 + 32 < count);
    total = __shfl_sync(0xffffffffu, upto, 31);
    least = max(1u, least >> sl.coarse);
    length = max(least, (total + sl.workers - 1) / sl.workers);
    worker = me;
    x = min((uint64_t)me * length, (uint64_t)total);
    end = min((uint64_t)x + length, (uint64_t)total);
    if (count > 32) {  // from the first again
      e0 = -32;
      upto = 0;
      units_upto = 0;
    }
  }
  // The next piece of the run; false: none is left.  Pieces may be empty.
  __device__ __forceinline__ bool next(const View& kv, const Batch& bt, const SharedQuery& q, const Slots& sl, Piece* piece) {
    const int lane = threadIdx.x & 31;
    if (x >= end) return false;
    uint32_t hit;
#pragma unroll 1
    while (!(hit = __ballot_sync(0xffffffffu, x < upto))) {
      if (e0 + 32 >= elements(bt, q, sl)) return false;  // (the numbers on the device have changed meanwhile)
      advance(kv, bt, q, sl);
    }
    const int at = __ffs(hit) - 1;
    Element e;
    e.row = __shfl_sync(0xffffffffu, el.row, at);
    e.first = __shfl_sync(0xffffffffu, el.first, at);
    e.tokens = __shfl_sync(0xffffffffu, el.tokens, at);
    e.begin = __shfl_sync(0xffffffffu, el.begin, at);
    e.end = __shfl_sync(0xffffffffu, el.end, at);
    const uint32_t each = __shfl_sync(0xffffffffu, work, at);
    const int32_t units = __shfl_sync(0xffffffffu, pairs, at) * kv.heads;
    const uint32_t into = x - (__shfl_sync(0xffffffffu, upto, at) - (uint32_t)units * each);
    const int32_t number = (int32_t)(into / each), pair = number / kv.heads, g = number - pair * kv.heads;
    uint32_t off = into - (uint32_t)number * each;
    const bool own = e0 + at >= (sl.has[0] ? q.count : 0);
    // of a pair the later block first
    const int32_t blocks = blocks_of(q, e), side = units_of(own, blocks);
    const int32_t first_unit = __shfl_sync(0xffffffffu, units_upto, at) - side * units;
    int32_t block = own ? blocks - 1 - pair : pair;
    int32_t n = tiles_of(q, e, own, block), which = 0;
    uint32_t of_unit = own && blocks > 1 && block != pair ? min(counted(sl, n), each) : each;
    if (off >= of_unit) {
      off -= of_unit;
      of_unit = each - of_unit;
      block = pair;
      n = tiles_of(q, e, own, block);
      which = 1;
    }
    const uint32_t unit_x = x - off, key_x = unit_x + lead(sl), to = min(end, unit_x + of_unit);
    if (to <= key_x) {  // the run ends in the unit's start
      x = end;
      return false;
    }
    const bool first = x <= key_x;
    piece->un = element_unit<ROWS>(q, e, block, g, !own);
    // all of a unit's tiles by the end of its work
    piece->from = first ? 0 : (int32_t)min((uint64_t)(x - key_x) << sl.coarse, (uint64_t)n);
    piece->to = to == unit_x + of_unit ? n : (int32_t)min((uint64_t)(to - key_x) << sl.coarse, (uint64_t)n);
    piece->slot = worker + first_unit + side * number + which;
    if ((uint32_t)piece->slot >= (uint32_t)sl.most) {  // sequences that overlap have more units than there are
      if (lane == 0) flag_error(bt.err, kErrTable);
      x = end;
      return false;
    }
    if (first) {
      const int32_t last = (int32_t)((unit_x + of_unit - 1) / length);  // the worker of the unit's last work
      const Unit& un = piece->un;
      int2* parts = sl.parts[own];
      for (int32_t r = lane; r < un.rows; r += 32) {
        const int32_t t = un.token_of(q, r);
        parts[((int64_t)(un.token0 + t) * kv.heads + g) * q.group + un.head0 + r - t * q.group] =
            make_int2(piece->slot * ROWS + r, last - worker + 1);
      }
    }
    x = to;
    return true;
  }
};
// Bounds on the host's side: of the units' numbers, and of the work in tiles.
inline int64_t most_units(const View& kv, const Query& q, int64_t elements, int rows) {
  return ((int64_t)q.tokens * q.group / rows + 2 * elements) * kv.heads;  // (an odd block of an element has a pair's two numbers)
}

}  // namespace kv
}  // namespace bfvgpu
