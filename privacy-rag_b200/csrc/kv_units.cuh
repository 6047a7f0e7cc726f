// Which rows and keys a block of the attention kernels works on.
#pragma once
#include "kv_attention.h"

namespace bfvgpu {
namespace kv {

// The rows of one unit: ROWS consecutive rows of one (sequence, key head), and the keys that any of them sees.
struct Unit {
  int32_t b = 0, g = 0;
  int32_t rows = 0;              // 0: none
  int32_t token0 = 0;            // the token of the first row in q and out,
  int32_t pos0 = 0;              // its position in the sequence,
  int32_t head0 = 0;             // and the first row's query head within the group
  int32_t sinks = 0, begin = 0;  // visible keys: [0, sinks) and [begin, begin + n - sinks)
  int32_t n = 0;
  __device__ __forceinline__ int32_t token(int32_t i) const { return i < sinks ? i : i - sinks + begin; }
  // tokens from the first row's to row r's
  __device__ __forceinline__ int32_t token_of(const Query& q, int32_t r) const {
    return (int32_t)(((uint32_t)(head0 + r) * q.group_inverse) >> kGroupShift);
  }
  // position of row r's token
  __device__ __forceinline__ int32_t position(const Query& q, int32_t r) const { return pos0 + token_of(q, r); }
  // row r's query, and its place in out
  __device__ __forceinline__ const uint16_t* query(const Query& q, int32_t r) const {
    const int32_t t = token_of(q, r);
    return q.q + (int64_t)(token0 + t) * q.token_stride + (int64_t)(g * q.group + head0 + r - t * q.group) * q.head_stride;
  }
  // (results: of the first row's token; result_row: dense rows from there to row r's)
  __device__ __forceinline__ uint16_t* results(const View& kv, const Query& q) const {
    return q.out + ((int64_t)token0 * kv.heads + g) * q.group * kv.dim;
  }
  __device__ __forceinline__ int32_t result_row(const View& kv, const Query& q, int32_t r) const {
    return token_of(q, r) * (kv.heads - 1) * q.group + head0 + r;
  }
  __device__ __forceinline__ uint16_t* result(const View& kv, const Query& q, int32_t r) const {
    return results(kv, q) + (int64_t)result_row(kv, q, r) * kv.dim;
  }
};

// The `at`-th ROWS rows of sequence un.b, which has the new tokens from `first` on.
template <int ROWS>
__device__ __forceinline__ void fill_unit(Unit& un, const View& kv, const Batch& bt, const Query& q, int32_t first,
                                          int32_t tokens, int32_t length, uint32_t at) {
  const uint32_t all = (uint32_t)tokens * q.group, row0 = at * ROWS;
  if (at >= (all + ROWS - 1) / ROWS) return;  // numbers that wrapped, of starts that overlap
  un.rows = (int32_t)min(all - row0, (uint32_t)ROWS);
  const int32_t before = (int32_t)(row0 / (uint32_t)q.group);
  un.head0 = (int32_t)(row0 - (uint32_t)before * q.group);
  un.token0 = first + before;
  un.pos0 = checked_length(bt, kv, length) - tokens + before;
  // positions of the unit's first and last row
  const int32_t lo = un.pos0, hi = un.position(q, un.rows - 1);
  if (hi >= 0) {
    un.begin = q.window && lo + 1 > q.window ? lo + 1 - q.window : 0;
    un.sinks = q.sinks < un.begin ? q.sinks : un.begin;
    if (un.sinks == un.begin) un.sinks = un.begin = 0;  // nothing is left out between them
    un.n = un.sinks + hi + 1 - un.begin;
  }
}

// The sequences' new tokens have to be all of the batch's: a token that belongs to none has no row, and nothing is
// written for it.  Unit 0 records that; its two numbers are asked for before the search, in the same round trip.
struct Covered {
  int32_t first = 0, last;
  __device__ __forceinline__ Covered(const Batch& bt, const Query& q, uint32_t u) : last(q.tokens) {
    if (u == 0 && (threadIdx.x & 31) == 0) {
      first = bt.starts[0];
      last = bt.starts[bt.seqs];
    }
  }
  __device__ __forceinline__ void record(const Batch& bt, const Query& q) const {
    if (first != 0 || last != q.tokens) flag_error(bt.err, kErrTable);
  }
};

// Units are numbered [block of ROWS rows of the batch][key head]; surplus numbers find no rows.  Every
// warp of a block finds its unit by itself.  In 32 bits (the entry points keep rows and units below
// 2^31): this runs once, before anything else of its block can, and 64-bit divisions would be most of it.
template <int ROWS>
__device__ __forceinline__ Unit find_unit(const View& kv, const Batch& bt, const Query& q, uint32_t u) {
  Unit un;
  const uint32_t block = u / (uint32_t)kv.heads;
  un.g = (int32_t)(u - block * kv.heads);
  int32_t first = 0, tokens = 1, length = 0;
  uint32_t at = 0;  // the block of rows within the sequence
  if (bt.starts) {
    const Covered all(bt, q, u);
    // blocks of the sequences before this one, 32 sequences a step
    const int lane = threadIdx.x & 31;
    uint32_t before = 0;
    bool found = false;
    for (int32_t b0 = 0; b0 < bt.seqs && !found; b0 += 32) {
      uint32_t mine = 0;
      int32_t s = 0, e = 0, held = 0;
      if (b0 + lane < bt.seqs) {
        held = bt.lengths[b0 + lane];  // in one round trip with the starts
        s = bt.starts[b0 + lane];
        e = bt.starts[b0 + lane + 1];
        if (s < 0 || e < s || e > q.tokens) {
          flag_error(bt.err, kErrTable);
          s = e = 0;
        }
        mine = ((uint32_t)(e - s) * q.group + ROWS - 1) / ROWS;
      }
      uint32_t upto = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const uint32_t o = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += o;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, block - before < upto);
      if (hit) {
        const int from = __ffs(hit) - 1;
        un.b = b0 + from;
        at = block - before - __shfl_sync(0xffffffffu, upto - mine, from);
        first = __shfl_sync(0xffffffffu, s, from);
        tokens = __shfl_sync(0xffffffffu, e, from) - first;
        length = __shfl_sync(0xffffffffu, held, from);
        found = true;
      } else {
        before += __shfl_sync(0xffffffffu, upto, 31);
      }
    }
    all.record(bt, q);
    if (!found) return un;
  } else {
    const uint32_t per = (q.group + ROWS - 1) / ROWS;
    un.b = (int32_t)(block / per);
    at = block - un.b * per;
    first = un.b;
    if (un.b >= bt.seqs) return un;
    length = bt.lengths[un.b];
  }
  fill_unit<ROWS>(un, kv, bt, q, first, tokens, length, at);
  return un;
}

// The same units of up to 32 sequences in the order of their rows' positions, the last first: those with the
// most keys, whichever sequence they belong to.  A unit's level is its place in its sequence in steps of ROWS
// rows; one lane a sequence counts its units of a level or above.
template <int ROWS>
__device__ __forceinline__ Unit find_unit_ranked(const View& kv, const Batch& bt, const Query& q, uint32_t u) {
  Unit un;
  const uint32_t rank = u / (uint32_t)kv.heads;
  un.g = (int32_t)(u - rank * kv.heads);
  const int lane = threadIdx.x & 31;
  const Covered all(bt, q, u);
  int32_t s = 0, tokens = 0, length = 0;
  if (lane < bt.seqs) {
    length = bt.lengths[lane];
    s = bt.starts[lane];
    const int32_t e = bt.starts[lane + 1];
    if (s < 0 || e < s || e > q.tokens) flag_error(bt.err, kErrTable);
    else tokens = e - s;
  }
  all.record(bt, q);
  const uint32_t mine = ((uint32_t)tokens * q.group + ROWS - 1) / ROWS;
  // (a length outside its range is recorded by its units; here it only orders them)
  const uint64_t rows_before = (uint64_t)max(max(min(length, bt.width << kv.page_log), 0) - tokens, 0) * q.group;
  const uint32_t first = (uint32_t)min(rows_before / ROWS, (uint64_t)1 << 30);
  auto from = [&](uint32_t level) {  // units of this level or above
    return __reduce_add_sync(0xffffffffu, first + mine > level ? first + mine - max(first, level) : 0);
  };
  // the highest level that `rank` units have not passed
  uint32_t low = __reduce_min_sync(0xffffffffu, mine ? first : 0xffffffffu), high = __reduce_max_sync(0xffffffffu, mine ? first + mine : 0);
  if (low >= high || from(low) <= rank) return un;
  uint32_t above = 0;  // units of level `high` or above
  while (high - low > 1) {
    const uint32_t mid = low + (high - low) / 2, n = from(mid);
    if (n > rank) low = mid;
    else high = mid, above = n;
  }
  const uint32_t here = __ballot_sync(0xffffffffu, mine && first <= low && low < first + mine);
  const uint32_t lower = __popc(here & ((1u << lane) - 1));
  const int owner = __ffs(__ballot_sync(0xffffffffu, (here >> lane & 1) && lower == rank - above)) - 1;
  un.b = owner;
  const uint32_t at = low - __shfl_sync(0xffffffffu, first, owner);
  fill_unit<ROWS>(un, kv, bt, q, __shfl_sync(0xffffffffu, s, owner), __shfl_sync(0xffffffffu, tokens, owner),
                  __shfl_sync(0xffffffffu, length, owner), at);
  return un;
}

}  // namespace kv
}  // namespace bfvgpu
