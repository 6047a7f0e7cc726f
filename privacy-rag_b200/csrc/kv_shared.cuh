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

}  // namespace kv
}  // namespace bfvgpu
