// Attention of prompts over the paged cache on the 5th-generation tensor cores.
//
// Rows of one (sequence, key head) are packed token by token, the query heads of the group side by
// side, so that a block's 256 rows (two tiles of 128) share every key it loads.  Per tile of 128 keys:
//   S = Q K^T            tcgen05.mma 128 x 128 x dim, Q and K from shared memory, S in tensor memory
//   P = 2^(c S - m)      16 rows a warp, their scores in registers; P in 16 bits
//   O += P V             tcgen05.mma 128 x dim x 128, P from tensor memory, V from shared memory
// m is the row's reference exponent.  It starts as the running maximum and follows it only when the
// maximum has grown by more than 8: until then weights of up to 2^8 stay far inside both 16-bit types
// and the 32-bit sums, and O need not be rescaled.  The sum of the weights is kept in 32 bits, from
// the weights before they are rounded to 16 bits for the product.  That rounding is a choice: the product takes 16-bit
// operands, a second one for the remainder (as in the row kernel) would make half again as much work of the pipe that
// bounds 128 dims, and there is no room in tensor memory for its operand beside S, P and O.  It costs a quarter to a
// third of the error against 64 bits (eight prompts of 512 tokens: 1.6e-3 -> 2.0e-3 of the results' norm in bfloat16,
// chunks of 1024 in float16: 2.0e-4 -> 2.5e-4); the results' own rounding is the rest.
//
// Roles: warps 0-7 and 8-15 hold the rows of tile 0 and 1, four threads a row, so that a row's maximum needs no
// other warp (with a row's halves in two warps, which met for every key tile, 64 dims took 12 % longer);
// warp 16 issues S of both tiles in turn, warp 17 the products with V, warp 18 finds the rows and loads K and
// V, warp 19 loads the queries.  While one tile's rows are in their exponentials, the other tile's products
// run.  A block is resident on its SM for the whole launch and takes over the blocks that have not started
// yet (cluster launch control), so that the loads of the next rows and the results of the last ones run under
// the products in between.
// K and V arrive by TMA page by page as the table names them, in the 128-byte swizzle (K as K-major,
// V as MN-major operand).  Only visible tokens of V are loaded: what no row of the block sees may
// hold NaN (unwritten rest of a page, pages given up), and 0 x NaN would reach every row.  Such
// pages are read in rows, the others filled with zeros.
//
// What bounds it: of a pair of row tiles and 128 keys the exponentials take 2048 cycles of the special-function pipe,
// with 128 dims the products as many of the tensor pipe; measured 2500 cycles with 64 dims, 3000 with 128.  16384
// tokens, 16 query heads on 8 of 128: 835 us, 1320 TFLOP/s (950 us once the power limit lowers the clock); of 64: 630
// us; 8191 tokens with a window of 1024: 86 us back to back (94 in a long run, at the power limit); eight prompts of 512:
// 23 us, of which the start of the blocks (first S 3.3 us after it) and the results (2 us after the last product) are a
// quarter.
//
// Where there are too few rows to fill the GPU, the key tiles of a block's rows are dealt to several
// blocks, which leave (m, sum, O) in 32 bits for a second kernel to join in a fixed order.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "kv_attention.h"
#include "kv_units.cuh"

namespace bfvgpu {
namespace kv {
namespace {

constexpr int kTileRows = 128;
constexpr int kBlockRows = 2 * kTileRows;
constexpr int kTileKeys = 128;
// Two warpgroups per row tile (a thread has 64 scores: with one, the time of a row's
// exponentials and of the products that wait for them added up, and two warps per scheduler could not
// fill it), and one of the issuing warps.
constexpr int kThreads = 640;
constexpr int kScoreWarp = 16, kValueWarp = 17, kLoadWarp = 18, kQueryWarp = 19;
constexpr int kReaders = 19;          // warps that are told of the next rows: all but the loads' own
// Registers a thread: launched with 96 (640 x 96 of the SM's 65536); the issuing warpgroup keeps 64 and the
// rows take 104: 128 x 64 + 512 x 104 = 640 x 96.
constexpr int kIssueRegs = 64, kRowRegs = 104;
constexpr float kLag = 8.f;           // how far m may stay behind the running maximum
constexpr uint32_t kPolls = 1u << 20;     // of a wait for the next step before it gives up
constexpr uint32_t kLongPolls = 1u << 27; // of a wait that may span all keys of other rows
constexpr int kPartTiles = 8;         // key tiles that a part has at least
constexpr int kMaxParts = 16;

// A row tile's part of an item.
struct Span {
  int32_t lo = 0, hi = -1;  // positions of the rows (hi < 0: no row sees a key)
  // the key tiles that it needs: [from, first) and [begin, end), none from `to` on
  int32_t first = 0, begin = 0, end = 0, from = 0, to = 0;
  __device__ __forceinline__ int32_t at_or_after(int32_t i) const {  // to: none
    i = i < first ? i : max(i, begin);
    return i < end ? i : to;
  }
  __device__ __forceinline__ bool needs(int32_t i) const { return i < end && (i < first || i >= begin); }
  __device__ __forceinline__ int32_t start() const { return at_or_after(from); }
  __device__ __forceinline__ bool active() const { return start() < to; }
};

// Key tiles of the rows, numbered 0 .. n-1: `first` tiles of first tokens, then the window's from tile `from`
// on.  A row tile may take part in a tile that it sees nothing of; every tile is needed by one row tile.
struct Plan {
  int32_t n = 0, first = 0, from = 0;
  int32_t end = 0;                // keys the rows see: [0, sinks) and [begin, end)
  __device__ __forceinline__ int32_t key0(int32_t i) const { return (i < first ? i : i - first + from) * kTileKeys; }
};

// What the loading warp tells the others: the rows, and which of their key tiles.
struct Item {
  Unit un;
  Plan plan;
  int32_t begin = 0, end = 0;  // key tiles
  Span span[2];
  int32_t parts = 1;           // of the unit; 1: the rows' results are final
  int32_t slot = 0;            // of the partial results
  int32_t more = 0;            // 0: no further rows
};

template <int DP>
struct Smem {
  static constexpr int kHalves = DP / 64;                 // 64 dims = one 128-byte swizzled row
  static constexpr int kHalfBytes = kTileKeys * 128;
  static constexpr int kTileBytes = kHalves * kHalfBytes; // Q, K or V tile
  static constexpr int kStages = DP == 128 ? 2 : 4;
  // Pieces of P, whose products begin as they are ready.  With 64 dims the products are short, and another wait
  // costs more than an early start gives: 6 chunks of 1024 tokens 95 us with one piece, 102 with two; with 128
  // dims 8191 tokens and a window of 1024 91 us with one, 88 with two.
  static constexpr int kPieces = DP == 128 ? 2 : 1;
  // Tensor memory columns: S, P of tile 0 and 1, O of tile 0 and 1.  The row tiles share one S, which is free
  // again as soon as the rows have read it: there is no room for two with 128 dims, and with 64, where there
  // is, taking turns keeps one tile's exponentials beside the other's maxima and exchanges (16384 tokens
  // causal: 686 us, with an S each 807).
  static constexpr int kColP = kTileKeys, kColO = kColP + kTileKeys;
  static_assert(kColO + 2 * DP <= 512, "tensor memory");
  static constexpr int kQ = 0;
  static constexpr int kK = kQ + 2 * kTileBytes;
  static constexpr int kV = kK + kStages * kTileBytes;
  static constexpr int kStats = kV + kStages * kTileBytes;  // (m, sum) of the rows of both tiles, of two items in turn
  static constexpr int kAnswer = kStats + 4 * kTileRows * 8;  // of the launch control, 16 bytes
  static constexpr int kItems = kAnswer + 16;             // two
  static constexpr int kBar = kItems + ((2 * (int)sizeof(Item) + 7) & ~7);
  static constexpr int kBars = 4 + 4 * kStages + 2 + 2 + 2 * kPieces + 4 + 2 + 8 + 4 + 1 + 2;
  static constexpr int kBytes = kBar + kBars * 8 + 16;    // + tensor memory address, abort flag
  static constexpr int kLaunch = kBytes + 1024;           // slack for the 1024-byte alignment
  static_assert(kLaunch > 115 * 1024 && kLaunch <= 227 * 1024, "one block, and its tensor memory, per SM");
};

struct Maps {
  CUtensorMap q;         // 64 dims of a token's heads that share a key head; of 128 rows where they fill them
  CUtensorMap q_row;     // 64 dims of one row
  CUtensorMap k, v;      // one page (or 128 tokens of it) x 64 dims
  CUtensorMap v_rows;    // eight tokens x 64 dims
  CUtensorMap v_row;     // one
};

// ---- tcgen05, mbarrier and TMA ------------------------------------------------------------------
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  return done;
}
// Bounded; gives up early when another role has.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile uint32_t* abort, uint32_t* err,
                                         uint32_t polls = kPolls) {
  for (uint32_t i = 0; i < polls; ++i) {
    if (bar_try(bar, parity)) return true;
    if ((i & 1023) == 1023 && *abort) return false;
  }
  *abort = 1;
  flag_error(err, kErrWait);
  return false;
}
// Asks the launch control for a block of this grid that has not started; the answer (16 bytes) arrives on
// the barrier.  Not to be asked again after a refusal.
__device__ __forceinline__ void ask_for_block(uint32_t answer, uint32_t bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
               ::"r"(answer), "r"(bar) : "memory");
}
// The block of an answer; -1: none is left.
__device__ __forceinline__ int64_t answered_block(uint32_t answer) {
  uint32_t yes, x;
  asm volatile(
      "{\n\t.reg .b128 a;\n\t.reg .pred p;\n\t.reg .b32 y, z, w;\n\tld.shared.b128 a, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\n\tselp.b32 %0, 1, 0, p;\n\tmov.b32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, y, z, w}, a;\n\t}"
      : "=r"(yes), "=r"(x) : "r"(answer) : "memory");
  return yes ? (int64_t)x : -1;
}
// One thread of a converged warp, always the same.
__device__ __forceinline__ bool elected() {
  uint32_t yes;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(yes));
  return yes;
}
// The same value in every lane, known to the compiler as such.
__device__ __forceinline__ int32_t same(int32_t x) { return __shfl_sync(0xffffffffu, x, 0); }
__device__ __forceinline__ void tma_box(uint32_t to, const CUtensorMap* map, int32_t x, int32_t token, int32_t head,
                                        int32_t page, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(to), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(token), "r"(head), "r"(page), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_rows(uint32_t to, const CUtensorMap* map, int32_t x, int32_t head, int32_t token,
                                         uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(to), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(head), "r"(token), "r"(bar) : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Shared-memory operand descriptor, 128-byte swizzle: start address, leading and stride byte offset in
// 16-byte units, version 1, layout 2.  K-major: rows of 128 bytes, 8-row groups `stride` apart (1024).
// MN-major: chunks of 64 MN elements `leading` apart, groups of 8 K rows `stride` apart (1024).
// The upper word is the same for all; the lower one is what moves.
constexpr uint32_t kOperandHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t operand(uint32_t at, uint32_t leading) {
  return ((at >> 4) & 0x3fff) | ((leading >> 4) << 16);
}
// Instruction descriptor, kind::f16: D 32-bit float, A and B of type T, A K-major, B K-major or
// MN-major, M = 128.
template <class T>
constexpr uint32_t instruction(int n, bool b_mn) {
  const uint32_t type = T::kind == 0 ? 1 : 0;
  return (1u << 4) | (type << 7) | (type << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 x, {%1, %5};\n\tmov.b64 y, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}"
      ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(add), "n"(kOperandHigh) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 y, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}"
      ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(add), "n"(kOperandHigh) : "memory");
}
// 16 consecutive columns of this thread's lane.
__device__ __forceinline__ void tmem_load16(uint32_t at, float* x) {
  uint32_t* r = reinterpret_cast<uint32_t*>(x);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at));
}
__device__ __forceinline__ void tmem_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// 16 lanes x 32 (64) columns: of each 8 columns a thread has two of row lane / 4, then the same two of row
// lane / 4 + 8.
__device__ __forceinline__ void tmem_load_rows(uint32_t at, float (&x)[32]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(x);
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at));
}
__device__ __forceinline__ void tmem_load_rows(uint32_t at, float (&x)[16]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(x);
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at));
}
__device__ __forceinline__ void tmem_store_rows(uint32_t at, const float (&x)[16]) {
  const uint32_t* r = reinterpret_cast<const uint32_t*>(x);
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
// 16 lanes x 16 columns, packed pairs of the layout above: of each 4 columns a thread has one of either row.
__device__ __forceinline__ void tmem_store_pairs(uint32_t at, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(at), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// ---- two floats at a time (subnormal numbers kept: the scale may be one, and -inf times a flushed one is NaN) ----
__device__ __forceinline__ uint64_t two(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void split(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// Bits first .. last of a word whose bits stand for the numbers from `base` on.
__device__ __forceinline__ uint32_t bits_of(int32_t first, int32_t last, int32_t base) {
  const int32_t a = max(first - base, 0), b = min(last - base, 31);
  return a > b ? 0 : (0xffffffffu >> (31 - b)) & (0xffffffffu << a);
}

// ---- which key tiles the rows and each of their row tiles need -----------------------------------
__device__ __forceinline__ Plan make_plan(const Unit& un) {
  Plan p;
  if (un.n > 0) {
    p.end = un.begin + un.n - un.sinks;
    p.from = un.begin / kTileKeys;
    p.first = min(p.from, (un.sinks + kTileKeys - 1) / kTileKeys);
    p.n = p.first + (p.end - 1) / kTileKeys - p.from + 1;
  }
  return p;
}
__device__ __forceinline__ Span make_span(const Item& it, const Query& q, int t) {
  const Unit& un = it.un;
  const Plan& p = it.plan;
  Span s;
  s.from = it.begin;
  s.to = it.end;
  if (t * kTileRows >= un.rows) return s;
  s.lo = un.position(q, t * kTileRows);
  s.hi = un.position(q, min(un.rows, (t + 1) * kTileRows) - 1);
  if (s.hi < 0) return s;
  s.first = p.first;
  s.end = min(it.end, p.first + s.hi / kTileKeys - p.from + 1);
  s.begin = p.first;
  // the window tiles before the row tile's own, unless first tokens reach into them
  if (un.begin > 0 && un.sinks <= p.from * kTileKeys) s.begin += max(0, (s.lo + 1 - q.window) / kTileKeys - p.from);
  return s;
}
// Parts of a unit of n key tiles where the launch has `most`.
__device__ __forceinline__ int32_t parts_of(int32_t n, int32_t most) {
  return max(1, min(most, (n + kPartTiles - 1) / kPartTiles));
}
// Partial results: per slot [row][DP] O, then [row][m, sum].
template <int DP>
constexpr int64_t kSlotFloats = (int64_t)kBlockRows * (DP + 2);

// 32 bytes to a 16-byte aligned place.
__device__ __forceinline__ void store32(void* to, const uint32_t* w, bool whole, int32_t bytes) {
  if (whole) {  // 32-byte aligned, all 32 wanted
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                 "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
  } else {
    if (bytes > 0) *static_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
    if (bytes > 16) *(static_cast<uint4*>(to) + 1) = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

template <class T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
    k_kv_prompt(const __grid_constant__ Maps maps, View kv, Batch bt, Query q, int64_t units, int32_t most_parts,
                float* scratch, uint32_t q_tokens, bool ranked) {
  using S = Smem<DP>;
  extern __shared__ uint8_t raw[];
  const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
  uint8_t* sm = raw + (base - smem_addr(raw));
  const int warp = same(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const uint32_t bars = base + S::kBar;
  const uint32_t q_full = bars, q_empty = q_full + 16, k_full = q_empty + 16, k_empty = k_full + 8 * S::kStages,
                 v_full = k_empty + 8 * S::kStages, v_empty = v_full + 8 * S::kStages, s_full = v_empty + 8 * S::kStages,
                 s_read = s_full + 16, p_full = s_read + 16, o_done = p_full + 16 * S::kPieces, o_empty = o_done + 32,
                 met = o_empty + 16, item_full = met + 64,
                 item_empty = item_full + 16, drain = item_empty + 16, answered = drain + 16;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + S::kBar + S::kBars * 8);
  volatile uint32_t* abort = tmem_slot + 1;
  Item* items = reinterpret_cast<Item*>(sm + S::kItems);

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      bar_init(q_full + 8 * t, 1);
      bar_init(q_empty + 8 * t, 1);
      bar_init(s_full + 8 * t, 1);
      bar_init(s_read + 8 * t, 2 * kTileRows);
      for (int b = 0; b < S::kPieces; ++b) bar_init(p_full + 8 * (t * S::kPieces + b), 2 * kTileRows);
      for (int b = 0; b < 2; ++b) bar_init(o_done + 16 * t + 8 * b, 1);
      bar_init(o_empty + 8 * t, 2 * kTileRows);
      for (int w = 0; w < 4; ++w) bar_init(met + 32 * t + 8 * w, 64);
      bar_init(item_full + 8 * t, 1);
      bar_init(item_empty + 8 * t, kReaders);
      bar_init(drain + 8 * t, 1);
    }
    for (int i = 0; i < 4 * S::kStages; ++i) bar_init(k_full + 8 * i, 1);
    bar_init(answered, 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kLoadWarp && lane < sizeof(Maps) / sizeof(CUtensorMap))
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.q) + lane * sizeof(CUtensorMap)) : "memory");
  if (warp == kScoreWarp) {
    // not before the kernel ahead has ended: a block of it on this SM might still want tensor memory
    cudaGridDependencySynchronize();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(tmem_slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;
  cudaGridDependencySynchronize();

  // the next item, for every warp but the loads'; false: no more (or given up).  It stays where it is until
  // the warp gives its place back.
  uint32_t item_turn = 0;
  bool ok = true;
  auto next_item = [&] {
    const uint32_t at = item_turn & 1;
    ok = __all_sync(0xffffffffu, bar_wait(item_full + 8 * at, (item_turn >> 1) & 1, abort, bt.err, kLongPolls));
    return ok && items[at].more != 0;
  };
  auto end_item = [&] {
    __syncwarp();
    if (lane == 0) bar_arrive(item_empty + 8 * (item_turn & 1));
    ++item_turn;
  };

  if (warp >= kScoreWarp) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
  if (warp == kLoadWarp) {
    // ---- items, and loads of K and V: lane j has the j-th page of a key tile ----
    const int32_t page_tokens = 1 << kv.page_log, box = min(page_tokens, kTileKeys), boxes = kTileKeys / box;
    int64_t block = blockIdx.x;
    uint32_t turn = 0, answers = 0, k_issued = 0, v_issued = 0;
    bool asked = false;
    auto tell = [&](const Item& it) {
      const uint32_t at = item_turn & 1;
      ok = __all_sync(0xffffffffu, bar_wait(item_empty + 8 * at, ((item_turn >> 1) & 1) ^ 1, abort, bt.err, kLongPolls));
      if (!ok) return;
      if (lane == 0) {
        items[at] = it;
        bar_arrive(item_full + 8 * at);
      }
      __syncwarp();
      ++item_turn;
    };
    auto ask = [&] {
      if (asked) return;
      asked = true;
      if (lane == 0) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the last answer has been read
        bar_expect(answered, 16);
        ask_for_block(base + S::kAnswer, answered);
      }
      __syncwarp();
    };
    while (ok && block >= 0) {
      // the blocks with the most keys come first
      const uint32_t from_end = (uint32_t)block / (uint32_t)most_parts, u = (uint32_t)units - 1 - from_end;
      const int32_t part = (int32_t)((uint32_t)block - from_end * most_parts);
      Item it;
      it.un = ranked ? find_unit_ranked<kBlockRows>(kv, bt, q, from_end) : find_unit<kBlockRows>(kv, bt, q, u);
      const Unit& un = it.un;
      const Plan& plan = it.plan;
      it.plan = make_plan(un);
      it.parts = parts_of(plan.n, most_parts);
      it.begin = plan.n * part / it.parts;  // n < 2^23
      it.end = plan.n * (part + 1) / it.parts;
      it.span[0] = make_span(it, q, 0);
      it.span[1] = make_span(it, q, 1);
      it.slot = (int32_t)(u * most_parts + part);
      it.more = 1;
      if (un.rows > 0 && part < it.parts) {
        tell(it);
        const int32_t* row = bt.table + (int64_t)un.b * bt.width;
        // lane j's box of a key tile; its page is looked up one tile ahead
        auto box_at = [&](int32_t i) { return plan.key0(i) + lane * box; };
        auto seen = [&](int32_t k) { return k < un.sinks || (k < plan.end && k + box > un.begin); };
        auto look_up = [&](int32_t i) {
          const int32_t k = box_at(i);
          return i < it.end && lane < boxes && seen(k) ? __ldg(row + (k >> kv.page_log)) : kv.pages;
        };
        int32_t ahead = look_up(it.begin);
        for (int32_t i = it.begin; i < it.end && ok; ++i, ++turn) {
          const int st = turn % S::kStages;
          const uint32_t parity = ((turn / S::kStages) & 1) ^ 1;
          const int32_t t0 = box_at(i), t1 = t0 + box;
          int32_t page = ahead;  // a box outside the pages reads zeros
          ahead = look_up(i + 1);
          bool whole = true;
          if (lane < boxes && seen(t0)) {
            whole = t1 <= un.sinks || (t0 >= un.begin && t1 <= plan.end);
            if ((uint32_t)page >= (uint32_t)kv.pages) {
              flag_error(bt.err, kErrTable);
              page = kv.pages;
            }
          }
          const int32_t at = t0 & (page_tokens - 1);
          const uint32_t kb = base + S::kK + st * S::kTileBytes, vb = base + S::kV + st * S::kTileBytes;
          ok = __all_sync(0xffffffffu, bar_wait(k_empty + 8 * st, parity, abort, bt.err));
          if (!ok) break;
          if (lane == 0) bar_expect(k_full + 8 * st, S::kTileBytes);
          __syncwarp();
          if (lane < boxes)
#pragma unroll
            for (int h = 0; h < S::kHalves; ++h)
              tma_box(kb + h * S::kHalfBytes + lane * box * 128, &maps.k, h * 64, at, un.g, page, k_full + 8 * st);
          k_issued = turn + 1;
          if (i + 1 == it.end) ask();
          ok = __all_sync(0xffffffffu, bar_wait(v_empty + 8 * st, parity, abort, bt.err));
          if (!ok) break;
          if (lane == 0) bar_expect(v_full + 8 * st, S::kTileBytes);
          __syncwarp();
          if (lane < boxes && whole)
#pragma unroll
            for (int h = 0; h < S::kHalves; ++h)
              tma_box(vb + h * S::kHalfBytes + lane * box * 128, &maps.v, h * 64, at, un.g, page, v_full + 8 * st);
          // pages that are seen in part: eight rows at a time where those are all seen or all not, else one
          for (uint32_t left = __ballot_sync(0xffffffffu, !whole); left; left &= left - 1) {
            const int j = __ffs(left) - 1;
            const int32_t pj = __shfl_sync(0xffffffffu, page, j), tj = __shfl_sync(0xffffffffu, t0, j);
            const int32_t aj = __shfl_sync(0xffffffffu, at, j);
            auto v_box = [&](const CUtensorMap* map, int32_t r, bool in) {
#pragma unroll
              for (int h = 0; h < S::kHalves; ++h)
                tma_box(vb + h * S::kHalfBytes + (j * box + r) * 128, map, h * 64, aj + r, un.g, in ? pj : kv.pages,
                        v_full + 8 * st);
            };
            auto row_seen = [&](int32_t k) { return k < un.sinks || (k >= un.begin && k < plan.end); };
            const int32_t r8 = lane * 8, k8 = tj + r8;
            const bool some = r8 < box && (k8 < un.sinks || (k8 < plan.end && k8 + 8 > un.begin));
            const bool all = r8 < box && (k8 + 8 <= un.sinks || (k8 >= un.begin && k8 + 8 <= plan.end));
            if (r8 < box && some == all) v_box(&maps.v_rows, r8, all);
            for (uint32_t mixed = __ballot_sync(0xffffffffu, some != all); mixed; mixed &= mixed - 1) {
              const int32_t r = (__ffs(mixed) - 1) * 8 + lane;
              if (lane < 8) v_box(&maps.v_row, r, row_seen(tj + r));
            }
          }
          v_issued = turn + 1;
        }
      }
      if (!ok) break;
      ask();
      ok = __all_sync(0xffffffffu, bar_wait(answered, answers & 1, abort, bt.err));
      if (!ok) break;
      block = answered_block(base + S::kAnswer);
      __syncwarp();
      ++answers;
      asked = false;
    }
    if (ok) tell(Item{});
    if (!ok) {
      // given up: what is in flight into shared memory lands before the block ends
      auto land = [&](uint32_t full, uint32_t issued) {
        for (uint32_t j = issued > S::kStages ? issued - S::kStages : 0; j < issued; ++j)
          for (uint32_t n = 0; n < kPolls && !bar_try(full + 8 * (j % S::kStages), (j / S::kStages) & 1); ++n) {
          }
      };
      land(k_full, k_issued);
      land(v_full, v_issued);
      for (uint32_t n = 0; asked && n < kPolls && !bar_try(answered, answers & 1); ++n) {
      }
    }
  } else if (warp == kScoreWarp) {
    // ---- S of both row tiles in turn, ahead of the rows.  The whole warp runs the loop and one thread
    // issues: descriptors in uniform registers go to the tensor core at once (from inside a one-thread
    // branch each product took about 100 cycles to issue).  Beside the rows' warps every instruction here
    // takes many cycles, so the rows must not have to wait for them: S of the next key tile follows as
    // soon as its columns have been read, not when this tile's weights are used up. ----
    const uint32_t tm = same(tmem);
    const uint32_t q_desc = same(operand(base + S::kQ, 16)), q_desc1 = same(operand(base + S::kQ + S::kTileBytes, 16)), k_desc = operand(base + S::kK, 16);
    uint32_t turn = 0, q_turn = 0;                 // key tiles so far; bit t: turns of tile t's queries
    uint32_t read_turn = 0x3, last = 0;            // bit t: parity of the last phase of s_read[t]; tile of the last S
    auto wait = [&](uint32_t bar, uint32_t parity) {
      ok = ok && __all_sync(0xffffffffu, bar_wait(bar, parity, abort, bt.err));
    };
    while (next_item()) {
      const Item& it = items[item_turn & 1];
      const int32_t to = same(it.end);
#pragma unroll 1
      for (int32_t i = same(it.begin); i < to && ok; ++i, ++turn) {
        const uint32_t st = turn % S::kStages;
        wait(k_full + 8 * st, (turn / S::kStages) & 1);
        const uint32_t b = same(k_desc + st * (S::kTileBytes >> 4));
#pragma unroll
        for (uint32_t t = 0; t < 2; ++t) {
          const Span& span = it.span[t];
          if (!same(span.needs(i))) continue;
          if (same(i == span.start())) wait(q_full + 8 * t, q_turn >> t & 1);
          // all that can be is worked out before the wait: the rows wait for what stands behind it
          const bool early = span.at_or_after(i + 1) >= to;
          wait(s_read + 8 * last, read_turn >> last & 1);  // the S before has been read
          if (!ok) break;
          last = t;
          read_turn ^= 1u << t;
          const bool end = same(early);
          if (end) q_turn ^= 1u << t;
          const uint32_t a = t ? q_desc1 : q_desc, d = tm;
          fence_after();
          if (elected()) {
#pragma unroll
            for (uint32_t ks = 0; ks < DP / 16; ++ks) {
              const uint32_t off = (ks >> 2) * (S::kHalfBytes >> 4) + (ks & 3) * 2;
              mma_ss(d, a + off, b + off, instruction<T>(kTileKeys, false), ks > 0);
            }
            mma_commit(s_full + 8 * t);
            if (end) mma_commit(q_empty + 8 * t);
          }
          __syncwarp();
        }
        if (ok && elected()) mma_commit(k_empty + 8 * st);
        __syncwarp();
      }
      if (!ok) break;
      end_item();
    }
    if (!ok) {  // products in flight end before the tensor memory is given back
      if (elected()) mma_commit(drain);
      for (uint32_t n = 0; n < kPolls && !bar_try(drain, 0); ++n) {
      }
    }
    __syncwarp();
  } else if (warp == kValueWarp) {
    // ---- O += P V of both row tiles in turn ----
    const uint32_t tm = same(tmem), v_desc = operand(base + S::kV, S::kHalfBytes);
    uint32_t turn = 0, p_turn[2] = {0, 0}, active = 0;  // bit t of active: items of tile t
    auto wait = [&](uint32_t bar, uint32_t parity) {
      ok = ok && __all_sync(0xffffffffu, bar_wait(bar, parity, abort, bt.err));
    };
    while (next_item()) {
      const Item& it = items[item_turn & 1];
      const int32_t to = same(it.end);
#pragma unroll 1
      for (int32_t i = same(it.begin); i < to && ok; ++i, ++turn) {
        const uint32_t st = turn % S::kStages;
        wait(v_full + 8 * st, (turn / S::kStages) & 1);
        const uint32_t b = same(v_desc + st * (S::kTileBytes >> 4));
#pragma unroll
        for (uint32_t t = 0; t < 2; ++t) {
          const Span& span = it.span[t];
          if (!same(span.needs(i))) continue;
          const uint32_t add = same(i == span.start() ? 0 : 1);
          if (!add) {
            wait(o_empty + 8 * t, (active >> t & 1) ^ 1);  // the last O has been read
            active ^= 1u << t;
          }
#pragma unroll
          for (int h = 0; h < S::kPieces; ++h) {
            wait(p_full + 8 * (t * S::kPieces + h), p_turn[t] & 1);
            if (!ok) break;
            fence_after();
            if (elected()) {
#pragma unroll
              for (int ks = h * (kTileKeys / 16 / S::kPieces); ks < (h + 1) * (kTileKeys / 16 / S::kPieces); ++ks)
                mma_ts(tm + S::kColO + t * DP, tm + S::kColP + t * (kTileKeys / 2) + ks * 8, b + ks * 128,
                       instruction<T>(DP, true), ks > 0 ? 1 : add);
              if (h == S::kPieces - 1) mma_commit(o_done + 16 * t + 8 * (p_turn[t] & 1));
            }
            __syncwarp();
          }
          ++p_turn[t];
        }
        if (ok && elected()) mma_commit(v_empty + 8 * st);
        __syncwarp();
      }
      if (!ok) break;
      end_item();
    }
    if (!ok) {
      if (elected()) mma_commit(drain + 8);
      for (uint32_t n = 0; n < kPolls && !bar_try(drain + 8, 0); ++n) {
      }
    }
    __syncwarp();
  } else if (warp == kQueryWarp) {
    // ---- queries, as soon as the products have used up the last ones: one box where the heads of whole
    // tokens fill the 128 rows (q_tokens of them), else a box per token, and a row at a time what is
    // cut off at either end ----
    uint32_t turn = 0;  // bit t: of tile t
    for (; next_item(); end_item()) {
      const Item& it = items[item_turn & 1];
      const Unit& un = it.un;
#pragma unroll 1
      for (int t = 0; t < 2 && ok; ++t) {
        if (!it.span[t].active()) continue;
        ok = __all_sync(0xffffffffu, bar_wait(q_empty + 8 * t, (turn >> t & 1) ^ 1, abort, bt.err, kLongPolls));
        if (!ok) break;
        turn ^= 1u << t;
        const uint32_t to = base + S::kQ + t * S::kTileBytes, bar = q_full + 8 * t;
        const int32_t rows = q_tokens ? kTileRows : min(un.rows - t * kTileRows, kTileRows);
        if (lane == 0) bar_expect(bar, rows * 128 * S::kHalves);
        __syncwarp();
        const int32_t token0 = un.token_of(q, t * kTileRows);
        if (q_tokens) {
          if (lane < S::kHalves)
            tma_rows(to + lane * S::kHalfBytes, &maps.q, lane * 64, un.g * q.group, un.token0 + token0, bar);
          continue;
        }
        for (int32_t k = token0 + lane;; k += 32) {
          const int32_t r0 = k * q.group - un.head0 - t * kTileRows, r1 = r0 + q.group;  // rows of token k
          if (r0 >= rows) break;
          const bool whole = r0 >= 0 && r1 <= rows;
          for (int32_t r = max(r0, 0); r < min(r1, rows); r += whole ? q.group : 1)
#pragma unroll
            for (int h = 0; h < S::kHalves; ++h)
              tma_rows(to + h * S::kHalfBytes + r * 128, whole ? &maps.q : &maps.q_row, h * 64, un.g * q.group + r - r0,
                       un.token0 + k, bar);
        }
        __syncwarp();
      }
      if (!ok) break;
    }
    if (!ok) {
      // what is in flight lands before the block ends
      for (int t = 0; t < 2; ++t)
        for (uint32_t n = 0; n < kPolls && !bar_try(q_full + 8 * t, (turn >> t & 1) ^ 1); ++n) {
        }
    }
  } else {
    // ---- rows ----
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRowRegs));
    // A warp has 16 rows: of each 8 keys, a thread two scores of row lane / 4 and two of row lane / 4 + 8 of them.
    const int t = warp >> 3, half = warp >> 2 & 1;
    const int row0 = (warp & 3) * 32 + half * 16 + lane / 4, pair = (lane & 3) * 2;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32 + half * 16) << 16;
    const uint32_t s_at = tmem + lanes, p_at = tmem + S::kColP + t * (kTileKeys / 2) + lanes, o_at = tmem + S::kColO + t * DP;
    const uint32_t meets = met + 32 * t + 8 * (warp & 3);
    const float c = q.scale_log2;
    uint32_t turn = 0;     // key tiles of the row tile so far
    uint32_t results = 0;  // items with results
    // The n-th product into O.  Two barriers in turn: the product n - 2 is done when S of n arrives, so a
    // parity is that of n's own phase or of the one before.
    auto added = [&](uint32_t n) { return bar_wait(o_done + 16 * t + 8 * (n & 1), (n >> 1) & 1, abort, bt.err); };
    for (; next_item(); end_item()) {
      const Item& it = items[item_turn & 1];
      const Unit& un = it.un;
      if (t * kTileRows >= un.rows) continue;
      const Plan plan = it.plan;
      const Span span = it.span[t];
      // positions of the thread's rows, and of the warp's first and last (rows past the last do its work again)
      int32_t pos[2];
      for (int r = 0; r < 2; ++r) pos[r] = un.position(q, min(t * kTileRows + row0 + 8 * r, un.rows - 1));
      const int32_t lo = __shfl_sync(0xffffffffu, pos[0], 0), hi = __shfl_sync(0xffffffffu, pos[1], 31);
      const int32_t alive = un.rows - t * kTileRows;  // rows of the tile
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0, 0};
      bool fresh = true;
      for (int32_t i = span.start(); i < span.end; i = span.at_or_after(i + 1)) {
        const int32_t key0 = plan.key0(i);
        ok = __all_sync(0xffffffffu, bar_wait(s_full + 8 * t, turn & 1, abort, bt.err));
        if (!ok) break;
        fence_after();
        float x[2][32];  // of 64 keys each: [key / 8][row][key % 2]
        tmem_load_rows(s_at, x[0]);
        tmem_load_rows(s_at + 64, x[1]);
        tmem_load_wait();
        fence_before();
        bar_arrive(s_read + 8 * t);
        // which of the four 32 keys any row of the warp sees; not all rows may see them all
        uint32_t live = 0xf;
        if (key0 + kTileKeys - 1 > lo || (q.window && key0 <= hi - q.window && key0 + kTileKeys > q.sinks)) {
          live = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int32_t k = key0 + 32 * j;
            if (k <= hi && (!q.window || k + 31 > lo - q.window || k < q.sinks)) live |= 1u << j;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const int32_t last = pos[r] - k, first = q.window ? last - q.window + 1 : 0, sk = min(q.sinks - 1 - k, last);
              const uint32_t in = (bits_of(first, last, 0) | bits_of(0, sk, 0)) >> pair;
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (!(in >> (e / 2 * 8 + e % 2) & 1)) x[j / 2][(j % 2 * 4 + e / 2) * 4 + r * 2 + e % 2] = -INFINITY;
            }
          }
        }
        float now[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float top[2] = {x[0][2 * r], x[0][2 * r + 1]};
#pragma unroll
          for (int j = 1; j < 16; j += 2)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float a = x[j / 8][j % 8 * 4 + 2 * r + e];
              const float b = j + 1 < 16 ? x[(j + 1) / 8 & 1][(j + 1) % 8 * 4 + 2 * r + e] : -INFINITY;
              top[e] = fmaxf(fmaxf(top[e], a), b);
            }
          // rows past the last hold the scores of whatever query lay there before: they must not move the others' m
          now[r] = row0 + 8 * r < alive ? fmaxf(top[0], top[1]) * c : -INFINITY;
        }
        // of the thread's scores; those of the whole rows are of interest only where some exceed m by too much
        if (__any_sync(0xffffffffu, fresh || now[0] > m[0] + kLag || now[1] > m[1] + kLag)) {
          float f[2];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            now[r] = fmaxf(now[r], __shfl_xor_sync(0xffffffffu, now[r], 1));
            now[r] = fmaxf(m[r], fmaxf(now[r], __shfl_xor_sync(0xffffffffu, now[r], 2)));
            f[r] = exp2_fast(m[r] - (now[r] == -INFINITY ? 0.f : now[r]));
            l[r] *= f[r];
            m[r] = now[r];
          }
          if (!fresh) {
            ok = __all_sync(0xffffffffu, added(turn - 1));  // O is at rest
            if (!ok) break;
            fence_after();
#pragma unroll 1
            for (int j = 0; j < DP; j += 32) {
              float o[16];
              tmem_load_rows(o_at + lanes + j, o);
              tmem_load_wait();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] *= f[e >> 1 & 1];
              tmem_store_rows(o_at + lanes + j, o);
            }
          }
          fresh = false;
        }
        if (turn > 0) {
          ok = __all_sync(0xffffffffu, added(turn - 1));  // the last P has been used up
          if (!ok) break;
        }
        fence_after();
        const uint64_t scale = two(c, c);
        uint64_t shift[2], sum[2] = {0, 0};
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float ref = m[r] == -INFINITY ? 0.f : m[r];
          shift[r] = two(-ref, -ref);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t p[8] = {};
          if (live >> j & 1) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int at = j % 2 * 16 + e * 2;
              uint64_t y = fma2(two(x[j / 2][at], x[j / 2][at + 1]), scale, shift[e & 1]);
              float p0, p1;
              split(y, p0, p1);
              p0 = exp2_fast(p0);
              p1 = exp2_fast(p1);
              y = two(p0, p1);
              sum[e & 1] = add2(sum[e & 1], y);
              p[e] = T::pack(p0, p1);
            }
          }
          tmem_store_pairs(p_at + j * 16, p);
          constexpr int kSteps = 4 / S::kPieces;
          if (j % kSteps == kSteps - 1) {
            tmem_store_wait();
            fence_before();
            bar_arrive(p_full + 8 * (t * S::kPieces + j / kSteps));
          }
        }
        if (!ok) break;
        ++turn;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float l0, l1;
          split(sum[r], l0, l1);
          l[r] += l0 + l1;
        }
      }
      if (!ok) break;
      // ---- results: a thread has a row, and half of its dims; m and l of it come through shared memory ----
      float2* ml = reinterpret_cast<float2*>(sm + S::kStats) + ((results++ & 1) * 2 + t) * kTileRows;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        if (pair == 0) ml[row0 + 8 * r] = make_float2(m[r], l[r]);
      }
      bar_arrive(meets);
      ok = __all_sync(0xffffffffu, bar_wait(meets, (results & 1) ^ 1, abort, bt.err));
      if (!ok) break;
      const int32_t row = (warp & 3) * 32 + lane, at_row = t * kTileRows + row;
      const bool mine_live = at_row < un.rows;
      const float sum = ml[row].y;
      float* slot = scratch + it.slot * kSlotFloats<DP>;
      if (it.parts > 1 && half == 0 && mine_live) *reinterpret_cast<float2*>(slot + kBlockRows * DP + at_row * 2) = ml[row];
      if (fresh) {  // no row of the tile sees a key of the item
        if (it.parts == 1 && half == 0 && mine_live)
          for (int32_t d = 0; d < kv.dim; d += 8) *reinterpret_cast<uint4*>(un.result(kv, q, at_row) + d) = make_uint4(0, 0, 0, 0);
        continue;
      }
      ok = __all_sync(0xffffffffu, added(turn - 1));
      if (!ok) break;
      fence_after();
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      const uint32_t from = o_at + half * (DP / 2) + ((uint32_t)(warp & 3) << 21);
      const int32_t d0 = half * (DP / 2);
      uint16_t* out = un.result(kv, q, at_row) + d0;
      float* part = slot + (int64_t)at_row * DP + d0;
      const bool sectors = ((reinterpret_cast<uintptr_t>(out) | (uint32_t)kv.dim * 2) & 31) == 0;
#pragma unroll 1
      for (int j = 0; j < DP / 2; j += 16) {  // a loop: code that runs once an item waits for its instructions
        float o[16];
        tmem_load16(from + j, o);
        tmem_load_wait();
        if (j == DP / 2 - 16) {
          fence_before();
          bar_arrive(o_empty + 8 * t);
        }
        if (!mine_live) continue;
        if (it.parts == 1) {
          uint32_t w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] = sum == 0.f ? 0 : T::pack(o[2 * e] * inv, o[2 * e + 1] * inv);
          const int32_t bytes = (kv.dim - d0 - j) * 2;
          store32(out + j, w, sectors && bytes >= 32, bytes);
        } else {
          const bool sectors = (reinterpret_cast<uintptr_t>(part) & 31) == 0;
          store32(part + j, reinterpret_cast<const uint32_t*>(o), sectors, 32);
          store32(part + j + 8, reinterpret_cast<const uint32_t*>(o) + 8, sectors, 32);
        }
      }
    }
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  if (warp == kScoreWarp) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

// Joins the parts of a unit, in order: 32 rows a block, four a warp, whose numbers are asked for together
// (finding the unit takes longer than a row: with eight rows a block the join took 25 us where this
// takes 8).
constexpr int kJoinRows = 32, kJoinThreads = 256;
template <class T, int DP>
__global__ void __launch_bounds__(kJoinThreads)
    k_kv_prompt_join(View kv, Batch bt, Query q, int32_t most_parts, const float* scratch) {
  cudaGridDependencySynchronize();
  constexpr int kLanes = DP / 4, kAtOnce = 32 / kLanes;             // lanes a row, rows an access
  constexpr int kPasses = kJoinRows / (kJoinThreads / 32) / kAtOnce;  // of a warp
  const Unit un = find_unit<kBlockRows>(kv, bt, q, blockIdx.x);
  const int32_t parts = parts_of(make_plan(un).n, most_parts);
  const int lane = threadIdx.x & 31, d = lane % kLanes * 4;
  const int32_t row0 = blockIdx.y * kJoinRows + (threadIdx.x >> 5) * kAtOnce * kPasses + lane / kLanes;
  if (parts == 1 || row0 >= un.rows || d >= kv.dim) return;
  const float* from = scratch + (int64_t)blockIdx.x * most_parts * kSlotFloats<DP>;
  float top[kPasses], sum[kPasses] = {}, v[kPasses][4] = {};
#pragma unroll
  for (int i = 0; i < kPasses; ++i) top[i] = -INFINITY;
  for (int32_t p = 0; p < parts; ++p)
#pragma unroll
    for (int i = 0; i < kPasses; ++i)
      top[i] = fmaxf(top[i], from[p * kSlotFloats<DP> + kBlockRows * DP + (row0 + i * kAtOnce) * 2]);
#pragma unroll 2
  for (int32_t p = 0; p < parts; ++p) {
    const float* slot = from + p * kSlotFloats<DP>;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int32_t row = row0 + i * kAtOnce;  // rows past the unit's read its slot's rest, and are not stored
      const float2 ml = *reinterpret_cast<const float2*>(slot + kBlockRows * DP + row * 2);
      const float4 x = *reinterpret_cast<const float4*>(slot + (int64_t)row * DP + d);
      const bool some = ml.x != -INFINITY || ml.y != 0.f;  // else nothing was seen, and no O stored
      const float f = some ? exp2_fast(ml.x - top[i]) : 0.f;
      sum[i] += some ? f * ml.y : 0.f;
      v[i][0] += some ? f * x.x : 0.f;
      v[i][1] += some ? f * x.y : 0.f;
      v[i][2] += some ? f * x.z : 0.f;
      v[i][3] += some ? f * x.w : 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int32_t row = row0 + i * kAtOnce;
    if (row >= un.rows) break;
    const float inv = sum[i] == 0.f ? 0.f : 1.f / sum[i];
    *reinterpret_cast<uint2*>(un.result(kv, q, row) + d) =
        make_uint2(T::pack(v[i][0] * inv, v[i][1] * inv), T::pack(v[i][2] * inv, v[i][3] * inv));
  }
}

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
  static std::atomic<void*> known{nullptr};
  void* p = known.load();
  if (!p) {
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      return nullptr;
    known.store(p);
  }
  return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
}

CUtensorMapDataType type_of(int dtype) {
  return dtype == 0 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

// Queries: boxes of 64 dims x heads x tokens.
bool encode_q(CUtensorMap* map, const View& kv, const Query& q, int dtype, uint32_t heads, uint32_t tokens) {
  const auto enc = encoder();
  if (!enc) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)kv.dim, (cuuint64_t)kv.heads * q.group, (cuuint64_t)q.tokens};
  const cuuint64_t strides[2] = {(cuuint64_t)q.head_stride * 2, (cuuint64_t)q.token_stride * 2};
  const cuuint32_t box[3] = {64, heads, tokens}, ones[3] = {1, 1, 1};
  return enc(map, type_of(dtype), 3, const_cast<uint16_t*>(q.q), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool encode(CUtensorMap* map, const View& kv, int dtype, uint16_t* pages, uint32_t tokens) {
  const auto enc = encoder();
  if (!enc) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)kv.dim, cuuint64_t(1) << kv.page_log, (cuuint64_t)kv.heads, (cuuint64_t)kv.pages};
  // the stride of a single head or page is not used, but has to be a valid one
  const cuuint64_t strides[3] = {(cuuint64_t)kv.token_stride * 2, (cuuint64_t)std::max<int64_t>(kv.head_stride, 8) * 2,
                                 (cuuint64_t)std::max<int64_t>(kv.page_stride, 8) * 2};
  const cuuint32_t box[4] = {64, tokens, 1, 1}, ones[4] = {1, 1, 1, 1};
  return enc(map, type_of(dtype), 4, pages, dims, strides,
             box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class T, int DP>
cudaError_t launch(const View& kv, const Batch& bt, const Query& q, int dtype, const PromptSplit& sp, float* scratch,
                   cudaStream_t st, int* launches) {
  static std::atomic<uint64_t> allowed{0};
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  if (device >= 64 || !(allowed.load() >> device & 1)) {
    e = cudaFuncSetAttribute(k_kv_prompt<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<DP>::kLaunch);
    if (e != cudaSuccess) return e;
    if (device < 64) allowed.fetch_or(uint64_t(1) << device);
  }
  Maps maps;
  const uint32_t box = (uint32_t)std::min(1 << kv.page_log, kTileKeys);
  // whole tokens fill a row tile where the group divides it (units begin at multiples of 256 rows)
  const uint32_t q_tokens = q.group <= kTileRows && kTileRows % q.group == 0 ? kTileRows / q.group : 0;
  if (!encode_q(&maps.q, kv, q, dtype, q.group <= kTileRows ? q.group : 1, std::max(q_tokens, 1u)) ||
      !encode_q(&maps.q_row, kv, q, dtype, 1, 1))
    return cudaErrorInvalidValue;
  if (!encode(&maps.k, kv, dtype, kv.k, box) || !encode(&maps.v, kv, dtype, kv.v, box) ||
      !encode(&maps.v_rows, kv, dtype, kv.v, 8) || !encode(&maps.v_row, kv, dtype, kv.v, 1))
    return cudaErrorInvalidValue;
  e = launch_next(k_kv_prompt<T, DP>, dim3((unsigned)(sp.units * sp.parts)), kThreads, Smem<DP>::kLaunch, st, 1, maps, kv, bt, q,
                  sp.units, sp.parts, scratch, q_tokens, sp.ranked);
  if (e != cudaSuccess) return e;
  *launches += 1;
  if (sp.parts > 1) {
    e = launch_next(k_kv_prompt_join<T, DP>, dim3((unsigned)sp.units, kBlockRows / kJoinRows), kJoinThreads, 0, st, 1, kv, bt, q,
                    sp.parts, scratch);
    if (e != cudaSuccess) return e;
    *launches += 1;
  }
  return cudaGetLastError();
}

}  // namespace

uint64_t PromptSplit::scratch_floats() const {
  return parts > 1 ? (uint64_t)units * parts * kBlockRows * (dim_padded + 2) : 0;
}

bool prompt_strides(const Query& q) {
  const int64_t most = int64_t(1) << 38;
  return q.head_stride >= 8 && q.head_stride < most && q.token_stride >= 8 && q.token_stride < most;
}

PromptSplit plan_prompt(const View& kv, const Batch& bt, const Query& q, int sms) {
  PromptSplit sp;
  sp.dim_padded = kv.dim <= 64 ? 64 : 128;
  // at most ceil(rows / 256) units per sequence and key head
  sp.units = ((int64_t)q.tokens * q.group / kBlockRows + bt.seqs) * kv.heads;
  int64_t keys = (int64_t)bt.width << kv.page_log;
  if (q.window) keys = std::min<int64_t>(keys, (int64_t)q.window + q.sinks + 2 * kTileKeys + kBlockRows);
  // As many parts as bring the blocks near the number of processors, where that leaves each some key tiles: more
  // of them balance better, but each leaves its results in 32 bits for the join.  8192 keys, 8 key heads, 256,
  // 1024 and 2048 rows: 36, 50 and 79 us so, 131, 129 and 128 in one part, 36, 61 and 84 in twice as many.
  const int64_t most = std::min<int64_t>(kMaxParts, keys / (kPartTiles * kTileKeys));
  const int64_t near = (2 * sms + sp.units) / std::max<int64_t>(1, 2 * sp.units);
  sp.parts = (int32_t)std::max<int64_t>(1, std::min(most, near));
  // a few waves are balanced best with the longest units of all sequences first (8 prompts of 512 tokens: 26.9 us in
  // the sequences' order, 24.2 so; 4 of 1024: 35.4 and 30.0; 8 of up to 2000, 2 key heads: 55.8 and 45.7; 32 of up to 256:
  // 25.4 and 23.8; what it costs where there is nothing to balance: 2 of 1024 23.6 and 24.1, 6 of 700 with a window of 200
  // 27.0 and 27.5); with more waves a sequence's units follow one another, for its keys to stay in L2
  sp.ranked = sp.parts == 1 && bt.seqs > 1 && bt.seqs <= 32 && sp.units <= 4 * (int64_t)sms;
  return sp;
}

cudaError_t launch_prompt(const View& kv, const Batch& bt, const Query& q, int dtype, const PromptSplit& sp,
                          float* scratch, cudaStream_t st, int* launches) {
  const bool small = sp.dim_padded == 64;
  if (dtype == 0)
    return small ? launch<Bf16, 64>(kv, bt, q, dtype, sp, scratch, st, launches)
                 : launch<Bf16, 128>(kv, bt, q, dtype, sp, scratch, st, launches);
  return small ? launch<Fp16, 64>(kv, bt, q, dtype, sp, scratch, st, launches)
               : launch<Fp16, 128>(kv, bt, q, dtype, sp, scratch, st, launches);
}

}  // namespace kv
}  // namespace bfvgpu
