// Attention of prompts over the paged cache on the 5th-generation tensor cores.
//
// Rows of one (sequence, key head) are packed token by token, the query heads of the group side by
// side, so that a block's 256 rows (two tiles of 128) share every key it loads.  Per tile of 128 keys:
//   S = Q K^T            tcgen05.mma 128 x 128 x dim, Q and K from shared memory, S in tensor memory
//   P = 2^(c S - m)      one thread per row, the row's 128 scores in registers; P in 16 bits
//   O += P V             tcgen05.mma 128 x dim x 128, P from tensor memory, V from shared memory
// m is the row's reference exponent.  It starts as the running maximum and follows it only when the
// maximum has grown by more than 8: until then weights of up to 2^8 stay far inside both 16-bit types
// and the 32-bit sums, and O need not be rescaled.  The sum of the weights is kept in 32 bits, from
// the weights before they are rounded to 16 bits for the product.
//
// Roles: warps 0-3 and 4-7 hold the rows of tile 0 and 1, warp 8 issues the products, warp 9 the loads of K
// and V, warps 10 and 11 load the queries of tile 0 and 1.  While one tile's rows are in their
// exponentials, the other tile's products run.  A block is resident on its SM for the whole launch and
// takes over the blocks that have not started yet (cluster launch control), so that the loads of the
// next rows and the results of the last ones run under the products in between.
// K and V arrive by TMA page by page as the table names them, in the 128-byte swizzle (K as K-major,
// V as MN-major operand).  Only visible tokens of V are loaded: what no row of the block sees may
// hold NaN (unwritten rest of a page, pages given up), and 0 x NaN would reach every row.  Such
// pages are read row by row, the other rows filled with zeros.
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
constexpr int kThreads = 384;         // two warpgroups of rows, one of the issuing warps
constexpr int kMmaWarp = 8, kLoadWarp = 9, kQueryWarp = 10;
constexpr int kReaders = 11;          // warps that are told of the next rows: all but the loads' own
// Registers a thread: launched with 168 (384 x 168 of the SM's 65536); the issuing warpgroup keeps 64 and
// the rows take 216: 128 x 64 + 256 x 216 <= 384 x 168.
constexpr int kIssueRegs = 64, kRowRegs = 216;
constexpr float kLag = 8.f;           // how far m may stay behind the running maximum
constexpr uint32_t kPolls = 1u << 20;     // of a wait for the next step before it gives up
constexpr uint32_t kLongPolls = 1u << 27; // of a wait that may span all keys of other rows
constexpr int kPolynomial = 6;             // of every 8 weights, the two from this one on go by polynomial
constexpr int kPartTiles = 8;         // key tiles that a part has at least
constexpr int kMaxParts = 16;

// What the loading warp tells the others: the rows, and which of their key tiles.
struct Item {
  Unit un;
  int32_t begin = 0, end = 0;  // key tiles
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
  // Tensor memory columns: S of tile 0 and 1, O of tile 0 and 1, and with 64 dims P of tile 0 and 1.  With 128
  // there is no room for P but over its own S, so the next S waits until P is used up; with 64 it
  // follows as soon as S has been read.
  static constexpr bool kOwnP = DP == 64;
  static constexpr int kColO = 2 * kTileKeys, kColP = kOwnP ? kColO + 2 * DP : 0;
  static constexpr int kPitchP = kOwnP ? kTileKeys / 2 : kTileKeys;
  static constexpr int kQ = 0;
  static constexpr int kK = kQ + 2 * kTileBytes;
  static constexpr int kV = kK + kStages * kTileBytes;
  static constexpr int kOut = kV + kStages * kTileBytes;  // 128 bytes of each row, per warp
  static constexpr int kAnswer = kOut + 8 * 32 * 128;     // of the launch control, 16 bytes
  static constexpr int kItems = kAnswer + 16;             // two
  static constexpr int kBar = kItems + ((2 * (int)sizeof(Item) + 7) & ~7);
  static constexpr int kBars = 4 + 4 * kStages + 4 + 4 + 4 + 2 + 4 + 2;
  static constexpr int kBytes = kBar + kBars * 8 + 16;    // + tensor memory address, abort flag
  static constexpr int kLaunch = kBytes + 1024;           // slack for the 1024-byte alignment
  static_assert(kLaunch > 115 * 1024 && kLaunch <= 227 * 1024, "one block, and its tensor memory, per SM");
};

struct Maps {
  CUtensorMap k, v;      // one page (or 128 tokens of it) x 64 dims
  CUtensorMap v_row;     // one token x 64 dims
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
// The same in one place for the issuing warps, which read their instructions through caches that the rows'
// long loops keep sweeping: what counts for them is how little code they run.
__device__ __noinline__ bool bar_wait_shared(uint32_t bar, uint32_t parity, volatile uint32_t* abort, uint32_t* err,
                                             uint32_t polls) {
  return __all_sync(0xffffffffu, bar_wait(bar, parity, abort, err, polls));
}
__device__ __forceinline__ void tma_box(uint32_t to, const CUtensorMap* map, int32_t x, int32_t token, int32_t head,
                                        int32_t page, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(to), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(token), "r"(head), "r"(page), "r"(bar) : "memory");
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
// 32 consecutive columns of this thread's lane.
__device__ __forceinline__ void tmem_load(uint32_t at, float* x) {
  uint32_t* r = reinterpret_cast<uint32_t*>(x);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at));
}
__device__ __forceinline__ void tmem_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_store32(uint32_t at, const float* x) {
  const uint32_t* r = reinterpret_cast<const uint32_t*>(x);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
        "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
        "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// ---- two floats at a time, and weights without the special-function unit --------------------------
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
  asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.ftz.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.ftz.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max_or_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// 2^x for two x <= 8 on the multiply-add pipes: x = n + f, n the nearest integer (Cody and Waite's reduction,
// by adding and subtracting 1.5 2^23), 2^f by a degree-5 polynomial on [-1/2, 1/2] (Remez exchange on the
// relative error: 2^-22), times 2^n from the bits.  x below -127 gives 0, NaN gives NaN.
__device__ __forceinline__ uint64_t exp2_two(uint64_t x) {
  constexpr float kShift = 12582912.f;
  float a, b;
  split(x, a, b);
  x = two(max_or_nan(a, -127.f), max_or_nan(b, -127.f));
  const uint64_t n = add2(x, two(kShift, kShift));
  const uint64_t f = add2(x, mul2(add2(n, two(-kShift, -kShift)), two(-1.f, -1.f)));
  uint64_t p = two(1.3276472454890609e-3f, 1.3276472454890609e-3f);
  p = fma2(p, f, two(9.675540961325169e-3f, 9.675540961325169e-3f));
  p = fma2(p, f, two(5.550713092088699e-2f, 5.550713092088699e-2f));
  p = fma2(p, f, two(2.4022120237350464e-1f, 2.4022120237350464e-1f));
  p = fma2(p, f, two(6.931469440460205e-1f, 6.931469440460205e-1f));
  p = fma2(p, f, two(1.f, 1.f));
  split(n, a, b);
  return mul2(p, two(__int_as_float((__float_as_int(a) + 127) << 23), __int_as_float((__float_as_int(b) + 127) << 23)));
}
// Bits first .. last of a word whose bits stand for the numbers from `base` on.
__device__ __forceinline__ uint32_t bits_of(int32_t first, int32_t last, int32_t base) {
  const int32_t a = max(first - base, 0), b = min(last - base, 31);
  return a > b ? 0 : (0xffffffffu >> (31 - b)) & (0xffffffffu << a);
}

// ---- which key tiles the rows and each of their row tiles need -----------------------------------
// The rows' key tiles are numbered 0 .. n-1: `first` tiles of first tokens, then the window's from tile
// `from` on.  A row tile needs [0, first) and [begin, end).  It may take part in a tile that it sees
// nothing of; every tile is needed by one row tile.
struct Plan {
  int32_t n = 0, first = 0, from = 0;
  int32_t end = 0;                // keys the rows see: [0, sinks) and [begin, end)
  __device__ __forceinline__ int32_t key0(int32_t i) const { return (i < first ? i : i - first + from) * kTileKeys; }
};
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
struct Span {
  int32_t lo = 0, hi = -1;  // positions of the rows (hi < 0: no row sees a key)
  // the item's key tiles that the row tile needs: [from, first) and [begin, end), in the item's [from, to)
  int32_t first = 0, begin = 0, end = 0, from = 0, to = 0;
  __device__ __forceinline__ int32_t at_or_after(int32_t i) const {  // to: none
    i = i < first ? i : max(i, begin);
    return i < end ? i : to;
  }
  __device__ __forceinline__ int32_t start() const { return at_or_after(from); }
  __device__ __forceinline__ bool active() const { return start() < to; }
};
__device__ __forceinline__ Span make_span(const Item& it, const Query& q, const Plan& p, int t) {
  const Unit& un = it.un;
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

// 128 bytes of each of the warp's 32 rows: every lane has its own row's; stored by whole rows.
template <class To>
__device__ __forceinline__ void store_rows(uint8_t* stage, const uint32_t* w, int lane, int rows, int bytes, To to) {
#pragma unroll
  for (int c = 0; c < 8; ++c)
    *reinterpret_cast<uint4*>(stage + lane * 128 + ((c ^ (lane & 7)) << 4)) =
        make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
  __syncwarp();
  const int c = lane & 7;
#pragma unroll
  for (int n = 0; n < 8; ++n) {
    const int r = n * 4 + (lane >> 3);
    if (r < rows && c * 16 < bytes)
      *reinterpret_cast<uint4*>(to(r) + c * 16) = *reinterpret_cast<const uint4*>(stage + r * 128 + ((c ^ (r & 7)) << 4));
  }
  __syncwarp();
}

template <class T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
    k_kv_prompt(const __grid_constant__ Maps maps, View kv, Batch bt, Query q, int64_t units, int32_t most_parts,
                float* scratch) {
  using S = Smem<DP>;
  extern __shared__ uint8_t raw[];
  const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
  uint8_t* sm = raw + (base - smem_addr(raw));
  const int warp = same(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const uint32_t bars = base + S::kBar;
  const uint32_t q_full = bars, q_empty = q_full + 16, k_full = q_empty + 16, k_empty = k_full + 8 * S::kStages,
                 v_full = k_empty + 8 * S::kStages, v_empty = v_full + 8 * S::kStages, s_full = v_empty + 8 * S::kStages,
                 s_read = s_full + 16, p_half = s_read + 16, o_done = p_half + 32, o_empty = o_done + 32,
                 item_full = o_empty + 16,
                 item_empty = item_full + 16, answered = item_empty + 16, drain = answered + 8;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + S::kBar + S::kBars * 8);
  volatile uint32_t* abort = tmem_slot + 1;
  Item* items = reinterpret_cast<Item*>(sm + S::kItems);

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      bar_init(q_full + 8 * t, 32);
      bar_init(q_empty + 8 * t, 1);
      bar_init(s_full + 8 * t, 1);
      bar_init(p_half + 16 * t, kTileRows);
      bar_init(p_half + 16 * t + 8, kTileRows);
      bar_init(s_read + 8 * t, kTileRows);
      bar_init(o_done + 16 * t, 1);
      bar_init(o_done + 16 * t + 8, 1);
      bar_init(o_empty + 8 * t, kTileRows);
      bar_init(item_full + 8 * t, 1);
      bar_init(item_empty + 8 * t, kReaders);
    }
    for (int i = 0; i < 4 * S::kStages; ++i) bar_init(k_full + 8 * i, 1);
    bar_init(answered, 1);
    bar_init(drain, 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(tmem_slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;

  // the next item, for every warp but the loads'; false: no more (or given up)
  uint32_t item_turn = 0;
  bool ok = true;
  auto next_item = [&](Item& it) {
    const uint32_t at = item_turn & 1;
    ok = __all_sync(0xffffffffu, bar_wait(item_full + 8 * at, (item_turn >> 1) & 1, abort, bt.err, kLongPolls));
    if (!ok) return false;
    it = items[at];
    __syncwarp();
    if (lane == 0) bar_arrive(item_empty + 8 * at);
    ++item_turn;
    return it.more != 0;
  };

  if (warp >= kMmaWarp) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
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
      const int64_t u = units - 1 - block / most_parts;
      const int32_t part = (int32_t)(block % most_parts);
      Item it;
      it.un = find_unit<kBlockRows>(kv, bt, q, u);
      const Unit& un = it.un;
      const Plan plan = make_plan(un);
      it.parts = parts_of(plan.n, most_parts);
      it.begin = (int32_t)((int64_t)plan.n * part / it.parts);
      it.end = (int32_t)((int64_t)plan.n * (part + 1) / it.parts);
      it.slot = (int32_t)(u * most_parts + part);
      it.more = 1;
      if (un.rows > 0 && part < it.parts) {
        tell(it);
        const int32_t* row = bt.table + (int64_t)un.b * bt.width;
        for (int32_t i = it.begin; i < it.end && ok; ++i, ++turn) {
          const int st = turn % S::kStages;
          const uint32_t parity = ((turn / S::kStages) & 1) ^ 1;
          const int32_t t0 = plan.key0(i) + lane * box, t1 = t0 + box;
          int32_t page = kv.pages;  // a box outside the pages reads zeros
          bool whole = true;
          if (lane < boxes) {
            const bool in = t0 < un.sinks || (t0 < plan.end && t1 > un.begin);
            whole = !in || t1 <= un.sinks || (t0 >= un.begin && t1 <= plan.end);
            if (in) {
              page = __ldg(row + (t0 >> kv.page_log));
              if ((uint32_t)page >= (uint32_t)kv.pages) {
                flag_error(bt.err, kErrTable);
                page = kv.pages;
              }
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
          for (uint32_t left = __ballot_sync(0xffffffffu, !whole); left; left &= left - 1) {
            const int j = __ffs(left) - 1;
            const int32_t pj = __shfl_sync(0xffffffffu, page, j), tj = __shfl_sync(0xffffffffu, t0, j);
            const int32_t aj = __shfl_sync(0xffffffffu, at, j);
            for (int32_t r = lane; r < box; r += 32) {
              const int32_t tok = tj + r;
              const bool seen = tok < un.sinks || (tok >= un.begin && tok < plan.end);
#pragma unroll
              for (int h = 0; h < S::kHalves; ++h)
                tma_box(vb + h * S::kHalfBytes + (j * box + r) * 128, &maps.v_row, h * 64, aj + r, un.g,
                        seen ? pj : kv.pages, v_full + 8 * st);
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
  } else if (warp == kMmaWarp) {
    // ---- products.  The whole warp runs the loop and one thread issues: descriptors in uniform registers
    // go to the tensor core at once (from inside a one-thread branch each product took about 100 cycles
    // to issue).  One copy of the code serves both row tiles, which take turns as `x`: unrolled for the two,
    // the loop spent most of its time fetching instructions. ----
    struct Tile {
      uint32_t t = 0;                   // 0, 1
      Span span;
      int32_t s_next = 0, p_next = 0;   // next key tile of its S, and of its P
      uint32_t s_turn = 0, p_turn = 0, active = 0;
    };
    Tile x, y;
    y.t = 1;
    const uint32_t tm = same(tmem);
    const uint32_t q_desc = operand(base + S::kQ, 16), k_desc = operand(base + S::kK, 16),
                   v_desc = operand(base + S::kV, S::kHalfBytes);
    uint32_t turn0 = 0;  // the ring's turn of the item's first key tile
    auto wait = [&](uint32_t bar, uint32_t parity) {
      ok = ok && (bar_try(bar, parity) || bar_wait_shared(bar, parity, abort, bt.err, kPolls));
      ok = __all_sync(0xffffffffu, ok);
    };
    Item it;
    while (next_item(it)) {
      const Plan plan = make_plan(it.un);
      x.span = make_span(it, q, plan, 0);
      y.span = make_span(it, q, plan, 1);
      const int32_t from = same(x.span.from), to = same(x.span.to);
      x.s_next = x.p_next = x.span.start();
      y.s_next = y.p_next = y.span.start();
      // key tiles whose K and V are given back: as soon as both row tiles are past them, before this warp
      // waits for later ones
      int32_t k_free = from, v_free = from;
      auto turn_of = [&](int32_t i) { return turn0 + (uint32_t)(i - from); };
      auto give_back = [&](uint32_t empty, int32_t& done, int32_t free) {
#pragma unroll 1
        for (; done < free; ++done)
          if (elected()) mma_commit(empty + 8 * (turn_of(done) % S::kStages));
        __syncwarp();
      };
      auto product_s = [&](bool first) {
        const int32_t i = x.s_next;
        const uint32_t turn = turn_of(i), st = turn % S::kStages;
        if (first) wait(q_full + 8 * x.t, x.active & 1);
        if (S::kOwnP) wait(s_read + 8 * x.t, (x.s_turn & 1) ^ 1);  // the last S has been read
        wait(k_full + 8 * st, (turn / S::kStages) & 1);
        if (!ok) return;
        x.s_next = x.span.at_or_after(i + 1);
        fence_after();
        const bool last = x.s_next >= to;
        const uint32_t d = same(tm + x.t * kTileKeys), full = s_full + 8 * x.t, empty = q_empty + 8 * x.t;
        uint32_t a = same(q_desc + x.t * (S::kTileBytes >> 4)), b = same(k_desc + st * (S::kTileBytes >> 4));
        if (elected()) {
#pragma unroll 1
          for (uint32_t h = 0; h < S::kHalves; ++h) {
#pragma unroll
            for (uint32_t ks = 0; ks < 4; ++ks)
              mma_ss(d, a + 2 * ks, b + 2 * ks, instruction<T>(kTileKeys, false), ks > 0 ? 1 : h);
            a += S::kHalfBytes >> 4;
            b += S::kHalfBytes >> 4;
          }
          mma_commit(full);
          if (last) mma_commit(empty);
        }
        __syncwarp();
        ++x.s_turn;
        give_back(k_empty, k_free, min(x.s_next, y.s_next));
      };
      auto product_o = [&](int32_t i) {
        const uint32_t turn = turn_of(i), st = turn % S::kStages;
        const bool first = i == x.span.start();
        wait(v_full + 8 * st, (turn / S::kStages) & 1);
        if (first) wait(o_empty + 8 * x.t, (x.active & 1) ^ 1);
        x.p_next = x.span.at_or_after(i + 1);
        uint32_t add = same(first ? 0 : 1);
        const uint32_t d = same(tm + S::kColO + x.t * DP), done = o_done + 16 * x.t + 8 * (x.p_turn & 1);
        uint32_t a = same(tm + S::kColP + x.t * S::kPitchP), b = same(v_desc + st * (S::kTileBytes >> 4));
#pragma unroll 1
        for (uint32_t h = 0; h < 2; ++h) {
          wait(p_half + 16 * x.t + 8 * h, x.p_turn & 1);
          if (!ok) return;
          fence_after();
          if (elected()) {
#pragma unroll
            for (int ks = 0; ks < kTileKeys / 32; ++ks)
              mma_ts(d, a + ks * 8, b + ks * 128, instruction<T>(DP, true), ks > 0 ? 1 : add);
            if (h) mma_commit(done);
          }
          __syncwarp();
          add = 1;
          a += kTileKeys / 4;
          b += kTileKeys * 4;
        }
        ++x.p_turn;
        if (first) ++x.active;
        give_back(v_empty, v_free, min(x.p_next, y.p_next));
      };
      // before the first P: the first S of both; then P of both in turn, and the S that can follow
#pragma unroll 1
      for (int32_t i = from - 1; i < to && ok; ++i) {
#pragma unroll 1
        for (int n = 0; n < 2 && ok; ++n) {
          const bool mine = i < from || x.p_next == i;
          if (!S::kOwnP && mine && i >= from) product_o(i);
          if (mine && ok && x.s_next < to) product_s(i < from);
          const Tile other = y;
          y = x;
          x = other;
        }
        if (S::kOwnP && i >= from)
#pragma unroll 1
          for (int n = 0; n < 2 && ok; ++n) {
            if (x.p_next == i) product_o(i);
            const Tile other = y;
            y = x;
            x = other;
          }
      }
      if (!ok) break;
      turn0 += (uint32_t)(to - from);
    }
    if (!ok) {  // products in flight end before the tensor memory is given back
      if (elected()) mma_commit(drain);
      for (uint32_t n = 0; n < kPolls && !bar_try(drain, 0); ++n) {
      }
      __syncwarp();
    }
  } else if (warp >= kQueryWarp) {
    // ---- queries of one row tile, as soon as the products have used up the last ones ----
    const int t = warp - kQueryWarp;
    const uint32_t qs = base + S::kQ + t * S::kTileBytes;
    constexpr int kChunks = DP / 8;
    const int chunk = lane % kChunks;
    uint32_t turn = 0;
    Item it;
    while (next_item(it)) {
      const Plan plan = make_plan(it.un);
      if (!make_span(it, q, plan, t).active()) continue;
      ok = __all_sync(0xffffffffu, bar_wait(q_empty + 8 * t, (turn & 1) ^ 1, abort, bt.err, kLongPolls));
      if (!ok) break;
      // row lane / kChunks and every kStep-th after it; the query's place moves by a constant, and by another
      // where the heads of the group start over
      constexpr int kStep = 32 / kChunks;
      const int r0 = lane / kChunks, rows = it.un.rows - t * kTileRows;
      const int32_t dt = it.un.token_of(q, t * kTileRows + r0);
      int32_t head = it.un.head0 + t * kTileRows + r0 - dt * q.group;
      const uint16_t* from = it.un.query(q, t * kTileRows + r0) + chunk * 8;
      const int32_t tokens = kStep / q.group, heads = kStep - tokens * q.group;
      const int64_t step = tokens * q.token_stride + heads * q.head_stride, over = q.token_stride - q.group * q.head_stride;
#pragma unroll 8
      for (int r = r0; r < kTileRows; r += kStep) {
        const uint32_t n = r < rows && chunk * 8 < kv.dim ? 16 : 0;  // 0: zeros
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                     ::"r"(qs + (chunk >> 3) * S::kHalfBytes + r * 128 + (((chunk & 7) ^ (r & 7)) << 4)),
                     "l"(n ? from : q.q), "r"(n) : "memory");
        from += step;
        head += heads;
        if (head >= q.group) {
          head -= q.group;
          from += over;
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      bar_arrive(q_full + 8 * t);
      ++turn;
    }
  } else {
    // ---- rows ----
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRowRegs));
    const int t = warp >> 2, row = threadIdx.x & 127;
    uint8_t* stage = sm + S::kOut + warp * 32 * 128;
    const uint32_t quadrant = (uint32_t)(warp & 3) << 21;  // lanes 32 (warp % 4) ..
    const uint32_t s_at = tmem + t * kTileKeys + quadrant, o_at = tmem + S::kColO + t * DP + quadrant;
    const uint32_t p_at = tmem + S::kColP + t * S::kPitchP + quadrant;
    const float c = q.scale_log2;
    uint32_t turn = 0;  // key tiles of the row tile so far
    // The n-th product into O.  Two barriers in turn: the product n - 2 is done when S of n arrives, so a
    // parity is that of n's own phase or of the one before.
    auto added = [&](uint32_t n) { return bar_wait(o_done + 16 * t + 8 * (n & 1), (n >> 1) & 1, abort, bt.err); };
    Item it;
    while (next_item(it)) {
      const Unit& un = it.un;
      const int32_t row0 = t * kTileRows + (warp & 3) * 32, rows = un.rows - row0;  // the warp's
      if (t * kTileRows >= un.rows) continue;
      const Plan plan = make_plan(un);
      const Span span = make_span(it, q, plan, t);
      const int32_t pos = un.position(q, min(t * kTileRows + row, un.rows - 1));  // rows past the last do its work again
      float m = -INFINITY, l = 0;
      bool fresh = true;
      for (int32_t i = span.start(); i < it.end; i = span.at_or_after(i + 1)) {
        const int32_t key0 = plan.key0(i);
        ok = __all_sync(0xffffffffu, bar_wait(s_full + 8 * t, turn & 1, abort, bt.err));
        if (!ok) break;
        fence_after();
        float x[kTileKeys];
#pragma unroll
        for (int j = 0; j < kTileKeys; j += 32) tmem_load(s_at + j, x + j);
        tmem_load_wait();
        if (S::kOwnP) {
          fence_before();
          bar_arrive(s_read + 8 * t);
        }
        const bool cut_end = key0 + kTileKeys - 1 > span.lo;
        const bool cut_begin = q.window && key0 <= span.hi - q.window && key0 + kTileKeys > q.sinks;
        if (cut_end || cut_begin) {
          const int32_t hi = pos - key0, lo = q.window ? hi - q.window + 1 : 0, sk = min(q.sinks - 1 - key0, hi);
#pragma unroll
          for (int j = 0; j < kTileKeys; j += 32) {
            const uint32_t seen = bits_of(lo, hi, j) | bits_of(0, sk, j);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!(seen >> e & 1)) x[j + e] = -INFINITY;
          }
        }
        float top[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int j = 4; j + 8 <= kTileKeys + 4; j += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            top[e] = fmaxf(fmaxf(top[e], x[j + e]), j + 4 + e < kTileKeys ? x[j + 4 + e] : -INFINITY);
        const float now = fmaxf(m, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * c);
        if (fresh) {
          fresh = false;
          m = now;
        } else if (__any_sync(0xffffffffu, now > m + kLag)) {
          ok = __all_sync(0xffffffffu, added(turn - 1));  // O is at rest
          if (!ok) break;
          fence_after();
          const float f = exp2_fast(m - (now == -INFINITY ? 0.f : now));
          l *= f;
          m = now;
#pragma unroll
          for (int j = 0; j < DP; j += 32) {
            float o[32];
            tmem_load(o_at + j, o);
            tmem_load_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] *= f;
            tmem_store32(o_at + j, o);
          }
        }
        const float ref = m == -INFINITY ? 0.f : m;
        const uint64_t scale = two(c, c), shift = two(-ref, -ref);
        uint64_t sum[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < kTileKeys; j += 32) {
          uint32_t p[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            uint64_t y = fma2(two(x[j + e], x[j + e + 1]), scale, shift);
            float p0, p1;
            if (e % 8 == kPolynomial) {
              y = exp2_two(y);
              split(y, p0, p1);
            } else {
              split(y, p0, p1);
              p0 = exp2_fast(p0);
              p1 = exp2_fast(p1);
              y = two(p0, p1);
            }
            sum[e / 2 & 1] = add2(sum[e / 2 & 1], y);
            p[e / 2] = T::pack(p0, p1);
          }
          if (S::kOwnP && j == 0 && turn > 0) {  // the last P has been used up
            ok = __all_sync(0xffffffffu, added(turn - 1));
            if (!ok) break;
            fence_after();
          }
          tmem_store16(p_at + j / 2, p);
          if (j == kTileKeys / 2 - 32 || j == kTileKeys - 32) {  // the product of a half can begin
            tmem_store_wait();
            fence_before();
            bar_arrive(p_half + 16 * t + (j == kTileKeys - 32 ? 8 : 0));
          }
        }
        if (!ok) break;
        ++turn;
        float l0, l1;
        split(add2(sum[0], sum[1]), l0, l1);
        l += l0 + l1;
      }
      if (!ok) break;
      // ---- results ----
      const int32_t whole = min(rows, 32);
      float* slot = scratch + it.slot * kSlotFloats<DP>;
      if (it.parts > 1 && lane < rows)
        *reinterpret_cast<float2*>(slot + kBlockRows * DP + (row0 + lane) * 2) = make_float2(m, l);
      if (fresh) {  // no row of the tile sees a key of the item
        if (it.parts == 1)
          for (int r = 0; r < whole; ++r)
            if (lane * 8 < kv.dim) *reinterpret_cast<uint4*>(un.result(kv, q, row0 + r) + lane * 8) = make_uint4(0, 0, 0, 0);
        continue;
      }
      ok = __all_sync(0xffffffffu, added(turn - 1));
      if (!ok) break;
      fence_after();
      float o[DP];
#pragma unroll
      for (int j = 0; j < DP; j += 32) tmem_load(o_at + j, o + j);
      tmem_load_wait();
      fence_before();
      bar_arrive(o_empty + 8 * t);
      if (it.parts == 1) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        uint16_t* out = un.results(kv, q);
#pragma unroll
        for (int h = 0; h < S::kHalves; ++h) {
          uint32_t w[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) w[e] = l == 0.f ? 0 : T::pack(o[h * 64 + 2 * e] * inv, o[h * 64 + 2 * e + 1] * inv);
          store_rows(stage, w, lane, whole, (kv.dim - h * 64) * 2, [&](int r) {
            return reinterpret_cast<uint8_t*>(out + (int64_t)un.result_row(kv, q, row0 + r) * kv.dim + h * 64);
          });
        }
      } else {
#pragma unroll
        for (int j = 0; j < DP; j += 32)
          store_rows(stage, reinterpret_cast<const uint32_t*>(o + j), lane, whole, 128,
                     [&](int r) { return reinterpret_cast<uint8_t*>(slot + (row0 + r) * DP + j); });
      }
    }
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

// Joins the parts of 32 rows of a unit, in order.
template <class T, int DP>
__global__ void __launch_bounds__(256)
    k_kv_prompt_join(View kv, Batch bt, Query q, int32_t most_parts, const float* scratch) {
  const Unit un = find_unit<kBlockRows>(kv, bt, q, blockIdx.x);
  const int32_t parts = parts_of(make_plan(un).n, most_parts);
  if (parts == 1) return;
  const float* from = scratch + (int64_t)blockIdx.x * most_parts * kSlotFloats<DP>;
  for (int32_t e = threadIdx.x * 4; e < 32 * DP; e += 256 * 4) {
    const int32_t row = blockIdx.y * 32 + e / DP, d = e % DP;
    if (row >= un.rows || d >= kv.dim) continue;
    float top = -INFINITY;
    for (int32_t p = 0; p < parts; ++p) top = fmaxf(top, from[p * kSlotFloats<DP> + kBlockRows * DP + row * 2]);
    float sum = 0, v[4] = {0, 0, 0, 0};
    for (int32_t p = 0; p < parts; ++p) {
      const float* slot = from + p * kSlotFloats<DP>;
      const float2 ml = *reinterpret_cast<const float2*>(slot + kBlockRows * DP + row * 2);
      if (ml.x == -INFINITY && ml.y == 0.f) continue;  // nothing seen: no O was stored
      const float f = exp2_fast(ml.x - top);
      const float4 x = *reinterpret_cast<const float4*>(slot + (int64_t)row * DP + d);
      sum += f * ml.y;
      v[0] += f * x.x;
      v[1] += f * x.y;
      v[2] += f * x.z;
      v[3] += f * x.w;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    *reinterpret_cast<uint2*>(un.result(kv, q, row) + d) =
        make_uint2(T::pack(v[0] * inv, v[1] * inv), T::pack(v[2] * inv, v[3] * inv));
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

bool encode(CUtensorMap* map, const View& kv, int dtype, uint16_t* pages, uint32_t tokens) {
  const auto enc = encoder();
  if (!enc) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)kv.dim, cuuint64_t(1) << kv.page_log, (cuuint64_t)kv.heads, (cuuint64_t)kv.pages};
  // the stride of a single head or page is not used, but has to be a valid one
  const cuuint64_t strides[3] = {(cuuint64_t)kv.token_stride * 2, (cuuint64_t)std::max<int64_t>(kv.head_stride, 8) * 2,
                                 (cuuint64_t)std::max<int64_t>(kv.page_stride, 8) * 2};
  const cuuint32_t box[4] = {64, tokens, 1, 1}, ones[4] = {1, 1, 1, 1};
  return enc(map, dtype == 0 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, pages, dims, strides,
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
  if (!encode(&maps.k, kv, dtype, kv.k, box) || !encode(&maps.v, kv, dtype, kv.v, box) ||
      !encode(&maps.v_row, kv, dtype, kv.v, 1))
    return cudaErrorInvalidValue;
  k_kv_prompt<T, DP><<<(unsigned)(sp.units * sp.parts), kThreads, Smem<DP>::kLaunch, st>>>(maps, kv, bt, q, sp.units,
                                                                                           sp.parts, scratch);
  *launches += 1;
  if (sp.parts > 1) {
    k_kv_prompt_join<T, DP><<<dim3((unsigned)sp.units, kBlockRows / 32), 256, 0, st>>>(kv, bt, q, sp.parts, scratch);
    *launches += 1;
  }
  return cudaGetLastError();
}

}  // namespace

uint64_t PromptSplit::scratch_floats() const {
  return parts > 1 ? (uint64_t)units * parts * kBlockRows * (dim_padded + 2) : 0;
}

PromptSplit plan_prompt(const View& kv, const Batch& bt, const Query& q, int sms) {
  PromptSplit sp;
  sp.dim_padded = kv.dim <= 64 ? 64 : 128;
  // at most ceil(rows / 256) units per sequence and key head
  sp.units = ((int64_t)q.tokens * q.group / kBlockRows + bt.seqs) * kv.heads;
  int64_t keys = (int64_t)bt.width << kv.page_log;
  if (q.window) keys = std::min<int64_t>(keys, (int64_t)q.window + q.sinks + 2 * kTileKeys + kBlockRows);
  const int64_t most = std::min<int64_t>(kMaxParts, keys / (kPartTiles * kTileKeys));
  sp.parts = (int32_t)std::max<int64_t>(1, std::min<int64_t>(most, 3 * sms / std::max<int64_t>(1, sp.units)));
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
