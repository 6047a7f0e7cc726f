// Attention of prompts over the paged cache on the 5th-generation tensor cores.
//
// Rows of one (sequence, key head) are packed token by token, the query heads of the group side by
// side, so that a block's 256 rows (two tiles of 128) share every key it loads.  Per tile of 128 keys:
//   S = Q K^T            tcgen05.mma 128 x 128 x dim, Q and K from shared memory, S in tensor memory
//   P = 2^(c S - m)      one thread per row, the row's 128 scores in registers; P in 16 bits over S
//   O += P V             tcgen05.mma 128 x dim x 128, P from tensor memory, V from shared memory
// m is the row's reference exponent.  It starts as the running maximum and follows it only when the
// maximum has grown by more than 8: until then weights of up to 2^8 stay far inside both 16-bit types
// and the 32-bit sums, and O need not be rescaled.  The sum of the weights is kept in 32 bits, from
// the weights before they are rounded to 16 bits for the product.
//
// Roles: warps 0-3 and 4-7 hold the rows of tile 0 and 1, one thread of warp 8 issues the products,
// warp 9 the loads.  While one tile's rows are in their exponentials, the other tile's products run.
// K and V arrive by TMA page by page as the table names them, in the 128-byte swizzle (K as K-major,
// V as MN-major operand).  Only visible tokens of V are loaded: what no row of the block sees may
// hold NaN (unwritten rest of a page, pages given up), and 0 x NaN would reach every row.  Such
// pages are read row by row, the other rows filled with zeros.
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
constexpr int kThreads = 384;         // two warpgroups of rows, one of the issuing warps (two of its warps idle)
constexpr int kMmaWarp = 8, kLoadWarp = 9;
// Registers a thread: launched with 168 (384 x 168 of the SM's 65536); the issuing warpgroup keeps 64 and
// the rows take 216: 128 x 64 + 256 x 216 <= 384 x 168.
constexpr int kIssueRegs = 64, kRowRegs = 216;
constexpr float kLag = 8.f;           // how far m may stay behind the running maximum
constexpr uint32_t kPolls = 1u << 22; // of a wait before it gives up

template <int DP>
struct Smem {
  static constexpr int kHalves = DP / 64;                 // 64 dims = one 128-byte swizzled row
  static constexpr int kHalfBytes = kTileKeys * 128;
  static constexpr int kTileBytes = kHalves * kHalfBytes; // Q, K or V tile
  static constexpr int kStages = DP == 128 ? 2 : 4;
  static constexpr int kQ = 0;
  static constexpr int kK = kQ + 2 * kTileBytes;
  static constexpr int kV = kK + kStages * kTileBytes;
  static constexpr int kBar = kV + kStages * kTileBytes;
  // barriers: Q of tile 0/1; K full, K empty, V full, V empty per stage; S, P, O of tile 0/1; drain
  static constexpr int kBars = 2 + 4 * kStages + 6 + 1;
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
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile uint32_t* abort, uint32_t* err) {
  for (uint32_t i = 0; i < kPolls; ++i) {
    if (bar_try(bar, parity)) return true;
    if ((i & 1023) == 1023 && *abort) return false;
  }
  *abort = 1;
  flag_error(err, kErrWait);
  return false;
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
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Shared-memory operand descriptor, 128-byte swizzle: start address, leading and stride byte offset in
// 16-byte units, version 1, layout 2.  K-major: rows of 128 bytes, 8-row groups `stride` apart (1024).
// MN-major: chunks of 64 MN elements `leading` apart, groups of 8 K rows `stride` apart (1024).
__device__ __forceinline__ uint64_t operand(uint32_t at, uint32_t leading) {
  return (uint64_t)((at >> 4) & 0x3fff) | ((uint64_t)(leading >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
// Instruction descriptor, kind::f16: D 32-bit float, A and B of type T, A K-major, B K-major or
// MN-major, M = 128.
template <class T>
constexpr uint32_t instruction(int n, bool b_mn) {
  const uint32_t type = T::kind == 0 ? 1 : 0;
  return (1u << 4) | (type << 7) | (type << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add) : "memory");
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

// ---- which key tiles the block and each of its row tiles need ------------------------------------
// The block's key tiles are numbered 0 .. n-1: `first` tiles of first tokens, then the window's from tile
// `from` on.  A row tile needs [0, first) and [begin, end).  It may take part in a tile that it sees
// nothing of; every tile is needed by one row tile.
struct Span {
  int32_t lo = 0, hi = -1;        // positions of the rows (hi < 0: no row sees a key)
  int32_t begin = 0, end = 0;
};
struct Plan {
  int32_t n = 0, first = 0, from = 0;
  int32_t end = 0;                // keys the block sees: [0, sinks) and [begin, end)
  __device__ __forceinline__ int32_t key0(int32_t i) const { return (i < first ? i : i - first + from) * kTileKeys; }
  // the row tile's first key tile from i on; n: none
  __device__ __forceinline__ int32_t at_or_after(const Span& s, int32_t i) const {
    i = i < first ? i : max(i, s.begin);
    return i < s.end ? i : n;
  }
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
__device__ __forceinline__ Span make_span(const Unit& un, const Query& q, const Plan& p, int t) {
  Span s;
  if (t * kTileRows >= un.rows) return s;
  s.lo = un.position(q, t * kTileRows);
  s.hi = un.position(q, min(un.rows, (t + 1) * kTileRows) - 1);
  if (s.hi < 0) return s;
  s.end = p.first + s.hi / kTileKeys - p.from + 1;
  s.begin = p.first;
  // the block's window tiles before the row tile's own, unless first tokens reach into them
  if (un.begin > 0 && un.sinks <= p.from * kTileKeys) s.begin += max(0, (s.lo + 1 - q.window) / kTileKeys - p.from);
  return s;
}

template <class T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
    k_kv_prompt(const __grid_constant__ Maps maps, View kv, Batch bt, Query q, int64_t units) {
  using S = Smem<DP>;
  extern __shared__ uint8_t raw[];
  const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
  uint8_t* sm = raw + (base - smem_addr(raw));
  const int warp = same(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const uint32_t bars = base + S::kBar;
  const uint32_t q_full = bars, k_full = bars + 16, k_empty = k_full + 8 * S::kStages, v_full = k_empty + 8 * S::kStages,
                 v_empty = v_full + 8 * S::kStages, s_full = v_empty + 8 * S::kStages, p_full = s_full + 16,
                 o_full = p_full + 16, drain = o_full + 16;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + S::kBar + S::kBars * 8);
  volatile uint32_t* abort = tmem_slot + 1;

  if (threadIdx.x == 0) {
    bar_init(q_full, kTileRows);
    bar_init(q_full + 8, kTileRows);
    for (int i = 0; i < 4 * S::kStages; ++i) bar_init(k_full + 8 * i, 1);
    for (int t = 0; t < 2; ++t) {
      bar_init(s_full + 8 * t, 1);
      bar_init(p_full + 8 * t, kTileRows);
      bar_init(o_full + 8 * t, 1);
    }
    bar_init(drain, 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(tmem_slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  // the blocks with the most keys first
  const Unit un = find_unit<kBlockRows>(kv, bt, q, units - 1 - blockIdx.x);
  const Plan plan = make_plan(un);

  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;
  // tensor memory columns: S (and P over it) of tile 0 and 1, O of tile 0 and 1
  auto s_col = [&](int t) { return tmem + t * kTileKeys; };
  auto o_col = [&](int t) { return tmem + 2 * kTileKeys + t * DP; };

  if (warp >= kMmaWarp) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
  if (warp == kLoadWarp) {
    // ---- loads: lane j has the j-th page of a key tile ----
    const int32_t page_tokens = 1 << kv.page_log, box = min(page_tokens, kTileKeys), boxes = kTileKeys / box;
    const int32_t* row = bt.table + (int64_t)un.b * bt.width;
    bool ok = true;
    int32_t i = 0;
    for (; i < plan.n; ++i) {
      const int st = i % S::kStages;
      const uint32_t turn = (i / S::kStages) & 1;
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
      ok = bar_wait(k_empty + 8 * st, turn ^ 1, abort, bt.err);
      if (!__all_sync(0xffffffffu, ok)) break;
      if (lane == 0) bar_expect(k_full + 8 * st, S::kTileBytes);
      __syncwarp();
      if (lane < boxes)
#pragma unroll
        for (int h = 0; h < S::kHalves; ++h)
          tma_box(kb + h * S::kHalfBytes + lane * box * 128, &maps.k, h * 64, at, un.g, page, k_full + 8 * st);
      ok = bar_wait(v_empty + 8 * st, turn ^ 1, abort, bt.err);
      if (!__all_sync(0xffffffffu, ok)) break;
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
    }
    if (i < plan.n) {
      // given up: what is in flight into shared memory lands before the block ends
      for (int32_t j = max(0, i - S::kStages); j <= i; ++j) {
        if (j < plan.n)
          for (uint32_t n = 0; n < kPolls && !bar_try(k_full + 8 * (j % S::kStages), (j / S::kStages) & 1); ++n) {
            if (j == i && n > 1024) break;  // perhaps never issued
          }
        if (j < i)
          for (uint32_t n = 0; n < kPolls && !bar_try(v_full + 8 * (j % S::kStages), (j / S::kStages) & 1); ++n) {
          }
      }
    }
  } else if (warp == kMmaWarp) {
    // ---- products: S of a tile as soon as its P is used up, so that the two tiles take turns.  The
    // whole warp runs the loop and one thread issues: descriptors in uniform registers go to the
    // tensor core at once (from inside a one-thread branch each product took about 100 cycles to issue) ----
    Plan pl = plan;
    pl.n = same(pl.n);
    pl.first = same(pl.first);
    Span s0 = make_span(un, q, plan, 0), s1 = make_span(un, q, plan, 1);
    s0.begin = same(s0.begin);
    s0.end = same(s0.end);
    s1.begin = same(s1.begin);
    s1.end = same(s1.end);
    const uint32_t tm = same(tmem);
    bool ok = true;
    // next key tile of each row tile's S, and of its P; key tiles whose K is given back
    int32_t s_next[2] = {pl.at_or_after(s0, 0), pl.at_or_after(s1, 0)};
    int32_t p_next[2] = {s_next[0], s_next[1]}, released = 0;
    uint32_t p_turn[2] = {0, 0};
    const uint64_t q_desc = operand(base + S::kQ, 16), k_desc = operand(base + S::kK, 16),
                   v_desc = operand(base + S::kV, S::kHalfBytes);
    auto wait = [&](uint32_t bar, uint32_t parity) {
      ok = ok && __all_sync(0xffffffffu, bar_wait(bar, parity, abort, bt.err));
    };
    auto issue_s = [&](auto tile) {
      constexpr int t = decltype(tile)::value;
      const int32_t i = s_next[t];
      if (i >= pl.n) return;
      const int st = i % S::kStages;
      wait(k_full + 8 * st, (i / S::kStages) & 1);
      if (!ok) return;
      s_next[t] = pl.at_or_after(t ? s1 : s0, i + 1);
      const int32_t free = min(s_next[0], s_next[1]);
      fence_after();
      const uint64_t qd = q_desc + t * (S::kTileBytes >> 4), kd = k_desc + st * (S::kTileBytes >> 4);
      if (elected()) {
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
          constexpr uint32_t kHalf = S::kHalfBytes >> 4;
          const uint32_t off = (ks >> 2) * kHalf + (ks & 3) * 2;
          mma_ss(tm + t * kTileKeys, qd + off, kd + off, instruction<T>(kTileKeys, false), ks > 0);
        }
        mma_commit(s_full + 8 * t);
        for (int32_t r = released; r < free; ++r) mma_commit(k_empty + 8 * (r % S::kStages));
      }
      __syncwarp();
      released = max(released, free);
    };
    auto issue_o = [&](auto tile, int32_t i) {
      constexpr int t = decltype(tile)::value;
      if (!ok || p_next[t] != i) return;
      const int st = i % S::kStages;
      wait(v_full + 8 * st, (i / S::kStages) & 1);
      wait(p_full + 8 * t, p_turn[t] & 1);
      if (!ok) return;
      p_next[t] = pl.at_or_after(t ? s1 : s0, i + 1);
      fence_after();
      const uint64_t vd = v_desc + st * (S::kTileBytes >> 4);
      if (elected()) {
#pragma unroll
        for (int ks = 0; ks < kTileKeys / 16; ++ks)
          mma_ts(tm + 2 * kTileKeys + t * DP, tm + t * kTileKeys + ks * 8, vd + ks * 128, instruction<T>(DP, true),
                 ks > 0 || p_turn[t] > 0);
        if (p_next[t] >= pl.n) mma_commit(o_full + 8 * t);
      }
      __syncwarp();
      ++p_turn[t];
      issue_s(tile);
    };
    const std::integral_constant<int, 0> tile0;
    const std::integral_constant<int, 1> tile1;
    if (s0.end) wait(q_full, 0);
    issue_s(tile0);
    if (s1.end) wait(q_full + 8, 0);
    issue_s(tile1);
    for (int32_t i = 0; i < pl.n && ok; ++i) {
      issue_o(tile0, i);
      issue_o(tile1, i);
      if (ok && elected()) mma_commit(v_empty + 8 * (i % S::kStages));
      __syncwarp();
    }
    if (!ok) {  // products in flight end before the tensor memory is given back
      if (elected()) mma_commit(drain);
      for (uint32_t n = 0; n < kPolls && !bar_try(drain, 0); ++n) {
      }
      __syncwarp();
    }
  } else if (warp < kMmaWarp) {
    // ---- rows ----
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRowRegs));
    const int t = warp >> 2;
    if (t * kTileRows < un.rows) {
      const int tid = threadIdx.x & 127, row = tid;
      uint8_t* qs = sm + S::kQ + t * S::kTileBytes;
      constexpr int kChunks = DP / 8;
      constexpr int kLoads = kTileRows * kChunks / 128, kStep = 128 / kChunks;
      {
        const int chunk = tid % kChunks, r0 = tid / kChunks;
        uint4 x[kLoads];  // all in flight together
#pragma unroll
        for (int n = 0; n < kLoads; ++n) {
          const int r = r0 + n * kStep;
          x[n] = make_uint4(0, 0, 0, 0);
          if (t * kTileRows + r < un.rows && chunk * 8 < kv.dim)
            x[n] = __ldg(reinterpret_cast<const uint4*>(un.query(q, t * kTileRows + r) + chunk * 8));
        }
#pragma unroll
        for (int n = 0; n < kLoads; ++n) {
          const int r = r0 + n * kStep;
          *reinterpret_cast<uint4*>(qs + (chunk >> 3) * S::kHalfBytes + r * 128 + (((chunk & 7) ^ (r & 7)) << 4)) = x[n];
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      bar_arrive(q_full + 8 * t);

      const Span span = make_span(un, q, plan, t);
      const int32_t last_row = min(un.rows, (t + 1) * kTileRows) - 1;
      const int32_t my_row = min(t * kTileRows + row, last_row);  // rows past the last do its work again
      const int32_t pos = un.position(q, my_row);
      const uint32_t quadrant = (uint32_t)(warp & 3) << 21;  // lanes 32 (warp % 4) ..
      const uint32_t s_at = s_col(t) + quadrant, o_at = o_col(t) + quadrant;
      const float c = q.scale_log2;
      float m = -INFINITY, l = 0;
      int32_t done = 0;
      bool ok = true;
      for (int32_t i = plan.at_or_after(span, 0); i < plan.n; i = plan.at_or_after(span, i + 1)) {
        const int32_t key0 = plan.key0(i);
        ok = bar_wait(s_full + 8 * t, done & 1, abort, bt.err);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        fence_after();
        float x[kTileKeys];
#pragma unroll
        for (int j = 0; j < kTileKeys; j += 32) tmem_load(s_at + j, x + j);
        tmem_load_wait();
        const bool cut_end = key0 + kTileKeys - 1 > span.lo;
        const bool cut_begin = q.window && key0 <= span.hi - q.window && key0 + kTileKeys > q.sinks;
        if (cut_begin) {
          // keys lo .. hi of the tile are seen, and those below sk
          const int32_t hi = pos - key0, sk = q.sinks - key0;
          const uint32_t lo = (uint32_t)max(hi - q.window + 1, 0), n = (uint32_t)max(hi - (int32_t)lo + 1, 0);
          if (sk > 0) {
#pragma unroll
            for (int j = 0; j < kTileKeys; ++j)
              if ((uint32_t)j - lo >= n && (j >= sk || j > hi)) x[j] = -INFINITY;
          } else {
#pragma unroll
            for (int j = 0; j < kTileKeys; ++j)
              if ((uint32_t)j - lo >= n) x[j] = -INFINITY;
          }
        } else if (cut_end) {
          const int32_t hi = pos - key0;
#pragma unroll
          for (int j = 0; j < kTileKeys; ++j)
            if (j > hi) x[j] = -INFINITY;
        }
        float top[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int j = 4; j + 8 <= kTileKeys + 4; j += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            top[e] = fmaxf(fmaxf(top[e], x[j + e]), j + 4 + e < kTileKeys ? x[j + 4 + e] : -INFINITY);
        const float now = fmaxf(m, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * c);
        if (done == 0) {
          m = now;
        } else if (__any_sync(0xffffffffu, now > m + kLag)) {
          // O is at rest: the scores just read were issued after the last product into it
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
        float sum[4] = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < kTileKeys; j += 32) {
          uint32_t p[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float p0 = exp2_fast(fmaf(x[j + e], c, -ref)), p1 = exp2_fast(fmaf(x[j + e + 1], c, -ref));
            sum[e & 2] += p0;
            sum[(e & 2) + 1] += p1;
            p[e / 2] = T::pack(p0, p1);
          }
          tmem_store16(s_at + j / 2, p);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        tmem_store_wait();
        fence_before();
        bar_arrive(p_full + 8 * t);
        ++done;
      }
      // ---- results: through the tile's Q in shared memory, for whole rows ----
      if (ok && done) ok = bar_wait(o_full + 8 * t, 0, abort, bt.err);
      ok = __all_sync(0xffffffffu, ok);
      if (ok && !done) {  // no row of the tile sees a key
        for (int r = tid / kChunks; r < kTileRows && t * kTileRows + r < un.rows; r += kStep)
          if (tid % kChunks * 8 < kv.dim)
            *reinterpret_cast<uint4*>(un.result(kv, q, t * kTileRows + r) + tid % kChunks * 8) = make_uint4(0, 0, 0, 0);
      } else if (ok) {
        fence_after();
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int j = 0; j < DP; j += 32) {
          float o[32];
          tmem_load(o_at + j, o);
          tmem_load_wait();
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            uint32_t w[4];
#pragma unroll
            for (int h = 0; h < 4; ++h) w[h] = l == 0.f ? 0 : T::pack(o[e + 2 * h] * inv, o[e + 2 * h + 1] * inv);
            const int chunk = (j + e) / 8;
            *reinterpret_cast<uint4*>(qs + row * DP * 2 + ((chunk ^ (row & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        __syncwarp();  // a warp writes out its own 32 rows
        const int chunk = lane % kChunks;
#pragma unroll
        for (int n = 0; n < kChunks; ++n) {
          const int rr = (warp & 3) * 32 + lane / kChunks + n * (32 / kChunks);
          if (t * kTileRows + rr < un.rows && chunk * 8 < kv.dim)
            *reinterpret_cast<uint4*>(un.result(kv, q, t * kTileRows + rr) + chunk * 8) =
                *reinterpret_cast<const uint4*>(qs + rr * DP * 2 + ((chunk ^ (rr & 7)) << 4));
        }
      }
    }
  }
  fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
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
cudaError_t launch(const View& kv, const Batch& bt, const Query& q, int dtype, cudaStream_t st) {
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
  const int64_t units = prompt_units(kv, bt, q);
  k_kv_prompt<T, DP><<<(unsigned)units, kThreads, Smem<DP>::kLaunch, st>>>(maps, kv, bt, q, units);
  return cudaGetLastError();
}

}  // namespace

int64_t prompt_units(const View& kv, const Batch& bt, const Query& q) {
  return ((int64_t)q.tokens * q.group / kBlockRows + bt.seqs) * kv.heads;
}

cudaError_t launch_prompt(const View& kv, const Batch& bt, const Query& q, int dtype, cudaStream_t st) {
  const bool small = kv.dim <= 64;
  if (dtype == 0) return small ? launch<Bf16, 64>(kv, bt, q, dtype, st) : launch<Bf16, 128>(kv, bt, q, dtype, st);
  return small ? launch<Fp16, 64>(kv, bt, q, dtype, st) : launch<Fp16, 128>(kv, bt, q, dtype, st);
}

}  // namespace kv
}  // namespace bfvgpu
