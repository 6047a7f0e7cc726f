// Entry points of the attention over the paged cache: argument checks and the choice of kernel.
#include "kv_attention.h"

#include <algorithm>
#include <atomic>
#include <optional>

#include "kv_host.h"

namespace bfvgpu {
namespace kv {
namespace {

constexpr uint64_t kMost = 0x7ffffffe;

// Streaming multiprocessors of a device; the default of this GPU where there is none to ask.
int sm_count(int device) {
  constexpr int kDefault = 148, kDevices = 64;
  static std::atomic<int> known[kDevices];
  if (device < 0 || device >= kDevices) return kDefault;
  int n = known[device].load();
  if (!n) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || n < 1) return kDefault;
    known[device].store(n);
  }
  return n;
}

// Single tokens go to the row kernel, which reads a sequence's keys once per 16 query rows.  Prompts go there
// * where 16-row blocks x (keys + 200) x dims are few, that is, where the start of the prompt kernel counts more than
//   what its tiles save (at 512 keys of 128 dims and 8 key heads, 32, 64 and 128 rows: 9, 10 and 13 us against 13, 13
//   and 13; 4 sequences of 198 tokens with a window of 14, 4 key heads of 8 query heads: 42 us against 12), and
// * up to 16 rows per sequence and key head on average with up to 64 dims, where its blocks stream the keys (64
//   sequences of 5384 tokens, 16 rows: 98 us against 133), and up to 4 with more, where they multiply for longer
//   (128 sequences of 3469 tokens, 32 rows: 350 us against 171; 100 of 7585, 16 rows: 208 against 164).
// Over 130 prompts of 1 to 128 sequences, 2 to 1000 tokens and up to 16384 keys the choice cost 0.8 % of the time on
// average, always the prompt kernel 13 %, always the row kernel 43 %.
constexpr int64_t kFewRows = 16, kFewRowsWide = 4;
constexpr double kFewProducts = 8e6;
constexpr int64_t kStartKeys = 200;
bool few_rows(const View& kv, const Batch& bt, const Query& q, bool ragged) {
  const bool wide = kv.dim > 64;
  if (!ragged || (int64_t)q.tokens * q.group <= (wide ? kFewRowsWide : kFewRows) * bt.seqs) return true;
  int64_t keys = (int64_t)bt.width << kv.page_log;
  if (q.window) keys = std::min<int64_t>(keys, (int64_t)q.window + q.sinks);
  const int64_t blocks = ((int64_t)q.tokens * q.group / 16 + bt.seqs) * kv.heads;
  return (double)blocks * (double)(keys + kStartKeys) * (wide ? 128 : 64) <= kFewProducts;
}

// The kernel of a call: few rows, or queries whose strides the prompt kernel's loads cannot follow.
bool takes_rows(const View& kv, const Batch& bt, const Query& q, bool ragged) {
  return few_rows(kv, bt, q, ragged) || !prompt_strides(q);
}

struct Call {
  View view;
  Batch batch;
  Query query;
};

Call checked_call(const bfvgpu_kv* cache, int32_t layer, int64_t token_stride, int64_t head_stride, uint64_t q_heads,
                  uint64_t tokens, uint64_t seqs, uint64_t width, int32_t window, int32_t sinks) {
  Call c;
  need(layer >= 0, BFVGPU_E_SHAPE, "E_KV_LAYER");
  c.view = checked_view(cache, layer);
  need(q_heads >= 1 && q_heads <= kMost && q_heads % c.view.heads == 0, BFVGPU_E_SHAPE, "E_KV_HEADS");
  need(tokens <= kMost && seqs <= kMost && width <= kMost, BFVGPU_E_SHAPE, "E_KV_SHAPE");
  need(q_heads / c.view.heads <= kMaxGroup && tokens * (q_heads / c.view.heads) <= kMost, BFVGPU_E_SHAPE, "E_KV_SHAPE");
  // positions and their sums with the window stay in 32 bits
  need((width << c.view.page_log) <= (uint64_t(1) << 30), BFVGPU_E_SHAPE, "E_KV_WIDTH");
  need(window >= 0 && sinks >= 0, BFVGPU_E_ARGUMENT, "E_KV_WINDOW");
  const int32_t top = 1 << 30;
  c.query.group = (int32_t)(q_heads / c.view.heads);
  c.query.group_inverse = ((1u << kGroupShift) + c.query.group - 1) / c.query.group;
  c.query.tokens = (int32_t)tokens;
  // an axis of one element has no stride
  c.query.token_stride = tokens > 1 ? token_stride : c.view.dim;
  c.query.head_stride = q_heads > 1 ? head_stride : c.view.dim;
  c.query.window = window < top ? window : 0;  // a window past every position hides nothing
  c.query.sinks = std::min(sinks, top);
  c.batch.seqs = (int32_t)seqs;
  c.batch.width = (int32_t)width;
  return c;
}

void attend(bfvgpu_ctx* ctx, const bfvgpu_kv* cache, Call& c, const void* q, const int32_t* starts, const int32_t* table,
            const int32_t* lengths, float scale, uint64_t* scratch, void* out, void* stream) {
  const float scale_log2 = scale * 1.4426950408889634f;
  need(std::isfinite(scale_log2) && scale > 0, BFVGPU_E_ARGUMENT, "E_KV_SCALE");
  const Place at = checked_place(ctx, stream);
  if (!c.query.tokens) return;
  need(c.batch.seqs && q && table && c.batch.width && lengths && out, BFVGPU_E_ARGUMENT, "E_KV_ARGUMENT");
  need(aligned16(q) && aligned16(out) && c.query.token_stride % 8 == 0 && c.query.head_stride % 8 == 0, BFVGPU_E_ARGUMENT,
       "E_KV_ALIGNMENT");
  OnDevice scope(at.device);
  c.batch.table = table;
  c.batch.lengths = lengths;
  c.batch.starts = starts;
  c.batch.err = at.err;
  c.query.q = static_cast<const uint16_t*>(q);
  c.query.out = static_cast<uint16_t*>(out);
  c.query.scale_log2 = scale_log2;
  float* work = reinterpret_cast<float*>(scratch);
  auto need_scratch = [&](uint64_t floats) {
    need(floats == 0 || scratch, BFVGPU_E_ARGUMENT, "E_KV_SCRATCH");
    need(aligned16(scratch), BFVGPU_E_ARGUMENT, "E_KV_ALIGNMENT");
  };
  int launches = 0;
  if (takes_rows(c.view, c.batch, c.query, starts)) {
    const RowSplit sp = plan_rows(c.view, c.batch, c.query, at.device);
    need_scratch(sp.scratch_floats());
    need(sp.blocks16 * sp.parts <= (int64_t)(kMost / sp.cluster), BFVGPU_E_SHAPE, "E_KV_SHAPE");
    cuda_need(launch_rows(c.view, c.batch, c.query, cache->dtype, sp, work, at.stream, &launches), "kv attention");
  } else {
    const PromptSplit sp = plan_prompt(c.view, c.batch, c.query, sm_count(at.device));
    need_scratch(sp.scratch_floats());
    need(sp.units * sp.parts <= (int64_t)kMost, BFVGPU_E_SHAPE, "E_KV_SHAPE");
    cuda_need(launch_prompt(c.view, c.batch, c.query, cache->dtype, sp, work, at.stream, &launches), "kv attention");
  }
  internal_count_launch(launches);
}

// Words of scratch; 0 for arguments that the call itself refuses.
uint64_t scratch_words(const bfvgpu_ctx* ctx, const bfvgpu_kv* cache, uint64_t q_heads, uint64_t tokens, bool ragged,
                       uint64_t seqs, uint64_t width, int32_t window, int32_t sinks) {
  uint64_t words = 0;
  guarded([&] {
    Call c = checked_call(cache, 0, 0, 0, q_heads, tokens, seqs, width, window, sinks);
    static const int32_t some = 0;
    if (ragged) c.batch.starts = &some;  // only asked whether there is one
    int device = -1;
    internal_params(ctx, &device, nullptr);
    std::optional<OnDevice> scope;
    if (device >= 0) scope.emplace(device);
    // the row kernel's too where the strides of the queries, not known here, may send them there
    uint64_t floats = plan_rows(c.view, c.batch, c.query, device).scratch_floats();
    if (!few_rows(c.view, c.batch, c.query, ragged))
      floats = std::max(floats, plan_prompt(c.view, c.batch, c.query, sm_count(device)).scratch_floats());
    words = (floats + 1) / 2;
  });
  return words;
}

}  // namespace
}  // namespace kv
}  // namespace bfvgpu

using namespace bfvgpu;
using namespace bfvgpu::kv;

extern "C" uint64_t bfvgpu_kv_decode_scratch_words(const bfvgpu_ctx* ctx, const bfvgpu_kv* cache, uint64_t q_heads,
                                                   uint64_t seqs, uint64_t width, int32_t window, int32_t sinks) {
  return scratch_words(ctx, cache, q_heads, seqs, false, seqs, width, window, sinks);
}

extern "C" int32_t bfvgpu_kv_decode_device(bfvgpu_ctx* ctx, const bfvgpu_kv* cache, int32_t layer, const void* q,
                                           int64_t token_stride, int64_t head_stride, uint64_t q_heads,
                                           const int32_t* table, uint64_t width, const int32_t* lengths, uint64_t seqs,
                                           int32_t window, int32_t sinks, float scale, uint64_t* scratch, void* out,
                                           void* stream) {
  return guarded([&] {
    Call c = checked_call(cache, layer, token_stride, head_stride, q_heads, seqs, seqs, width, window, sinks);
    attend(ctx, cache, c, q, nullptr, table, lengths, scale, scratch, out, stream);
  });
}

extern "C" uint64_t bfvgpu_kv_prompt_scratch_words(const bfvgpu_ctx* ctx, const bfvgpu_kv* cache, uint64_t q_heads,
                                                   uint64_t tokens, uint64_t seqs, uint64_t width, int32_t window,
                                                   int32_t sinks) {
  return scratch_words(ctx, cache, q_heads, tokens, true, seqs, width, window, sinks);
}

extern "C" int32_t bfvgpu_kv_prompt_device(bfvgpu_ctx* ctx, const bfvgpu_kv* cache, int32_t layer, const void* q,
                                           int64_t token_stride, int64_t head_stride, uint64_t q_heads,
                                           uint64_t tokens, const int32_t* starts, const int32_t* table,
                                           uint64_t width, const int32_t* lengths, uint64_t seqs, int32_t window,
                                           int32_t sinks, float scale, uint64_t* scratch, void* out, void* stream) {
  return guarded([&] {
    need(starts || !tokens, BFVGPU_E_ARGUMENT, "E_KV_ARGUMENT");
    Call c = checked_call(cache, layer, token_stride, head_stride, q_heads, tokens, seqs, width, window, sinks);
    attend(ctx, cache, c, q, starts, table, lengths, scale, scratch, out, stream);
  });
}

extern "C" int32_t bfvgpu_kv_prompt_kernel(const bfvgpu_kv* cache, int64_t token_stride, int64_t head_stride,
                                           uint64_t q_heads, uint64_t tokens, uint64_t seqs, uint64_t width, int32_t window,
                                           int32_t sinks) {
  int32_t kernel = -1;
  guarded([&] {
    const Call c = checked_call(cache, 0, token_stride, head_stride, q_heads, tokens, seqs, width, window, sinks);
    kernel = takes_rows(c.view, c.batch, c.query, true) ? BFVGPU_KV_ROWS : BFVGPU_KV_TILES;
  });
  return kernel;
}
