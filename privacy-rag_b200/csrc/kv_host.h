// Host side of the paged key-value cache's entry points: argument checks, errors, device scope.
#pragma once
#include <cuda_runtime.h>

#include <cmath>
#include <exception>
#include <new>
#include <string>

#include "bfvgpu.h"
#include "ctx_internal.h"
#include "kv_common.cuh"

namespace bfvgpu {
namespace kv {

struct Refusal {
  int32_t code;
  std::string what;
};
[[noreturn]] inline void refuse(int32_t code, const char* what) { throw Refusal{code, what}; }
inline void need(bool ok, int32_t code, const char* what) {
  if (!ok) refuse(code, what);
}

// No C++ exception crosses the ABI.
template <class F>
int32_t guarded(F&& f) {
  try {
    f();
    return BFVGPU_OK;
  } catch (const Refusal& r) {
    try {
      internal_set_error(r.what);
    } catch (const std::exception&) {
    }
    return r.code;
  } catch (const std::bad_alloc&) {
    return BFVGPU_E_ALLOC;
  } catch (const std::exception&) {
    return BFVGPU_E_ARGUMENT;
  }
}

inline void cuda_need(cudaError_t e, const char* where) {
  if (e != cudaSuccess) throw Refusal{BFVGPU_E_CUDA, std::string("E_BFVGPU_CUDA: ") + where + ": " + cudaGetErrorString(e)};
}

class OnDevice {
 public:
  explicit OnDevice(int device) {
    if (cudaGetDevice(&previous_) != cudaSuccess) previous_ = -1;
    if (previous_ != device) {
      cuda_need(cudaSetDevice(device), "cudaSetDevice");
      changed_ = true;
    }
  }
  ~OnDevice() {
    if (changed_ && previous_ >= 0) cudaSetDevice(previous_);
  }
  OnDevice(const OnDevice&) = delete;
  OnDevice& operator=(const OnDevice&) = delete;

 private:
  int previous_ = -1;
  bool changed_ = false;
};

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// The cache's own description; layer < 0: all layers (the view is layer 0's).
inline View checked_view(const bfvgpu_kv* c, int32_t layer) {
  need(c && c->k && c->v, BFVGPU_E_ARGUMENT, "E_KV_ARGUMENT");
  need(c->dtype == BFVGPU_KV_BF16 || c->dtype == BFVGPU_KV_FP16, BFVGPU_E_ARGUMENT, "E_KV_DTYPE");
  need(c->layers >= 1 && c->pages >= 1 && c->heads >= 1 && c->heads <= 1024, BFVGPU_E_SHAPE, "E_KV_SHAPE");
  need(c->dim >= 8 && c->dim <= 128 && c->dim % 8 == 0, BFVGPU_E_SHAPE, "E_KV_DIM");
  need(c->page_tokens >= 16 && c->page_tokens <= 256 && !(c->page_tokens & (c->page_tokens - 1)), BFVGPU_E_SHAPE,
       "E_KV_PAGE_TOKENS");
  need(layer < c->layers, BFVGPU_E_SHAPE, "E_KV_LAYER");
  const int64_t strides[4] = {c->token_stride, c->head_stride, c->page_stride, c->layer_stride};
  const int32_t sizes[4] = {c->page_tokens, c->heads, c->pages, c->layers};
  for (int i = 0; i < 4; ++i) {
    if (sizes[i] == 1) continue;  // the stride of a single element is never used
    need(strides[i] >= c->dim && strides[i] < (int64_t(1) << 38), BFVGPU_E_SHAPE, "E_KV_STRIDE");
    need(strides[i] % 8 == 0, BFVGPU_E_ARGUMENT, "E_KV_ALIGNMENT");
  }
  need(aligned16(c->k) && aligned16(c->v), BFVGPU_E_ARGUMENT, "E_KV_ALIGNMENT");
  View w;
  const int64_t at = layer > 0 ? layer * c->layer_stride : 0;
  w.k = static_cast<uint16_t*>(c->k) + at;
  w.v = static_cast<uint16_t*>(c->v) + at;
  w.page_stride = c->pages > 1 ? c->page_stride : 0;
  w.head_stride = c->heads > 1 ? c->head_stride : 0;
  w.token_stride = c->token_stride;
  w.pages = c->pages;
  w.heads = c->heads;
  w.dim = c->dim;
  while ((1 << w.page_log) < c->page_tokens) ++w.page_log;
  return w;
}

struct Place {
  int device = -1;
  cudaStream_t stream = nullptr;
  uint32_t* err = nullptr;
  int reserved_sms = 0;
};

// After the arguments: the context's device and the call's stream.
inline Place checked_place(const bfvgpu_ctx* ctx, void* stream) {
  Place p;
  const DevParams* P = internal_params(ctx, &p.device, &p.stream);
  need(P != nullptr, BFVGPU_E_ARGUMENT, "E_BFVGPU_ARGUMENT");
  need(p.device >= 0, BFVGPU_E_DEVICE, "E_BFVGPU_HOST_ONLY_CONTEXT");
  if (stream) p.stream = static_cast<cudaStream_t>(stream);
  p.err = P->err;
  p.reserved_sms = P->reserved_sms;
  return p;
}

}  // namespace kv
}  // namespace bfvgpu
