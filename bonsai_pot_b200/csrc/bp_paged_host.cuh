// What the host sides of the paged operators share: errors, the checks of arguments, the context's device for the length of a call.
#pragma once

#include <stdio.h>

#include "../../include/bonsai_pages.h"
#include "bp_paged.cuh"

namespace bp {
namespace paged {

inline int fail(bp_paged_ctx* c, int status, const char* msg) {
  if (c) snprintf(c->msg, sizeof c->msg, "%s", msg);
  return status;
}

inline int fail_config(bp_paged_ctx* c, const char* what) {
  char buf[224];
  snprintf(buf, sizeof buf, "invalid config: %s", what);
  return fail(c, BP_ERR_CONFIG, buf);
}

inline int fail_cuda(bp_paged_ctx* c, cudaError_t e, const char* where) {
  char buf[224];
  const bool lost = e == cudaErrorIllegalAddress || e == cudaErrorLaunchFailure || e == cudaErrorIllegalInstruction ||
                    e == cudaErrorECCUncorrectable || e == cudaErrorHardwareStackError || e == cudaErrorMisalignedAddress;
  snprintf(buf, sizeof buf, lost ? "device lost (%s in %s)" : "CUDA error: %s in %s", cudaGetErrorString(e), where);
  if (lost) c->status = BP_ERR_DEVICE_LOST;
  return fail(c, lost ? BP_ERR_DEVICE_LOST : BP_ERR_CUDA, buf);
}

// The context's device for the length of a call; the caller's current device is put back.
struct OnDevice {
  int before = -1;
  cudaError_t err;
  explicit OnDevice(int device) {
    err = cudaGetDevice(&before);
    if (err == cudaSuccess && before != device) err = cudaSetDevice(device);
    else before = -1;
  }
  ~OnDevice() {
    if (before >= 0) (void)cudaSetDevice(before);
  }
};

inline int enter(bp_paged_ctx* c) {
  if (!c) return BP_ERR_NULL;
  if (c->status == BP_OK && c->err_host && static_cast<volatile uint32_t*>(c->err_host)[1] != 0) c->status = BP_ERR_TIMEOUT;
  if (c->status == BP_ERR_TIMEOUT) return fail(c, BP_ERR_TIMEOUT, "a bounded device-side wait gave up: create a new context");
  if (c->status != BP_OK) return fail(c, c->status, "device lost: context is unusable, create a new one");
  if (!c->err_dev) return fail(c, BP_ERR_CUDA, "the context was not created");
  return BP_OK;
}

inline const char* check_rows(const bp_rows* r, Rows* out) {
  if (reinterpret_cast<uintptr_t>(r->data) % 2) return "rows must be 2-byte aligned";
  *out = Rows{static_cast<uint16_t*>(r->data), r->tok_stride, r->head_stride};
  return nullptr;
}

inline const char* check_table(const bp_rope_table* t, uint32_t head_dim, Rope* out) {
  if (reinterpret_cast<uintptr_t>(t->cos_sin) % 8) return "a RoPE table must be 8-byte aligned";
  if (t->layout != BP_ROPE_HALF && t->layout != BP_ROPE_INTERLEAVED) return "the RoPE layout must be BP_ROPE_HALF or BP_ROPE_INTERLEAVED";
  if (t->rot_dim < 2 || t->rot_dim % 2 || t->rot_dim > head_dim) return "rot_dim must be even, at least 2 and at most head_dim";
  if (t->n_pos == 0) return "n_pos must be > 0";
  *out = Rope{static_cast<const float2*>(t->cos_sin), t->n_pos, t->rot_dim, t->layout};
  return nullptr;
}

inline const char* check_pool(const bp_kv4_pool* p, Pool* out) {
  if (p->head_dim != 64 && p->head_dim != 128) return "a 4-bit pool has head_dim 64 or 128";
  if (p->page_tokens != 16 && p->page_tokens != 32 && p->page_tokens != 64) return "page_tokens must be 16, 32 or 64";
  if (p->n_kv_head == 0 || p->n_kv_head > 65535) return "n_kv_head must be 1 .. 65535";
  if (p->n_pages == 0 || p->n_pages > 0x7fffffffu) return "n_pages must be 1 .. 2^31 - 1";
  if (reinterpret_cast<uintptr_t>(p->data) % 16) return "a pool must be 16-byte aligned";
  *out = Pool{static_cast<uint8_t*>(p->data), p->n_pages, p->page_tokens, p->page_tokens == 16 ? 4u : p->page_tokens == 32 ? 5u : 6u, p->n_kv_head};
  return nullptr;
}

inline bool aligned_to(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace paged
}  // namespace bp

#define BP_TRY(c, call)                                    \
  do {                                                     \
    cudaError_t e_ = (call);                               \
    if (e_ != cudaSuccess) return fail_cuda(c, e_, #call); \
  } while (0)
#define BP_CHECK(c, call)                             \
  do {                                                \
    const char* w_ = (call);                          \
    if (w_) return fail_config(c, w_);                \
  } while (0)
