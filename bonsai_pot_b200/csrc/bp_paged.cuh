// Shared declarations of the paged 4-bit cache operators (include/bonsai_paged.h): the context, the pool's layout as the
// kernels see it, and the conversions between the two 16-bit activation types and binary32.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/bonsai_paged.h"
#include "bp_common.cuh"
#include "bp_ptx.cuh"

struct bp_paged_ctx {
  int device;
  int sm_count;
  int status;          // latched: BP_ERR_DEVICE_LOST or BP_ERR_TIMEOUT
  uint32_t* err_host;  // pinned, mapped: [0] a token or page out of range, [1] a bounded wait gave up
  uint32_t* err_dev;   // device alias
  float* partials;     // split attention: partial results of the CTAs
  float* prefill_partials;  // the same of the kernel for many queries
  uint32_t* counters;  // split attention: partials that have arrived, zero between launches
  uint32_t* page_counter;  // page tables: CTAs that have ended, zero between launches
  char msg[256];
};

namespace bp {

// One tensor of rows on the device, strides in elements.
struct Rows {
  uint16_t* data;
  int64_t tok, head;
};

struct Rope {
  const float2* table;  // [n_pos][rot / 2]
  uint32_t n_pos, rot, layout;
};

// A pool: bytes of a page of one head, and of its parts.
struct Pool {
  uint8_t* data;
  uint32_t n_pages, page, log_page, n_kv_head;
};
template <int D>
struct PoolLayout {
  static constexpr uint32_t NB = D / 32;         // blocks of a row
  static constexpr uint32_t ROW = D / 2;         // bytes of codes of a row
  static constexpr uint32_t TOK = D * 5 / 4;     // bytes of a token of one head, K and V
  __host__ __device__ static constexpr uint32_t kd(uint32_t page) { return page * ROW; }
  __host__ __device__ static constexpr uint32_t km(uint32_t page) { return page * (ROW + 2 * NB); }
  __host__ __device__ static constexpr uint32_t v(uint32_t page) { return page * (TOK / 2); }  // the V part has the K part's order
  // byte offset of 16 bits (block b, chunk c of 8) of a V row, the changed-over halves included
  __device__ static uint32_t v16(uint32_t tok, uint32_t c, uint32_t b) {
    const uint32_t o = c * 2 * NB + 2 * b;
    return D == 128 ? o ^ ((tok & 2) << 4) : o;
  }
};

template <bool BF>
__device__ __forceinline__ float to_f32(uint16_t h) {
  return BF ? __uint_as_float(static_cast<uint32_t>(h) << 16) : __half2float(__ushort_as_half(h));
}
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if (BF) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}
template <bool BF>
__device__ __forceinline__ void unpack8(const uint4& u, float* x) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    x[2 * i] = to_f32<BF>(static_cast<uint16_t>(w[i]));
    x[2 * i + 1] = to_f32<BF>(static_cast<uint16_t>(w[i] >> 16));
  }
}
template <bool BF>
__device__ __forceinline__ uint4 pack8(const float* x) {
  return make_uint4(pack2<BF>(x[0], x[1]), pack2<BF>(x[2], x[3]), pack2<BF>(x[4], x[5]), pack2<BF>(x[6], x[7]));
}
// Eight consecutive values; VEC: 16-byte aligned, else one by one.
template <bool BF, bool VEC>
__device__ __forceinline__ void load8(const uint16_t* p, float* x) {
  if (VEC) {
    unpack8<BF>(*reinterpret_cast<const uint4*>(p), x);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = to_f32<BF>(p[i]);
  }
}
// Division of numbers below 2^31 by one divisor: with l = ceil(log2 d) and m = floor(2^32 (2^l - d) / d) + 1 the quotient is
// (mulhi(m, n) + n) >> l (Granlund and Montgomery, 1994).
struct FastDiv {
  uint32_t d, m, l;
  FastDiv() = default;
  explicit FastDiv(uint32_t by) : d(by), l(0) {
    while ((1ull << l) < by) l++;
    m = static_cast<uint32_t>((((1ull << l) - by) << 32) / by + 1);
  }
  __device__ uint32_t quotient(uint32_t n) const { return (__umulhi(m, n) + n) >> l; }
};

__device__ __forceinline__ __half2 h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
__device__ __forceinline__ uint32_t u2(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
// (x & mask) | 0x64006400 in one instruction: it has room for one constant, so the other one comes as a kernel argument
__device__ __forceinline__ __half2 biased(uint32_t x, uint32_t mask, uint32_t bias) { return h2(lop3<0xea>(x, mask, bias)); }

__device__ __forceinline__ void note_range(uint32_t* err) { *reinterpret_cast<volatile uint32_t*>(err) = 1; }

}  // namespace bp

// Launchers; the arguments have been checked.
cudaError_t bp_launch_rope_fill(cudaStream_t s, const bp_rope_config& cfg, float2* table);
cudaError_t bp_launch_rope(bp_paged_ctx* c, cudaStream_t s, bool bf, const bp::Rows& x, const bp::Rows& out, uint32_t n_tok, uint32_t n_head,
                           uint32_t head_dim, const int32_t* positions, const bp::Rope& rope, const uint16_t* w_norm, float eps, bool inverse);
cudaError_t bp_launch_kv4_append(bp_paged_ctx* c, cudaStream_t s, bool bf, const bp::Pool& pool, uint32_t head_dim, const bp::Rows& k,
                                 const bp::Rows& v, uint32_t n_tok, const int32_t* positions, const int64_t* slots, const bp::Rope& rope,
                                 const uint16_t* w_norm, float eps);
cudaError_t bp_launch_kv4_read(bp_paged_ctx* c, cudaStream_t s, bool bf, const bp::Pool& pool, uint32_t head_dim, const int64_t* slots,
                               uint32_t n_tok, const bp::Rows& k, const bp::Rows& v);
cudaError_t bp_pages_init(bp_paged_ctx* c);
cudaError_t bp_kv4_select_init(bp_paged_ctx* c);
cudaError_t bp_kv4_attention_init(bp_paged_ctx* c);
cudaError_t bp_launch_kv4_attention(bp_paged_ctx* c, cudaStream_t s, bool bf, const bp::Pool& pool, uint32_t head_dim, const bp_kv4_attn& a);
