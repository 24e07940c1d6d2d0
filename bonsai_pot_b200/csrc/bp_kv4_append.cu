// Keys and values into, and out of, a paged cache held in 4 bits (include/bonsai_paged.h has the format).
//
// append: K rows are normalised and rotated, then a block of 32 dims becomes 32 codes of 4 bits and two f16 numbers. Every
// step is an explicitly rounded binary32 operation in a fixed order, so that a token's bytes do not depend on what else is
// in the batch and a plain program can reproduce them. 4 D bytes in, 1.25 D out per (token, KV head).
// A row of D dims is D / 16 lanes: lane c has the eight dims of chunk c (8 c ..) and the eight of chunk c + D / 16, so that with
// the half layout over whole heads the two dims that turn together are in one lane, and a block is four lanes.
#include "bp_paged.cuh"

namespace {

using namespace bp;

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Eight dims of a block, of which four neighbouring lanes hold a quarter each: the codes, dim i at bits 4 i, and d, m.
__device__ __forceinline__ uint32_t quantise8(const float* x, __half* d_out, __half* m_out) {
  constexpr float LIM = 64512.f;
  float v[8], lo, hi;
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = min_nan(max_nan(x[i], -LIM), LIM);
  lo = min_nan(min_nan(min_nan(v[0], v[1]), min_nan(v[2], v[3])), min_nan(min_nan(v[4], v[5]), min_nan(v[6], v[7])));
  hi = max_nan(max_nan(max_nan(v[0], v[1]), max_nan(v[2], v[3])), max_nan(max_nan(v[4], v[5]), max_nan(v[6], v[7])));
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  // u = 2^(e - 10), e the exponent of the largest magnitude and a 64th: a power of two, so that * u and / u are exact
  const float top = __fmul_rn(fmaxf(fabsf(lo), fabsf(hi)), 1.015625f);
  const float u = fmaxf(__uint_as_float(__float_as_uint(top) & 0x7f800000u) * 0x1p-10f, 0x1p-24f);
  const float inv_u = __fdiv_rn(1.f, u);
  const float m = __fmul_rn(rintf(__fmul_rn(lo, inv_u)), u);
  const float d = __fmul_rn(rintf(__fmul_rn(__fmul_rn(__fsub_rn(hi, lo), 1.f / 15.f), inv_u)), u);
  const float inv = d > 0.f ? __fdiv_rn(1.f, d) : 0.f;
  uint32_t codes = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const float q = fminf(fmaxf(rintf(__fmul_rn(__fsub_rn(v[i], m), inv)), 0.f), 15.f);
    codes |= static_cast<uint32_t>(q) << (4 * i);
  }
  *d_out = __float2half_rn(d);
  *m_out = __float2half_rn(m);
  return codes;
}

// dims 0 .. 7 at bits 4 i -> the order of a K word: even dims in the low half, odd ones in the high half
__device__ __forceinline__ uint32_t k_word(uint32_t w) {
  uint32_t even = w & 0x0f0f0f0fu, odd = (w >> 4) & 0x0f0f0f0fu;
  even = (even | even >> 4) & 0x00ff00ffu;
  odd = (odd | odd >> 4) & 0x00ff00ffu;
  return ((even | even >> 8) & 0xffffu) | (((odd | odd >> 8) & 0xffffu) << 16);
}
__device__ __forceinline__ uint32_t k_word_back(uint32_t w) {
  uint32_t even = w & 0xffffu, odd = w >> 16;
  even = (even | even << 8) & 0x00ff00ffu;
  odd = (odd | odd << 8) & 0x00ff00ffu;
  even = (even | even << 4) & 0x0f0f0f0fu;
  odd = (odd | odd << 4) & 0x0f0f0f0fu;
  return even | odd << 4;
}

struct AppendArgs {
  Pool pool;
  Rows k, v;
  const int32_t* positions;  // null: no rotation
  const int64_t* slots;
  const uint16_t* w;
  uint32_t* err;
  Rope rope;
  uint32_t n_tok;
  float eps;
};

template <bool BF, bool VEC, int D>
__global__ void __launch_bounds__(256) kv4_append_kernel(const AppendArgs a) {
  using L = PoolLayout<D>;
  constexpr uint32_t LANES = D / 16;
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t c = threadIdx.x % LANES;
  const uint32_t row = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  // (lanes without a row stay for the shuffles, on row 0's data)
  const bool in = row < a.n_tok * a.pool.n_kv_head;
  const uint32_t tok = in ? row / a.pool.n_kv_head : 0, head = in ? row % a.pool.n_kv_head : 0;
  const int64_t slot = a.slots[tok];
  const int32_t pos = a.positions ? a.positions[tok] : 0;
  const bool over = slot >= static_cast<int64_t>(a.pool.n_pages) << a.pool.log_page || (a.positions && pos >= 0 && static_cast<uint32_t>(pos) >= a.rope.n_pos);
  const bool store = in && slot >= 0 && pos >= 0 && !over;
  if (in && over && slot >= 0 && pos >= 0 && c == 0) note_range(a.err);
  const uint16_t* k = a.k.data + tok * a.k.tok + head * a.k.head;
  const uint16_t* v = a.v.data + tok * a.v.tok + head * a.v.head;
  float x[2][8], y[2][8];
  load8<BF, VEC>(k + 8 * c, x[0]);
  load8<BF, VEC>(k + D / 2 + 8 * c, x[1]);
  float scale = 1.f;
  if (a.w) {
    float s[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      float q[8];
#pragma unroll
      for (int i = 0; i < 8; i++) q[i] = __fmul_rn(x[h][i], x[h][i]);
      s[h] = __fadd_rn(__fadd_rn(__fadd_rn(q[0], q[1]), __fadd_rn(q[2], q[3])), __fadd_rn(__fadd_rn(q[4], q[5]), __fadd_rn(q[6], q[7])));
#pragma unroll
      for (uint32_t o = 1; o < LANES; o <<= 1) s[h] = __fadd_rn(s[h], __shfl_xor_sync(0xffffffffu, s[h], o));
    }
    scale = __fdiv_rn(1.f, __fsqrt_rn(__fadd_rn(__fmul_rn(__fadd_rn(s[0], s[1]), 1.f / D), a.eps)));
#pragma unroll
    for (int h = 0; h < 2; h++) {
      float w[8];
      load8<BF, false>(a.w + h * (D / 2) + 8 * c, w);
#pragma unroll
      for (int i = 0; i < 8; i++) x[h][i] = __fmul_rn(__fmul_rn(x[h][i], scale), w[i]);
    }
  }
  auto turn = [](float own, float other, float cos, float sin) { return __fadd_rn(__fmul_rn(own, cos), __fmul_rn(other, sin)); };
#pragma unroll
  for (int h = 0; h < 2; h++)
#pragma unroll
    for (int i = 0; i < 8; i++) y[h][i] = x[h][i];
  if (a.positions) {
    const uint32_t half = a.rope.rot / 2;
    const float2* cs = a.rope.table + (store ? static_cast<size_t>(pos) * half : 0);
    if (a.rope.layout == BP_ROPE_INTERLEAVED) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const uint32_t p0 = (h * (D / 2) + 8 * c) / 2;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          if (p0 + i >= half) continue;
          const float2 t = cs[p0 + i];
          y[h][2 * i] = turn(x[h][2 * i], x[h][2 * i + 1], t.x, -t.y);
          y[h][2 * i + 1] = turn(x[h][2 * i + 1], x[h][2 * i], t.x, t.y);
        }
      }
    } else if (a.rope.rot == D) {
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float2 t = cs[8 * c + i];
        y[0][i] = turn(x[0][i], x[1][i], t.x, -t.y);
        y[1][i] = turn(x[1][i], x[0][i], t.x, t.y);
      }
    } else {  // part of a head: the other dim of a pair is read again
#pragma unroll
      for (int h = 0; h < 2; h++) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const uint32_t dim = h * (D / 2) + 8 * c + i;
          if (dim >= 2 * half) continue;
          const bool first = dim < half;
          const uint32_t other = first ? dim + half : dim - half;
          float z = to_f32<BF>(k[other]);
          if (a.w) z = __fmul_rn(__fmul_rn(z, scale), to_f32<BF>(a.w[other]));
          const float2 t = cs[first ? dim : other];
          y[h][i] = turn(x[h][i], z, t.x, first ? -t.y : t.y);
        }
      }
    }
  }
  load8<BF, VEC>(v + 8 * c, x[0]);
  load8<BF, VEC>(v + D / 2 + 8 * c, x[1]);
  const uint32_t page = a.pool.page, place = static_cast<uint32_t>(slot) & (page - 1);
  uint8_t* rec = a.pool.data;
  if (store) rec += (static_cast<size_t>(slot >> a.pool.log_page) * a.pool.n_kv_head + head) * (static_cast<size_t>(page) * L::TOK);
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const uint32_t j = c + h * LANES, b = j >> 2, q = j & 3;  // chunk j is quarter q of block b
    __half d, m;
    const uint32_t kw = k_word(quantise8(y[h], &d, &m));
    if (store) {
      *reinterpret_cast<uint32_t*>(rec + place * L::ROW + (q * L::NB + b) * 4) = kw;
      if (q == 0) {
        *reinterpret_cast<__half*>(rec + L::kd(page) + (place * L::NB + b) * 2) = d;
        *reinterpret_cast<__half*>(rec + L::km(page) + (place * L::NB + b) * 2) = m;
      }
    }
    const uint32_t vw = quantise8(x[h], &d, &m);
    if (store) {
      uint8_t* rv = rec + L::v(page);
      *reinterpret_cast<uint16_t*>(rv + place * L::ROW + L::v16(place, 2 * q, b)) = static_cast<uint16_t>(vw);
      *reinterpret_cast<uint16_t*>(rv + place * L::ROW + L::v16(place, 2 * q + 1, b)) = static_cast<uint16_t>(vw >> 16);
      if (q == 0) {
        *reinterpret_cast<__half*>(rv + L::kd(page) + (place * L::NB + b) * 2) = d;
        *reinterpret_cast<__half*>(rv + L::km(page) + (place * L::NB + b) * 2) = m;
      }
    }
  }
}

struct ReadArgs {
  Pool pool;
  Rows k, v;
  const int64_t* slots;
  uint32_t* err;
  uint32_t n_tok;
};

// A lane has one chunk of eight dims of K and of V.
template <bool BF, bool VEC, int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(const ReadArgs a) {
  using L = PoolLayout<D>;
  constexpr uint32_t LANES = D / 8;
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t j = threadIdx.x % LANES, row = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  if (row >= a.n_tok * a.pool.n_kv_head) return;
  const uint32_t tok = row / a.pool.n_kv_head, head = row % a.pool.n_kv_head;
  const int64_t slot = a.slots[tok];
  if (slot < 0) return;
  if (slot >= static_cast<int64_t>(a.pool.n_pages) << a.pool.log_page) {
    if (j == 0) note_range(a.err);
    return;
  }
  const uint32_t page = a.pool.page, place = static_cast<uint32_t>(slot) & (page - 1), b = j >> 2, q = j & 3;
  const uint8_t* rec = a.pool.data + (static_cast<size_t>(slot >> a.pool.log_page) * a.pool.n_kv_head + head) * (static_cast<size_t>(page) * L::TOK);
  const uint8_t* rv = rec + L::v(page);
  const uint32_t at = (place * L::NB + b) * 2;
  const uint32_t kw = k_word_back(*reinterpret_cast<const uint32_t*>(rec + place * L::ROW + (q * L::NB + b) * 4));
  const uint32_t vw = *reinterpret_cast<const uint16_t*>(rv + place * L::ROW + L::v16(place, 2 * q, b)) |
                      static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(rv + place * L::ROW + L::v16(place, 2 * q + 1, b))) << 16;
  const float kd = __half2float(*reinterpret_cast<const __half*>(rec + L::kd(page) + at)), km = __half2float(*reinterpret_cast<const __half*>(rec + L::km(page) + at));
  const float vd = __half2float(*reinterpret_cast<const __half*>(rv + L::kd(page) + at)), vm = __half2float(*reinterpret_cast<const __half*>(rv + L::km(page) + at));
  float x[8], y[8];
#pragma unroll
  for (int i = 0; i < 8; i++) {
    x[i] = fmaf(kd, static_cast<float>((kw >> (4 * i)) & 15), km);  // (exact: the product has 15 bits, the sum is an f16 number)
    y[i] = fmaf(vd, static_cast<float>((vw >> (4 * i)) & 15), vm);
  }
  store8<BF, VEC>(a.k.data + tok * a.k.tok + head * a.k.head + 8 * j, x);
  store8<BF, VEC>(a.v.data + tok * a.v.tok + head * a.v.head + 8 * j, y);
}

bool vec8(const Rows& r) { return reinterpret_cast<uintptr_t>(r.data) % 16 == 0 && r.tok % 8 == 0 && r.head % 8 == 0; }

}  // namespace

cudaError_t bp_launch_kv4_append(bp_paged_ctx* c, cudaStream_t s, bool bf, const Pool& pool, uint32_t head_dim, const Rows& k, const Rows& v,
                                 uint32_t n_tok, const int32_t* positions, const int64_t* slots, const Rope& rope, const uint16_t* w_norm, float eps) {
  const AppendArgs a{pool, k, v, rope.table ? positions : nullptr, slots, w_norm, c->err_dev, rope, n_tok, eps};
  auto go = [&](auto kernel, uint32_t lanes) {
    const uint32_t rows = n_tok * pool.n_kv_head, per = 256 / lanes;
    return bp_launch(true, kernel, dim3((rows + per - 1) / per), dim3(256), 0, s, a);
  };
  const bool vec = vec8(k) && vec8(v);
  if (head_dim == 128)
    return vec ? (bf ? go(kv4_append_kernel<true, true, 128>, 8) : go(kv4_append_kernel<false, true, 128>, 8))
               : (bf ? go(kv4_append_kernel<true, false, 128>, 8) : go(kv4_append_kernel<false, false, 128>, 8));
  return vec ? (bf ? go(kv4_append_kernel<true, true, 64>, 4) : go(kv4_append_kernel<false, true, 64>, 4))
             : (bf ? go(kv4_append_kernel<true, false, 64>, 4) : go(kv4_append_kernel<false, false, 64>, 4));
}

cudaError_t bp_launch_kv4_read(bp_paged_ctx* c, cudaStream_t s, bool bf, const Pool& pool, uint32_t head_dim, const int64_t* slots, uint32_t n_tok,
                               const Rows& k, const Rows& v) {
  const ReadArgs a{pool, k, v, slots, c->err_dev, n_tok};
  auto go = [&](auto kernel, uint32_t lanes) {
    const uint32_t rows = n_tok * pool.n_kv_head, per = 256 / lanes;
    return bp_launch(true, kernel, dim3((rows + per - 1) / per), dim3(256), 0, s, a);
  };
  const bool vec = vec8(k) && vec8(v);
  if (head_dim == 128)
    return vec ? (bf ? go(kv4_read_kernel<true, true, 128>, 16) : go(kv4_read_kernel<false, true, 128>, 16))
               : (bf ? go(kv4_read_kernel<true, false, 128>, 16) : go(kv4_read_kernel<false, false, 128>, 16));
  return vec ? (bf ? go(kv4_read_kernel<true, true, 64>, 8) : go(kv4_read_kernel<false, true, 64>, 8))
             : (bf ? go(kv4_read_kernel<true, false, 64>, 8) : go(kv4_read_kernel<false, false, 64>, 8));
}
