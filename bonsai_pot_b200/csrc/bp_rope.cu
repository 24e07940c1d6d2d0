// Rotary positions on rows of heads, and the table they read (include/bonsai_paged.h).
//
// y1 = x1 cos - x2 sin, y2 = x2 cos + x1 sin for every pair of dims that turn together; the inverse turns by -angle, which
// is the transpose and so the gradient. Bound by HBM: 2 bytes in and 2 out per value, 4 rot bytes of table per token.
#include "bp_paged.cuh"

namespace {

using namespace bp;

// theta_i per pair in binary64, one thread per (position, pair).
__global__ void __launch_bounds__(256) rope_fill_kernel(bp_rope_config cfg, float2* __restrict__ table) {
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t half = cfg.rot_dim / 2;
  const uint64_t at = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (at >= static_cast<uint64_t>(cfg.n_pos) * half) return;
  const uint32_t pos = static_cast<uint32_t>(at / half), i = static_cast<uint32_t>(at % half);
  const double rot = cfg.rot_dim, factor = cfg.factor;
  double base = cfg.freq_base, mscale = 1.0;
  if (cfg.scaling == BP_ROPE_SCALE_NTK) base *= pow(factor, rot / (rot - 2.0));
  double theta = pow(base, -2.0 * i / rot);
  if (cfg.scaling == BP_ROPE_SCALE_LINEAR) theta /= factor;
  if (cfg.scaling == BP_ROPE_SCALE_YARN) {
    // pair index at which a pair turns `beta` times within orig_ctx: theta orig_ctx = 2 pi beta
    auto index = [&](double beta) { return rot * log(cfg.orig_ctx / (beta * 6.283185307179586)) / (2.0 * log(base)); };
    const double low = fmax(floor(index(cfg.beta_fast)), 0.0), high = fmin(ceil(index(cfg.beta_slow)), rot - 1.0);
    const double ramp = fmin(fmax((i - low) / fmax(high - low, 0.001), 0.0), 1.0);
    theta = theta / factor * ramp + theta * (1.0 - ramp);
    if (factor > 1.0) mscale = 0.1 * log(factor) + 1.0;
  }
  double s, c;
  sincos(pos * theta, &s, &c);
  table[at] = make_float2(static_cast<float>(c * mscale), static_cast<float>(s * mscale));
}

struct RopeArgs {
  Rows x, out;
  const int32_t* positions;
  const uint16_t* w;
  uint32_t* err;
  Rope rope;
  uint32_t n_tok, n_head, dim;
  float eps, sign;  // sign: -1 turns back
};

// Any even dims, strides and alignment: a warp per row, a lane per pair, two bytes at a time.
template <bool BF>
__global__ void __launch_bounds__(256) rope_any_kernel(const RopeArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t lane = threadIdx.x & 31, row = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= a.n_tok * a.n_head) return;
  const uint32_t tok = row / a.n_head, head = row % a.n_head;
  const int32_t pos = a.positions[tok];
  if (pos < 0) return;
  if (static_cast<uint32_t>(pos) >= a.rope.n_pos) {
    note_range(a.err);
    return;
  }
  const uint16_t* x = a.x.data + tok * a.x.tok + head * a.x.head;
  uint16_t* out = a.out.data + tok * a.out.tok + head * a.out.head;
  const uint32_t half = a.rope.rot / 2, pairs = a.dim / 2;
  float x1[4], x2[4], sum = 0.f;  // 256 dims are four pairs per lane
  uint32_t i1[4], i2[4];
#pragma unroll
  for (int r = 0; r < 4; r++) {
    const uint32_t p = lane + 32 * r;
    if (p >= pairs) continue;
    i1[r] = 2 * p;
    i2[r] = 2 * p + 1;
    if (p < half && a.rope.layout == BP_ROPE_HALF) {
      i1[r] = p;
      i2[r] = p + half;
    }
    x1[r] = to_f32<BF>(x[i1[r]]);
    x2[r] = to_f32<BF>(x[i2[r]]);
    sum += x1[r] * x1[r] + x2[r] * x2[r];
  }
  float scale = 1.f;
  if (a.w) {
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    scale = __fdiv_rn(1.f, __fsqrt_rn(sum / a.dim + a.eps));
  }
  __syncwarp();  // out may be x: every lane has read its pairs
  const float2* row_cs = a.rope.table + static_cast<size_t>(pos) * half;
#pragma unroll
  for (int r = 0; r < 4; r++) {
    const uint32_t p = lane + 32 * r;
    if (p >= pairs) continue;
    if (a.w) {
      x1[r] = x1[r] * scale * to_f32<BF>(a.w[i1[r]]);
      x2[r] = x2[r] * scale * to_f32<BF>(a.w[i2[r]]);
    }
    if (p < half) {
      const float2 cs = row_cs[p];
      const float s = cs.y * a.sign, y1 = x1[r] * cs.x - x2[r] * s;
      x2[r] = x2[r] * cs.x + x1[r] * s;
      x1[r] = y1;
    }
    const uint32_t packed = pack2<BF>(x1[r], x2[r]);
    out[i1[r]] = static_cast<uint16_t>(packed);
    out[i2[r]] = static_cast<uint16_t>(packed >> 16);
  }
}

}  // namespace

cudaError_t bp_launch_rope_fill(cudaStream_t s, const bp_rope_config& cfg, float2* table) {
  const uint64_t n = static_cast<uint64_t>(cfg.n_pos) * (cfg.rot_dim / 2), blocks = (n + 255) / 256;
  if (blocks > 0x7fffffffull) return cudaErrorInvalidValue;
  return bp_launch(true, rope_fill_kernel, dim3(static_cast<uint32_t>(blocks)), dim3(256), 0, s, cfg, table);
}

cudaError_t bp_launch_rope(bp_paged_ctx* c, cudaStream_t s, bool bf, const Rows& x, const Rows& out, uint32_t n_tok, uint32_t n_head,
                           uint32_t head_dim, const int32_t* positions, const Rope& rope, const uint16_t* w_norm, float eps, bool inverse) {
  const RopeArgs a{x, out, positions, w_norm, c->err_dev, rope, n_tok, n_head, head_dim, eps, inverse ? -1.f : 1.f};
  const uint32_t rows = n_tok * n_head;
  return bp_launch(true, bf ? rope_any_kernel<true> : rope_any_kernel<false>, dim3((rows + 7) / 8), dim3(256), 0, s, a);
}
