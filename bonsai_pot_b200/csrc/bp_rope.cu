// Rotary positions on rows of heads, and the table they read (include/bonsai_paged.h).
//
// y1 = x1 cos - x2 sin, y2 = x2 cos + x1 sin for every pair of dims that turn together; the inverse turns by -angle, which
// is the transpose and so the gradient (a factor in cos and sin, as a YaRN table has, is applied either way). Moves 2 bytes in and 2 out per value, 4 rot bytes
// of table per token, and is bound by the latency of its loads with what fits on an SM (counters: 7.6 of 10 stalled warps per issue wait for memory).
// Measured: 16383 tokens x 24 heads x 64, 18.6 us = 5.6 TB/s of those bytes, 85 % of the rate of the measured copy; DRAM sees 62 of the 105 MB, the output stays in
// L2 (102.6 us with a warp per row and two bytes per lane, which rows of other shapes still get); 2048 x 32 x 128, 7.8 us = 4.4 TB/s (22.3 us). One token: 6.4 us
// from call to call, which is its issue from Python.
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

// Rows of 16-byte aligned chunks of eight dims, head_dim and rot_dim multiples of 16: a thread has one
// slot of 16 dims (chunks c and c + rot / 16 of the half layout, neighbours of the interleaved one, what is only copied behind) of R heads of
// a token, so that the table's row is read once for them and R rows are on their way at a time.
// G: lanes per row, the slots rounded up to a power of two, for the norm's sum.
template <bool BF, bool NORM, int R>
__global__ void __launch_bounds__(256) rope_rows_kernel(const RopeArgs a, const uint32_t log_g, const FastDiv groups_by) {
  pdl_launch_dependents();
  const uint32_t at = blockIdx.x * 256 + threadIdx.x, slot = at & ((1u << log_g) - 1), item = at >> log_g;
  const uint32_t groups = groups_by.d, tok = groups_by.quotient(item), head0 = item - tok * groups, slots = a.dim / 16, turned = a.rope.rot / 16;
  const bool in = tok < a.n_tok && slot < slots;
  // the two chunks of the slot
  uint32_t c0 = 2 * slot, c1 = 2 * slot + 1;
  if (slot < turned && a.rope.layout == BP_ROPE_HALF) {
    c0 = slot;
    c1 = slot + turned;
  }
  pdl_wait();
  int32_t pos = in ? a.positions[tok] : -1;
  if (pos >= 0 && static_cast<uint32_t>(pos) >= a.rope.n_pos) {
    note_range(a.err);
    pos = -1;
  }
  const bool go = pos >= 0;
  uint4 raw[R][2];
#pragma unroll
  for (int r = 0; r < R; r++) {
    const uint32_t head = head0 + r * groups;
    if (go && head < a.n_head) {
      const uint16_t* x = a.x.data + tok * a.x.tok + head * a.x.head;
      raw[r][0] = *reinterpret_cast<const uint4*>(x + 8 * c0);
      raw[r][1] = *reinterpret_cast<const uint4*>(x + 8 * c1);
    } else {
      raw[r][0] = raw[r][1] = make_uint4(0, 0, 0, 0);
    }
  }
  float cs[8], sn[8];  // of the slot's eight pairs
  const bool turns = go && slot < turned;
  if (turns) {
    const float4* row = reinterpret_cast<const float4*>(a.rope.table + static_cast<size_t>(pos) * (a.rope.rot / 2) + 8 * slot);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float4 t = row[i];
      cs[2 * i] = t.x;
      sn[2 * i] = t.y * a.sign;
      cs[2 * i + 1] = t.z;
      sn[2 * i + 1] = t.w * a.sign;
    }
  }
  float w[16];
  if (NORM && go) {
    if (reinterpret_cast<uintptr_t>(a.w) % 16 == 0) {
      load8<BF, true>(a.w + 8 * c0, w);
      load8<BF, true>(a.w + 8 * c1, w + 8);
    } else {
      load8<BF, false>(a.w + 8 * c0, w);
      load8<BF, false>(a.w + 8 * c1, w + 8);
    }
  }
#pragma unroll
  for (int r = 0; r < R; r++) {
    const uint32_t head = head0 + r * groups;
    float x[16];
    unpack8<BF>(raw[r][0], x);
    unpack8<BF>(raw[r][1], x + 8);
    if (NORM) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 16; i++) sum += x[i] * x[i];
      for (uint32_t o = 1; o < 1u << log_g; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const float scale = __fdiv_rn(1.f, __fsqrt_rn(sum / a.dim + a.eps));
      if (go) {
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] = x[i] * scale * w[i];
      }
    }
    if (turns) {
      if (a.rope.layout == BP_ROPE_HALF) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const float y = x[i] * cs[i] - x[8 + i] * sn[i];
          x[8 + i] = x[8 + i] * cs[i] + x[i] * sn[i];
          x[i] = y;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const float y = x[2 * i] * cs[i] - x[2 * i + 1] * sn[i];
          x[2 * i + 1] = x[2 * i + 1] * cs[i] + x[2 * i] * sn[i];
          x[2 * i] = y;
        }
      }
    }
    if (go && head < a.n_head) {
      uint16_t* out = a.out.data + tok * a.out.tok + head * a.out.head;
      *reinterpret_cast<uint4*>(out + 8 * c0) = pack8<BF>(x);
      *reinterpret_cast<uint4*>(out + 8 * c1) = pack8<BF>(x + 8);
    }
  }
}

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
  auto chunked = [](const Rows& r) { return reinterpret_cast<uintptr_t>(r.data) % 16 == 0 && r.tok % 8 == 0 && r.head % 8 == 0; };
  if (head_dim % 16 == 0 && rope.rot % 16 == 0 && chunked(x) && chunked(out) && reinterpret_cast<uintptr_t>(rope.table) % 16 == 0) {
    uint32_t log_g = 0;
    while (1u << log_g < head_dim / 16) log_g++;
    // heads of a thread: four where that still leaves every SM 2048 threads (the table's row is then read once for them), else one
    auto go = [&](auto kernel, uint32_t r) {
      const uint32_t groups = (n_head + r - 1) / r;
      const uint64_t blocks = ((static_cast<uint64_t>(n_tok) * groups << log_g) + 255) / 256;
      return bp_launch(true, kernel, dim3(static_cast<uint32_t>(blocks)), dim3(256), 0, s, a, log_g, FastDiv(groups));
    };
    const bool many = (static_cast<uint64_t>(n_tok) * n_head << log_g) / 4 >= 2048ull * c->sm_count;
    if (w_norm) return many ? go(bf ? rope_rows_kernel<true, true, 4> : rope_rows_kernel<false, true, 4>, 4) : go(bf ? rope_rows_kernel<true, true, 1> : rope_rows_kernel<false, true, 1>, 1);
    return many ? go(bf ? rope_rows_kernel<true, false, 4> : rope_rows_kernel<false, false, 4>, 4) : go(bf ? rope_rows_kernel<true, false, 1> : rope_rows_kernel<false, false, 1>, 1);
  }
  const uint32_t rows = n_tok * n_head;
  return bp_launch(true, bf ? rope_any_kernel<true> : rope_any_kernel<false>, dim3((rows + 7) / 8), dim3(256), 0, s, a);
}
