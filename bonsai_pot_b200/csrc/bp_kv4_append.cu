// Keys and values into, and out of, a paged cache held in 4 bits (include/bonsai_paged.h has the format).
//
// append: K rows are normalised and rotated, then a block of 32 dims becomes 32 codes of 4 bits and two f16 numbers. Every
// step is an explicitly rounded binary32 operation in a fixed order, so that a token's bytes do not depend on what else is
// in the batch and a plain program can reproduce them. 4 D bytes in, 1.25 D out per (token, KV head).
// Measured: 16383 tokens x 8 heads x 128 appended and read back 47 us (floor 27.5 at the measured copy rate): about 30 for the append, bound by instruction
// issue (71 % of the slots: five per code, the tree of squares, the rotation), 17 for the read-back, bound by the latency of slot -> row. With
// narrower loads and stores and codes rounded by conversions it was 56.
// A row of D dims is D / 16 lanes: lane c has the eight dims of chunk c (8 c ..) and the eight of chunk c + D / 16, so that with
// the half layout over whole heads the two dims that turn together are in one lane, and a block is four lanes.
#include "bp_paged.cuh"

namespace {

using namespace bp;

// A NaN among them is the result.
__device__ __forceinline__ float min3_nan(float a, float b, float c) {
  float r;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Bits of a code of dim i: in a K word even dims are in the low half, odd ones in the high half; in a V word in order.
template <bool K>
__host__ __device__ constexpr int code_at(int i) {
  return K ? 4 * (i >> 1) + 16 * (i & 1) : 4 * i;
}
constexpr float MAGIC = 12582912.f;  // 1.5 2^23: the low bits of x + MAGIC are rint(x)
constexpr uint32_t MAGIC_BITS = 0x4b400000u;

// Eight dims of a block, of which four neighbouring lanes hold a quarter each: the codes, and the block's d, m.
template <bool K>
__device__ __forceinline__ uint32_t quantise8(float* x, __half* d_out, __half* m_out) {
  constexpr float LIM = 64512.f;
  float lo = min3_nan(min3_nan(x[0], x[1], x[2]), min3_nan(x[3], x[4], x[5]), min3_nan(x[6], x[7], x[7]));
  float hi = max3_nan(max3_nan(x[0], x[1], x[2]), max3_nan(x[3], x[4], x[5]), max3_nan(x[6], x[7], x[7]));
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    lo = min3_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o), lo);
    hi = max3_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o), hi);
  }
  if (!(lo >= -LIM && hi <= LIM)) {  // rare: values beyond the limit, infinities, a NaN (which stays)
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = min3_nan(max3_nan(x[i], -LIM, -LIM), LIM, LIM);
    lo = min3_nan(max3_nan(lo, -LIM, -LIM), LIM, LIM);
    hi = min3_nan(max3_nan(hi, -LIM, -LIM), LIM, LIM);
  }
  // u = 2^(e - 10), e the exponent of the largest magnitude and a 64th: a power of two, so that * u and / u are exact
  const float top = __fmul_rn(fmaxf(fabsf(lo), fabsf(hi)), 1.015625f);
  const float u = fmaxf(__uint_as_float(__float_as_uint(top) & 0x7f800000u) * 0x1p-10f, 0x1p-24f);
  const float inv_u = __uint_as_float(0x7f000000u - __float_as_uint(u));  // (of a NaN: anything, m is one)
  const float m = __fmul_rn(rintf(__fmul_rn(lo, inv_u)), u);
  const float d = __fmul_rn(rintf(__fmul_rn(__fmul_rn(__fsub_rn(hi, lo), 1.f / 15.f), inv_u)), u);
  const float inv = d > 0.f ? __fdiv_rn(1.f, d) : 0.f;
  // q = rint((x - m) inv) is at least -0.5, which rounds to 0: m is at most u / 2 above the least value and d at least u. The low
  // bits of q + MAGIC are the code; what the other bits add up to is taken off at the end.
  uint32_t codes = 0, off = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const float q = fminf(__fadd_rn(__fmul_rn(__fsub_rn(x[i], m), inv), MAGIC), MAGIC + 15.f);
    codes += __float_as_uint(q) << code_at<K>(i);
    off += MAGIC_BITS << code_at<K>(i);
  }
  *d_out = __float2half_rn(d);
  *m_out = __float2half_rn(m);
  return codes - off;
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
  FastDiv heads;
  uint32_t table_vec;  // rows of the table are 16-byte aligned
};

template <bool VEC>
__device__ __forceinline__ uint4 load_raw(const uint16_t* p) {
  if (VEC) return *reinterpret_cast<const uint4*>(p);
  uint32_t h[8];
#pragma unroll
  for (int i = 0; i < 8; i++) h[i] = p[i];
  return make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
}

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
  const uint32_t tok = in ? a.heads.quotient(row) : 0, head = in ? row - tok * a.pool.n_kv_head : 0;
  const int64_t slot = a.slots[tok];
  const int32_t pos = a.positions ? a.positions[tok] : 0;
  const bool over = slot >= static_cast<int64_t>(a.pool.n_pages) << a.pool.log_page || (a.positions && pos >= 0 && static_cast<uint32_t>(pos) >= a.rope.n_pos);
  const bool store = in && slot >= 0 && pos >= 0 && !over;
  if (in && over && slot >= 0 && pos >= 0 && c == 0) note_range(a.err);
  const uint16_t* k = a.k.data + tok * a.k.tok + head * a.k.head;
  const uint16_t* v = a.v.data + tok * a.v.tok + head * a.v.head;
  uint4 raw[4];  // K, K, V, V: every load is on its way before the first is used
#pragma unroll
  for (int i = 0; i < 4; i++) raw[i] = load_raw<VEC>((i < 2 ? k : v) + (i & 1) * (D / 2) + 8 * c);
  float x[2][8], y[2][8];
  unpack8<BF>(raw[0], x[0]);
  unpack8<BF>(raw[1], x[1]);
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
      if (reinterpret_cast<uintptr_t>(a.w) % 16 == 0) load8<BF, true>(a.w + h * (D / 2) + 8 * c, w);
      else load8<BF, false>(a.w + h * (D / 2) + 8 * c, w);
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
        float2 four[4];
        if (p0 + 4 <= half && a.table_vec) {
          const float4 e = *reinterpret_cast<const float4*>(cs + p0), f = *reinterpret_cast<const float4*>(cs + p0 + 2);
          four[0] = make_float2(e.x, e.y);
          four[1] = make_float2(e.z, e.w);
          four[2] = make_float2(f.x, f.y);
          four[3] = make_float2(f.z, f.w);
        } else {
#pragma unroll
          for (int i = 0; i < 4; i++) four[i] = p0 + i < half ? cs[p0 + i] : make_float2(1.f, 0.f);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
          if (p0 + i >= half) continue;
          const float2 t = four[i];
          y[h][2 * i] = turn(x[h][2 * i], x[h][2 * i + 1], t.x, -t.y);
          y[h][2 * i + 1] = turn(x[h][2 * i + 1], x[h][2 * i], t.x, t.y);
        }
      }
    } else if (a.rope.rot == D) {
      float2 eight[8];
      if (a.table_vec) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float4 e = reinterpret_cast<const float4*>(cs + 8 * c)[i];
          eight[2 * i] = make_float2(e.x, e.y);
          eight[2 * i + 1] = make_float2(e.z, e.w);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; i++) eight[i] = cs[8 * c + i];
      }
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float2 t = eight[i];
        y[0][i] = turn(x[0][i], x[1][i], t.x, -t.y);
        y[1][i] = turn(x[1][i], x[0][i], t.x, t.y);
      }
    } else if (half % 8 == 0) {  // part of a head, whole chunks of eight: the chunk that this one turns with is read again
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const uint32_t dim = h * (D / 2) + 8 * c;
        if (dim >= 2 * half) continue;
        const bool first = dim < half;
        const uint32_t other = first ? dim + half : dim - half, pair = first ? dim : other;
        float z[8];
        unpack8<BF>(load_raw<VEC>(k + other), z);
        if (a.w) {
          float w[8];
          if (reinterpret_cast<uintptr_t>(a.w) % 16 == 0) load8<BF, true>(a.w + other, w);
          else load8<BF, false>(a.w + other, w);
#pragma unroll
          for (int i = 0; i < 8; i++) z[i] = __fmul_rn(__fmul_rn(z[i], scale), w[i]);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const float2 t = cs[pair + i];
          y[h][i] = turn(x[h][i], z[i], t.x, first ? -t.y : t.y);
        }
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
  unpack8<BF>(raw[2], x[0]);
  unpack8<BF>(raw[3], x[1]);
  const uint32_t page = a.pool.page, place = static_cast<uint32_t>(slot) & (page - 1);
  uint8_t* rec = a.pool.data;
  if (store) rec += (static_cast<size_t>(slot >> a.pool.log_page) * a.pool.n_kv_head + head) * (static_cast<size_t>(page) * L::TOK);
  // this lane's two blocks: chunk c is quarter q of block b, chunk c + LANES the same quarter of block b + NB / 2
  __half2 kd, km, vd, vm;
  uint32_t kw[2], vw[2];
  {
    __half d0, m0, d1, m1;
    kw[0] = quantise8<true>(y[0], &d0, &m0);
    kw[1] = quantise8<true>(y[1], &d1, &m1);
    kd = __halves2half2(d0, d1);
    km = __halves2half2(m0, m1);
    vw[0] = quantise8<false>(x[0], &d0, &m0);
    vw[1] = quantise8<false>(x[1], &d1, &m1);
    vd = __halves2half2(d0, d1);
    vm = __halves2half2(m0, m1);
  }
  const uint32_t at = place * 2 * L::NB;
  if constexpr (D == 128) {
    // Lanes c and c + 4 have the blocks 0, 2 and 1, 3 of the same quarter: the first takes the K words of both, the other the V
    // words, and each writes 16 bytes; the lanes of quarter 0 the four d's and m's as well.
    const bool upper = c & 4;
    auto swap = [&](uint32_t mine_k, uint32_t mine_v) { return __shfl_xor_sync(0xffffffffu, upper ? mine_k : mine_v, 4); };
    const uint32_t w0 = swap(kw[0], vw[0]), w1 = swap(kw[1], vw[1]), sd = swap(u2(kd), u2(vd)), sm = swap(u2(km), u2(vm));
    if (!store) return;
    uint8_t* part = rec + (upper ? L::v(page) : 0);
    const uint32_t q = c & 3;
    // blocks 0 .. 3 in order: the lower lane's first, the upper lane's first, the lower lane's second, the upper lane's second
    uint4 w;
    uint32_t da, db, ma, mb;
    if (upper) {
      const uint32_t b0 = w0, b1 = vw[0], b2 = w1, b3 = vw[1];
      w = make_uint4(prmt(b0, b1, 0x5410), prmt(b2, b3, 0x5410), prmt(b0, b1, 0x7632), prmt(b2, b3, 0x7632));
      da = prmt(sd, u2(vd), 0x5410), db = prmt(sd, u2(vd), 0x7632), ma = prmt(sm, u2(vm), 0x5410), mb = prmt(sm, u2(vm), 0x7632);
    } else {
      w = make_uint4(kw[0], w0, kw[1], w1);
      da = prmt(u2(kd), sd, 0x5410), db = prmt(u2(kd), sd, 0x7632), ma = prmt(u2(km), sm, 0x5410), mb = prmt(u2(km), sm, 0x7632);
    }
    *reinterpret_cast<uint4*>(part + place * L::ROW + (upper ? L::v16(place, 2 * q, 0) : 16 * q)) = w;
    if (q == 0) {
      *reinterpret_cast<uint2*>(part + L::kd(page) + at) = make_uint2(da, db);
      *reinterpret_cast<uint2*>(part + L::km(page) + at) = make_uint2(ma, mb);
    }
  } else {
    if (!store) return;
    uint8_t* rv = rec + L::v(page);
    *reinterpret_cast<uint2*>(rec + place * L::ROW + 8 * c) = make_uint2(kw[0], kw[1]);
    *reinterpret_cast<uint2*>(rv + place * L::ROW + 8 * c) = make_uint2(prmt(vw[0], vw[1], 0x5410), prmt(vw[0], vw[1], 0x7632));
    if (c == 0) {
      *reinterpret_cast<__half2*>(rec + L::kd(page) + at) = kd;
      *reinterpret_cast<__half2*>(rec + L::km(page) + at) = km;
      *reinterpret_cast<__half2*>(rv + L::kd(page) + at) = vd;
      *reinterpret_cast<__half2*>(rv + L::km(page) + at) = vm;
    }
  }
}

struct ReadArgs {
  Pool pool;
  Rows k, v;
  const int64_t* slots;
  uint32_t* err;
  uint32_t n_tok;
  FastDiv heads;
  uint32_t bias;  // 0x64006400: two f16 numbers 1024
};

template <bool BF>
__device__ __forceinline__ uint32_t from_half2(__half2 h) {
  if (!BF) return u2(h);
  const float2 f = __half22float2(h);
  return pack2<true>(f.x, f.y);
}
template <bool VEC>
__device__ __forceinline__ void store_words(uint16_t* p, const uint32_t (&w)[4]) {
  if (VEC) {
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) p[i] = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
  }
}

// Eight lanes per row: lane t < 4 has 16 (head_dim 64: 8) bytes of the K codes, a quarter of every block, lane 4 + t the same of V.
// A lane has READ rows, whose loads are on their way together. m + d q in f16 does not round, see the format.
constexpr int READ = 2;
template <bool BF, bool VEC, int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(const ReadArgs a) {
  using L = PoolLayout<D>;
  constexpr uint32_t ROWS = 256 / 8, NB = L::NB;
  pdl_launch_dependents();
  const uint32_t kind = threadIdx.x >> 2 & 1, t = threadIdx.x & 3, page = a.pool.page, n_rows = a.n_tok * a.pool.n_kv_head;
  const Rows& to = kind ? a.v : a.k;
  uint32_t tok[READ], head[READ], codes[READ][NB], d[READ][NB / 2], m[READ][NB / 2];
  int64_t slot[READ];
  pdl_wait();
#pragma unroll
  for (int r = 0; r < READ; r++) {
    const uint32_t row = blockIdx.x * (ROWS * READ) + r * ROWS + threadIdx.x / 8;
    tok[r] = a.heads.quotient(row);
    head[r] = row - tok[r] * a.pool.n_kv_head;
    slot[r] = row < n_rows ? a.slots[tok[r]] : -1;
    if (slot[r] >= static_cast<int64_t>(a.pool.n_pages) << a.pool.log_page) {
      note_range(a.err);
      slot[r] = -1;
    }
  }
#pragma unroll
  for (int r = 0; r < READ; r++) {
    if (slot[r] < 0) continue;
    const uint32_t place = static_cast<uint32_t>(slot[r]) & (page - 1);
    const uint8_t* part = a.pool.data + (static_cast<uint64_t>(slot[r] >> a.pool.log_page) * a.pool.n_kv_head + head[r]) * (page * L::TOK) + kind * L::v(page);
    const uint8_t *p = part + place * L::ROW + (kind ? L::v16(place, 2 * t, 0) : 4 * NB * t), *pd = part + L::kd(page) + place * 2 * NB, *pm = part + L::km(page) + place * 2 * NB;
    if constexpr (NB == 4) {
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      const uint2 e = *reinterpret_cast<const uint2*>(pd), f = *reinterpret_cast<const uint2*>(pm);
      codes[r][0] = u.x, codes[r][1] = u.y, codes[r][2] = u.z, codes[r][3] = u.w;
      d[r][0] = e.x, d[r][1] = e.y, m[r][0] = f.x, m[r][1] = f.y;
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      codes[r][0] = u.x, codes[r][1] = u.y;
      d[r][0] = *reinterpret_cast<const uint32_t*>(pd), m[r][0] = *reinterpret_cast<const uint32_t*>(pm);
    }
  }
  const __half2 off = __float2half2_rn(-1024.f), off16 = __float2half2_rn(-64.f), sixteenth = __float2half2_rn(0.0625f);
#pragma unroll
  for (int r = 0; r < READ; r++) {
    if (slot[r] < 0) continue;
    uint16_t* out = to.data + tok[r] * to.tok + head[r] * to.head + 8 * t;
    if (kind) {  // words: dims 0 .. 3 of two blocks, dims 4 .. 7 of them -> a word per block
#pragma unroll
      for (uint32_t i = 0; i < NB / 2; i++) {
        const uint32_t lo = codes[r][i], hi = codes[r][NB / 2 + i];
        // (in place: block 2 i in i, block 2 i + 1 in NB / 2 + i)
        codes[r][i] = prmt(lo, hi, 0x5410);
        codes[r][NB / 2 + i] = prmt(lo, hi, 0x7632);
      }
    }
#pragma unroll
    for (uint32_t b = 0; b < NB; b++) {
      const uint32_t w = kind ? codes[r][(b & 1) * (NB / 2) + (b >> 1)] : codes[r][b], w8 = w >> 8, sel = b & 1 ? 0x3232u : 0x1010u;
      const __half2 dd = h2(prmt(d[r][b >> 1], 0, sel)), mm = h2(prmt(m[r][b >> 1], 0, sel));
      // the codes at bits 4 i of both halves
      uint32_t x[4] = {u2(__hfma2(__hadd2(biased(w, 0x000f000fu, a.bias), off), dd, mm)), u2(__hfma2(__hfma2(biased(w, 0x00f000f0u, a.bias), sixteenth, off16), dd, mm)),
                       u2(__hfma2(__hadd2(biased(w8, 0x000f000fu, a.bias), off), dd, mm)), u2(__hfma2(__hfma2(biased(w8, 0x00f000f0u, a.bias), sixteenth, off16), dd, mm))};
      if (kind) {  // dims (i, i + 4) -> in order; K has (2 i, 2 i + 1)
        const uint32_t y[4] = {prmt(x[0], x[1], 0x5410), prmt(x[2], x[3], 0x5410), prmt(x[0], x[1], 0x7632), prmt(x[2], x[3], 0x7632)};
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = y[i];
      }
#pragma unroll
      for (int i = 0; i < 4; i++) x[i] = from_half2<BF>(h2(x[i]));
      store_words<VEC>(out + 32 * b, x);
    }
  }
}

bool vec8(const Rows& r) { return reinterpret_cast<uintptr_t>(r.data) % 16 == 0 && r.tok % 8 == 0 && r.head % 8 == 0; }

}  // namespace

cudaError_t bp_launch_kv4_append(bp_paged_ctx* c, cudaStream_t s, bool bf, const Pool& pool, uint32_t head_dim, const Rows& k, const Rows& v,
                                 uint32_t n_tok, const int32_t* positions, const int64_t* slots, const Rope& rope, const uint16_t* w_norm, float eps) {
  const AppendArgs a{pool, k, v, rope.table ? positions : nullptr, slots, w_norm, c->err_dev, rope, n_tok, eps, FastDiv(pool.n_kv_head),
                     reinterpret_cast<uintptr_t>(rope.table) % 16 == 0 && rope.rot % 4 == 0};
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
  const ReadArgs a{pool, k, v, slots, c->err_dev, n_tok, FastDiv(pool.n_kv_head), 0x64006400u};
  auto go = [&](auto kernel) {
    const uint32_t rows = n_tok * pool.n_kv_head, per = 256 / 8 * READ;
    return bp_launch(true, kernel, dim3((rows + per - 1) / per), dim3(256), 0, s, a);
  };
  const bool vec = vec8(k) && vec8(v);
  if (head_dim == 128)
    return vec ? (bf ? go(kv4_read_kernel<true, true, 128>) : go(kv4_read_kernel<false, true, 128>))
               : (bf ? go(kv4_read_kernel<true, false, 128>) : go(kv4_read_kernel<false, false, 128>));
  return vec ? (bf ? go(kv4_read_kernel<true, true, 64>) : go(kv4_read_kernel<false, true, 64>))
             : (bf ? go(kv4_read_kernel<true, false, 64>) : go(kv4_read_kernel<false, false, 64>));
}
