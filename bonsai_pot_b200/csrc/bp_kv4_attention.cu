// Attention of several requests over a paged 4-bit cache (include/bonsai_paged.h has the cache's format).
//
// A row is one query head of one token; the n_head / n_kv_head rows of a token share a KV head. Keys go through the tensor cores
// in tiles of 16 tokens, eight rows at a time:
//   S^T[token][row] = K Q^T    mma m16n8k16, A = the codes themselves: a nibble in an f16's low bits is the number q 2^-24
//                              (q 2^-20 one nibble up; the query's dims there are scaled by 1/16), exact in the tensor core.
//                              A block's sum is then multiplied by its d in binary32; the m's go through one m16n8k8 with the
//                              query's block sums (f16 high and low part).
//   O^T[dim][row] += V^T P^T   A = V as f16 (m + d q, which does not round by the format's choice of m and d), B = P^T, which
//                              movmatrix makes from the S^T fragments
// with a running maximum and sum per row. Queries are scaled per row by a power of two so that the largest element lies in
// [1, 2): bf16 queries then fit f16.
#include "bp_paged.cuh"

namespace {

using namespace bp;

constexpr unsigned FULL = 0xffffffffu;
constexpr float NEG_BIG = -1e30f;
constexpr float P_UP = 10.f;   // P is stored as f16 times 2^10: it keeps its bits down to 2^-24 of the maximum
constexpr uint32_t UNIT = 64;  // keys a warp works on between two looks at the maximum

struct AttnArgs {
  Pool pool;
  Rows q, out;
  const int32_t *q_start, *kv_len, *page_table;
  uint32_t* err;
  uint32_t n_req, n_head, group, total_q, max_q, max_kv, table_stride, window;
  float scale_log2;
};

// The token of a 16-token tile that a lane's MMA row r holds. K rows 2 j and 2 j + 1 then differ in parity and the values of
// MMA columns 2 t (t = 0 .. 3) lie in tokens that differ mod 4: no shared-memory bank is met twice (rows of 64 bytes).
__device__ __forceinline__ uint32_t tile_token(uint32_t r) { return (r & 8) + ((r & 1) ? 4 + (((r >> 1) & 3) ^ 1) : ((r >> 1) & 3)); }

__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ void mma_1688(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(b0));
}
__device__ __forceinline__ __half2 h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
__device__ __forceinline__ uint32_t u2(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

// Which keys a row sees: j in [lo, hi).
struct Seen {
  int lo, hi;
};

// State of one warp for one tile of eight rows.
template <int D>
struct WarpState {
  static constexpr int NB = D / 32;
  uint32_t q[NB][4];  // B fragments of S^T: dims 32 b + 8 t + {0,1}, {2,3} / 16, {4,5}, {6,7} / 16 of row g
  uint32_t qsum;      // B fragment of the m's: block sums of row g
  float s_scale[2];   // rows 2 t, 2 t + 1: softmax scale (log2) times the row's power of two
  Seen seen[2];
  float m[2], l[2];   // running maximum (log2 units) and this lane's part of the sum, of rows 2 t, 2 t + 1
  float o[2 * NB][4]; // [m-tile i][dims 32 (i / 2) + 4 g + 2 (i % 2) + {0, 1}] x rows 2 t, 2 t + 1: {d0 r0, d0 r1, d1 r0, d1 r1}
};

// Loads row g's queries; `row` counts the rows of this (request, KV head), n_rows of them.
template <int D, bool BF>
__device__ __forceinline__ void load_queries(WarpState<D>& w, const AttnArgs& a, uint32_t kv_head, uint32_t row0, uint32_t n_rows, uint32_t q0,
                                             int q_len, int kv_len, uint32_t lane) {
  constexpr int NB = D / 32;
  const uint32_t g = lane >> 2, t = lane & 3, row = row0 + g;
  float x[NB][8], big = 0.f;
#pragma unroll
  for (int b = 0; b < NB; b++)
#pragma unroll
    for (int i = 0; i < 8; i++) x[b][i] = 0.f;
  if (row < n_rows) {
    const uint16_t* p = a.q.data + static_cast<int64_t>(q0 + row / a.group) * a.q.tok + static_cast<int64_t>(kv_head * a.group + row % a.group) * a.q.head;
    const bool vec = (reinterpret_cast<uintptr_t>(p) & 15) == 0;
#pragma unroll
    for (int b = 0; b < NB; b++) {
      if (vec) load8<BF, true>(p + 32 * b + 8 * t, x[b]);
      else load8<BF, false>(p + 32 * b + 8 * t, x[b]);
#pragma unroll
      for (int i = 0; i < 8; i++) big = fmaxf(big, fabsf(x[b][i]));
    }
  }
  big = fmaxf(big, __shfl_xor_sync(FULL, big, 1));
  big = fmaxf(big, __shfl_xor_sync(FULL, big, 2));
  // 2^e <= big: its exponent bits; tiny or zero rows keep e = -126
  const uint32_t ebits = min(max(__float_as_uint(big) & 0x7f800000u, 0x00800000u), 0x7e800000u);
  const float up = __uint_as_float(0x7f000000u - ebits), down = __uint_as_float(ebits);  // 2^-e, 2^e
  float sum[NB];
#pragma unroll
  for (int b = 0; b < NB; b++) {
    sum[b] = 0.f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const __half2 h = __floats2half2_rn(x[b][2 * j] * up, x[b][2 * j + 1] * up);
      sum[b] += __low2float(h) + __high2float(h);
      w.q[b][j] = u2((j & 1) ? __hmul2(h, __float2half2_rn(0.0625f)) : h);
    }
    sum[b] += __shfl_xor_sync(FULL, sum[b], 1);
    sum[b] += __shfl_xor_sync(FULL, sum[b], 2);
  }
  // k slots 2 t, 2 t + 1 of the m's MMA: blocks (0, 1), (2, 3) in the high part, then the low part
  float a0 = sum[0], a1 = sum[1];
  if (NB == 4 && (t & 1)) {
    a0 = sum[NB - 2];
    a1 = sum[NB - 1];
  }
  const __half2 hi = __floats2half2_rn(a0, a1);
  const __half2 lo = __floats2half2_rn(a0 - __low2float(hi), a1 - __high2float(hi));
  const uint32_t lo_from = NB == 4 ? 2 : 1;
  w.qsum = t < lo_from ? u2(hi) : t < 2 * lo_from ? u2(lo) : 0u;
#pragma unroll
  for (int c = 0; c < 2; c++) {
    w.s_scale[c] = a.scale_log2 * __shfl_sync(FULL, down, 4 * (2 * t + c));
    const uint32_t r = row0 + 2 * t + c;
    const int pos = kv_len - q_len + static_cast<int>(r / a.group);
    w.seen[c].hi = r < n_rows ? min(pos + 1, kv_len) : 0;
    w.seen[c].lo = a.window ? max(pos + 1 - static_cast<int>(min(a.window, 0x7fffffffu)), 0) : 0;
    w.m[c] = NEG_BIG;
    w.l[c] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < 2 * NB; i++)
#pragma unroll
    for (int k = 0; k < 4; k++) w.o[i][k] = 0.f;
}

// S^T of 16 tokens: K codes at kc (rows of ROW bytes), d and m at kd, km (rows of 2 NB bytes).
template <int D>
__device__ __forceinline__ void scores16(const WarpState<D>& w, const uint8_t* kc, const uint8_t* kd, const uint8_t* km, uint32_t lane, float (&s)[4]) {
  using L = PoolLayout<D>;
  constexpr int NB = D / 32;
  const uint32_t g = lane >> 2, t = lane & 3, ta = tile_token(g), tb = ta + 8;
  uint32_t wa[NB], wb[NB];
  float da[NB], db[NB];
  uint32_t ma, mb;
  if constexpr (NB == 4) {
    const uint4 u = *reinterpret_cast<const uint4*>(kc + ta * L::ROW + 16 * t), v = *reinterpret_cast<const uint4*>(kc + tb * L::ROW + 16 * t);
    wa[0] = u.x; wa[1] = u.y; wa[2] = u.z; wa[3] = u.w;
    wb[0] = v.x; wb[1] = v.y; wb[2] = v.z; wb[3] = v.w;
    const uint2 e = *reinterpret_cast<const uint2*>(kd + ta * 8), f = *reinterpret_cast<const uint2*>(kd + tb * 8);
    const float2 e0 = __half22float2(h2(e.x)), e1 = __half22float2(h2(e.y)), f0 = __half22float2(h2(f.x)), f1 = __half22float2(h2(f.y));
    da[0] = e0.x; da[1] = e0.y; da[2] = e1.x; da[3] = e1.y;
    db[0] = f0.x; db[1] = f0.y; db[2] = f1.x; db[3] = f1.y;
    ma = *reinterpret_cast<const uint32_t*>(km + ta * 8 + 4 * (t & 1));
    mb = *reinterpret_cast<const uint32_t*>(km + tb * 8 + 4 * (t & 1));
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>(kc + ta * L::ROW + 8 * t), v = *reinterpret_cast<const uint2*>(kc + tb * L::ROW + 8 * t);
    wa[0] = u.x; wa[1] = u.y;
    wb[0] = v.x; wb[1] = v.y;
    const float2 e = __half22float2(h2(*reinterpret_cast<const uint32_t*>(kd + ta * 4))), f = __half22float2(h2(*reinterpret_cast<const uint32_t*>(kd + tb * 4)));
    da[0] = e.x; da[1] = e.y;
    db[0] = f.x; db[1] = f.y;
    ma = *reinterpret_cast<const uint32_t*>(km + ta * 4);
    mb = *reinterpret_cast<const uint32_t*>(km + tb * 4);
  }
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, low[4] = {0.f, 0.f, 0.f, 0.f};
  mma_1688(low, ma, mb, w.qsum);
#pragma unroll
  for (int b = 0; b < NB; b++) {
    float p[4] = {0.f, 0.f, 0.f, 0.f};
    mma_16816(p, wa[b] & 0x000f000fu, wb[b] & 0x000f000fu, wa[b] & 0x00f000f0u, wb[b] & 0x00f000f0u, w.q[b][0], w.q[b][1]);
    const uint32_t xa = wa[b] >> 8, xb = wb[b] >> 8;
    mma_16816(p, xa & 0x000f000fu, xb & 0x000f000fu, xa & 0x00f000f0u, xb & 0x00f000f0u, w.q[b][2], w.q[b][3]);
    acc[0] = fmaf(da[b], p[0], acc[0]);
    acc[1] = fmaf(da[b], p[1], acc[1]);
    acc[2] = fmaf(db[b], p[2], acc[2]);
    acc[3] = fmaf(db[b], p[3], acc[3]);
  }
#pragma unroll
  for (int k = 0; k < 4; k++) s[k] = fmaf(acc[k], 0x1p24f, low[k]) * w.s_scale[k & 1];
}

// O^T += V^T P^T of 16 tokens of which the first `valid` (>= 16: all) have been written. p0, p1: B fragments of P^T.
template <int D>
__device__ __forceinline__ void values16(WarpState<D>& w, const uint8_t* vc, const uint8_t* vd, const uint8_t* vm, uint32_t place, uint32_t valid,
                                         uint32_t lane, uint32_t p0, uint32_t p1) {
  using L = PoolLayout<D>;
  constexpr int NB = D / 32;
  const uint32_t g = lane >> 2, t = lane & 3;
  // pair 0: MMA columns 2 t, 2 t + 1; pair 1: 2 t + 8, 2 t + 9
  uint32_t av[2][NB][4];
#pragma unroll
  for (int pr = 0; pr < 2; pr++) {
    const uint32_t ta = tile_token(2 * t + 8 * pr), tb = tile_token(2 * t + 1 + 8 * pr);
    uint32_t a[NB / 2], b[NB / 2], ad[NB / 2], bd[NB / 2], am[NB / 2], bm[NB / 2];
    if constexpr (NB == 4) {
      const uint2 x = *reinterpret_cast<const uint2*>(vc + ta * L::ROW + L::v16(place + ta, g, 0)), y = *reinterpret_cast<const uint2*>(vc + tb * L::ROW + L::v16(place + tb, g, 0));
      a[0] = x.x; a[1] = x.y;
      b[0] = y.x; b[1] = y.y;
      const uint2 e = *reinterpret_cast<const uint2*>(vd + ta * 8), f = *reinterpret_cast<const uint2*>(vd + tb * 8);
      ad[0] = e.x; ad[1] = e.y;
      bd[0] = f.x; bd[1] = f.y;
      const uint2 i = *reinterpret_cast<const uint2*>(vm + ta * 8), j = *reinterpret_cast<const uint2*>(vm + tb * 8);
      am[0] = i.x; am[1] = i.y;
      bm[0] = j.x; bm[1] = j.y;
    } else {
      a[0] = *reinterpret_cast<const uint32_t*>(vc + ta * L::ROW + L::v16(place + ta, g, 0));
      b[0] = *reinterpret_cast<const uint32_t*>(vc + tb * L::ROW + L::v16(place + tb, g, 0));
      ad[0] = *reinterpret_cast<const uint32_t*>(vd + ta * 4);
      bd[0] = *reinterpret_cast<const uint32_t*>(vd + tb * 4);
      am[0] = *reinterpret_cast<const uint32_t*>(vm + ta * 4);
      bm[0] = *reinterpret_cast<const uint32_t*>(vm + tb * 4);
    }
    if (valid < 16) {  // places that nobody has written may hold any bits: P is 0 there, the values must be numbers
      const bool za = ta >= valid, zb = tb >= valid;
#pragma unroll
      for (int i = 0; i < NB / 2; i++) {
        ad[i] = za ? 0u : ad[i];
        am[i] = za ? 0u : am[i];
        bd[i] = zb ? 0u : bd[i];
        bm[i] = zb ? 0u : bm[i];
      }
    }
    const __half2 off = __float2half2_rn(-1024.f), off16 = __float2half2_rn(-64.f), sixteenth = __float2half2_rn(0.0625f);
#pragma unroll
    for (int bl = 0; bl < NB; bl++) {
      const uint32_t sel = (bl & 1) ? 0x7632u : 0x5410u;
      const uint32_t x = prmt(a[bl >> 1], b[bl >> 1], sel), y = x >> 8;
      const __half2 d = h2(prmt(ad[bl >> 1], bd[bl >> 1], sel)), m = h2(prmt(am[bl >> 1], bm[bl >> 1], sel));
      // 1024 + q and 1024 + 16 q as f16 numbers
      const __half2 q0 = __hadd2(h2((x & 0x000f000fu) | 0x64006400u), off), q1 = __hfma2(h2((x & 0x00f000f0u) | 0x64006400u), sixteenth, off16);
      const __half2 q2 = __hadd2(h2((y & 0x000f000fu) | 0x64006400u), off), q3 = __hfma2(h2((y & 0x00f000f0u) | 0x64006400u), sixteenth, off16);
      av[pr][bl][0] = u2(__hfma2(q0, d, m));
      av[pr][bl][1] = u2(__hfma2(q1, d, m));
      av[pr][bl][2] = u2(__hfma2(q2, d, m));
      av[pr][bl][3] = u2(__hfma2(q3, d, m));
    }
  }
#pragma unroll
  for (int bl = 0; bl < NB; bl++) {
    mma_16816(w.o[2 * bl], av[0][bl][0], av[0][bl][1], av[1][bl][0], av[1][bl][1], p0, p1);
    mma_16816(w.o[2 * bl + 1], av[0][bl][2], av[0][bl][3], av[1][bl][2], av[1][bl][3], p0, p1);
  }
}

// P, still as the S^T fragments of up to four tiles, from the scores: masks, maximum, exponentials, sums; O is rescaled.
template <int D>
__device__ __forceinline__ void softmax64(WarpState<D>& w, float (&s)[4][4], int key0, uint32_t lane) {
  constexpr int NB = D / 32;
  const uint32_t g = lane >> 2;
  const bool cut = key0 + static_cast<int>(UNIT) > min(w.seen[0].hi, w.seen[1].hi) || key0 < max(w.seen[0].lo, w.seen[1].lo);
  if (__any_sync(FULL, cut)) {
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int key = key0 + 16 * i + static_cast<int>(tile_token(g + 8 * (k >> 1)));
        if (key < w.seen[k & 1].lo || key >= w.seen[k & 1].hi) s[i][k] = __int_as_float(0xff800000);
      }
  }
  float mx[2];
#pragma unroll
  for (int c = 0; c < 2; c++) {
    mx[c] = fmaxf(s[0][c], s[0][c + 2]);
#pragma unroll
    for (int i = 1; i < 4; i++) mx[c] = fmaxf(mx[c], fmaxf(s[i][c], s[i][c + 2]));
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) mx[c] = fmaxf(mx[c], __shfl_xor_sync(FULL, mx[c], o));
  }
  if (__any_sync(FULL, mx[0] > w.m[0] || mx[1] > w.m[1])) {
    float corr[2];
#pragma unroll
    for (int c = 0; c < 2; c++) {
      const float m_new = fmaxf(w.m[c], mx[c]);
      corr[c] = ex2(w.m[c] - m_new);
      w.m[c] = m_new;
      w.l[c] *= corr[c];
    }
#pragma unroll
    for (int i = 0; i < 2 * NB; i++)
#pragma unroll
      for (int k = 0; k < 4; k++) w.o[i][k] *= corr[k & 1];
  }
  const float top[2] = {w.m[0] - P_UP, w.m[1] - P_UP};
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int k = 0; k < 4; k++) {
      s[i][k] = ex2(s[i][k] - top[k & 1]);
      w.l[k & 1] += s[i][k];
    }
}

// One warp per (eight rows, KV head, request), all keys one behind the other.
template <int D, bool BF>
__global__ void __launch_bounds__(32) kv4_attention_plain_kernel(const AttnArgs a) {
  using L = PoolLayout<D>;
  constexpr int NB = D / 32;
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t lane = threadIdx.x, r = blockIdx.z, head = blockIdx.y, row0 = blockIdx.x * 8;
  int q0 = max(a.q_start[r], 0), q1 = min(a.q_start[r + 1], static_cast<int>(a.total_q));
  const int q_given = max(q1 - q0, 0), q_len = min(q_given, static_cast<int>(a.max_q));
  const uint32_t n_rows = q_len * a.group;
  if (row0 >= n_rows) return;
  const uint32_t most = min(a.max_kv, a.table_stride << a.pool.log_page);
  const int given = max(a.kv_len[r], 0), kv_len = min(given, static_cast<int>(most));
  if ((given > kv_len || q_given > q_len) && lane == 0) note_range(a.err);
  WarpState<D> w;
  load_queries<D, BF>(w, a, head, row0, n_rows, q0, q_len, kv_len, lane);
  const uint32_t page = a.pool.page;
  int lo = min(w.seen[0].lo, w.seen[1].lo), hi = max(w.seen[0].hi, w.seen[1].hi);
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    lo = min(lo, __shfl_xor_sync(FULL, lo, o));
    hi = max(hi, __shfl_xor_sync(FULL, hi, o));
  }
  for (int key0 = lo / static_cast<int>(UNIT) * static_cast<int>(UNIT); key0 < hi; key0 += UNIT) {
    float s[4][4];
    const uint8_t* rec[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int key = key0 + 16 * i;
      rec[i] = nullptr;
#pragma unroll
      for (int k = 0; k < 4; k++) s[i][k] = __int_as_float(0xff800000);
      if (key >= kv_len) continue;
      const uint32_t id = static_cast<uint32_t>(a.page_table[static_cast<size_t>(r) * a.table_stride + (key >> a.pool.log_page)]);
      if (id >= a.pool.n_pages) {
        if (lane == 0 && key + 16 > lo) note_range(a.err);
        continue;
      }
      rec[i] = a.pool.data + (static_cast<size_t>(id) * a.pool.n_kv_head + head) * (static_cast<size_t>(page) * L::TOK);
      const uint32_t place = key & (page - 1);
      scores16<D>(w, rec[i] + place * L::ROW, rec[i] + L::kd(page) + place * 2 * NB, rec[i] + L::km(page) + place * 2 * NB, lane, s[i]);
    }
    softmax64<D>(w, s, key0, lane);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if (!rec[i]) continue;
      const int key = key0 + 16 * i;
      const uint32_t place = key & (page - 1);
      const uint8_t* v = rec[i] + L::v(page);
      const uint32_t p0 = movmatrix(pack2<false>(s[i][0], s[i][1])), p1 = movmatrix(pack2<false>(s[i][2], s[i][3]));
      values16<D>(w, v + place * L::ROW, v + L::kd(page) + place * 2 * NB, v + L::km(page) + place * 2 * NB, place, kv_len - key, lane, p0, p1);
    }
  }
  const uint32_t g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int c = 0; c < 2; c++) {
    float l = w.l[c];
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(FULL, l, o);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const uint32_t row = row0 + 2 * t + c;
    if (row >= n_rows) continue;
    uint16_t* out = a.out.data + static_cast<int64_t>(q0 + row / a.group) * a.out.tok + static_cast<int64_t>(head * a.group + row % a.group) * a.out.head;
#pragma unroll
    for (int i = 0; i < 2 * NB; i++) {
      const uint32_t h = pack2<BF>(w.o[i][c] * inv, w.o[i][c + 2] * inv), dim = 32 * (i >> 1) + 4 * g + 2 * (i & 1);
      out[dim] = static_cast<uint16_t>(h);
      out[dim + 1] = static_cast<uint16_t>(h >> 16);
    }
  }
}

}  // namespace

cudaError_t bp_kv4_attention_init(bp_paged_ctx* c) {
  (void)c;
  return cudaSuccess;
}

cudaError_t bp_launch_kv4_attention(bp_paged_ctx* c, cudaStream_t s, bool bf, const Pool& pool, uint32_t head_dim, const bp_kv4_attn& in) {
  AttnArgs a;
  a.pool = pool;
  a.q = Rows{static_cast<uint16_t*>(in.q.data), in.q.tok_stride, in.q.head_stride};
  a.out = Rows{static_cast<uint16_t*>(in.out.data), in.out.tok_stride, in.out.head_stride};
  a.q_start = static_cast<const int32_t*>(in.q_start);
  a.kv_len = static_cast<const int32_t*>(in.kv_len);
  a.page_table = static_cast<const int32_t*>(in.page_table);
  a.err = c->err_dev;
  a.n_req = in.n_req;
  a.n_head = in.n_head;
  a.group = in.n_head / pool.n_kv_head;
  a.total_q = in.total_q;
  a.max_q = in.max_q < in.total_q ? in.max_q : in.total_q;
  a.max_kv = in.max_kv;
  a.table_stride = in.table_stride < (0x7fffffffu >> pool.log_page) ? in.table_stride : (0x7fffffffu >> pool.log_page);
  a.window = in.window;
  a.scale_log2 = in.scale * 1.4426950408889634f;
  const dim3 grid((a.max_q * a.group + 7) / 8, pool.n_kv_head, in.n_req);
  if (head_dim == 128) return bp_launch(true, bf ? kv4_attention_plain_kernel<128, true> : kv4_attention_plain_kernel<128, false>, grid, dim3(32), 0, s, a);
  return bp_launch(true, bf ? kv4_attention_plain_kernel<64, true> : kv4_attention_plain_kernel<64, false>, grid, dim3(32), 0, s, a);
}
