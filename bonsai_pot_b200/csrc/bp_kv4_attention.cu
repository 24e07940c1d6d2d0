// Attention of several requests over a paged 4-bit cache (include/bonsai_paged.h has the cache's format).
//
// A row is one query head of one token; the n_head / n_kv_head rows of a token share a KV head. Keys go through the tensor cores
// in tiles of 16 tokens, eight rows at a time:
//   S^T[token][row] = K Q^T    mma m16n8k16, A = the codes themselves: a nibble in an f16's low bits is the number q 2^-24
//                              (q 2^-20 one nibble up; the query's dims there are scaled by 1/16), exact in the tensor core.
//                              A block's sum is then multiplied by its d in binary32; the m's go through one m16n8k8 with the
//                              query's block sums (f16 high and low part). The mantissa of the softmax scale comes in with these two, so
//                              that a power of two per row is left: taking the maximum off is then one operation that rounds the product of
//                              no score, and scores may be of any size (2^24 and more, where a rounded maximum is off by powers of two).
//   O^T[dim][row] += V^T P^T   A = V as f16 (m + d q, which does not round by the format's choice of m and d), B = P^T, which
//                              movmatrix makes from the S^T fragments
// with a running maximum and sum per row. Queries are multiplied per row by a power of two (RowPower): bf16 queries then fit f16. P is rounded to f16 because
// its other factor, a value of the cache, is an f16 number, which these instructions multiply by f16 alone: 2^-11 of a weight at most, where the result
// is rounded to 2^-12 (f16) or 2^-9 of itself (bf16). Against 64 bits f16 outputs err 1.1 to 1.4 times as much as with 32-bit weights, bf16 ones as much.
//
// Work is cut into units of 64 keys of one item (request, KV head, 8 NT rows), all of them in one line, of which every CTA takes
// an equal stretch and every warp of it an equal part: batches of any lengths fill the device evenly. A warp fetches its own keys and
// values (cp.async.bulk into a ring of buffers) and waits for nobody.
// Where an item ends inside a warp's stretch its rows are written at once; pieces of an item are joined, first those of a CTA's warps
// in shared memory, then those of several CTAs by the CTA that comes last (a counter per item; nobody waits), always in the order of
// the keys, so that results do not depend on who comes when.
//
// Bound by HBM in principle (1.25 head_dim bytes per key and KV head: 31.6 us for a batch of 64 requests of up to 8191 keys, 32 / 8 heads of 128, 207 MB),
// in practice by the instructions that expand the codes (about 270 per 16 tokens and warp are the formulation's, 330 were counted; the counters have 53 % of the
// issue slots used, 19 % of the tensor pipe) and by what lies
// around the stream: measured 57 us for that batch, of which 40 stream at 5.1 TB/s, 4.5 pass before a warp has its first keys and its queries, and 8
// at the end (the warps of a CTA end 1 to 3 us apart, joining a CTA's pieces takes 3, meeting the other CTAs 2, joining theirs 1 to 3). One request of 32768 keys:
// 22.5 us (floor 6.4), 11 of them streaming. Why so: with one warp per item and no split these took 772 and 3064 us; with two CTAs of eight warps and two
// buffers per warp 70 and 28; with joins by all threads of a CTA behind barriers, one item after the other, 86 and 31. 16 requests of up to 5 drafted tokens,
// 5 query heads of 64 per KV head, behind up to 4096 keys of which a window shows 1024: 19.1 us (floor 1.2).
#include <math.h>

#include <type_traits>

#include "bp_kv4_attention.cuh"

namespace {

using namespace bp;
using namespace bp::kv4;

constexpr uint32_t UNIT = 64;  // keys a warp works on between two looks at the maximum

// The token of a 16-token tile that a lane's MMA row r holds. K rows 2 j and 2 j + 1 then differ in parity and the values of
// MMA columns 2 t (t = 0 .. 3) lie in tokens that differ mod 4: no shared-memory bank is met twice (rows of 64 bytes).
__device__ __forceinline__ uint32_t tile_token(uint32_t r) { return (r & 8) + ((r & 1) ? 4 + (((r >> 1) & 3) ^ 1) : ((r >> 1) & 3)); }

__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
// D = A B, as mma_16816 without C; and of eight k's.
__device__ __forceinline__ void mma_16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_1688_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%7,%7,%7};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(b0), "f"(0.f));
}
// State of one warp for NT tiles of eight rows.
template <int D, int NT>
struct WarpState {
  static constexpr int NB = D / 32;
  uint32_t q[NT][NB][4];  // B fragments of S^T: dims 32 b + 8 t + {0,1}, {2,3} / 16, {4,5}, {6,7} / 16 of row g
  uint32_t qsum[NT];      // B fragment of the m's: block sums of row g
  float s_scale[NT][2];   // rows 2 t, 2 t + 1: the softmax scale's power of two (log2 units) times the row's (its sign is the query's, its mantissa in the scores)
  float m[NT][2], l[NT][2];   // running maximum (log2 units) and this lane's part of the sum, of rows 2 t, 2 t + 1
  float o[NT][2 * NB][4]; // [m-tile i][dims 32 (i / 2) + 4 g + 2 (i % 2) + {0, 1}] x rows 2 t, 2 t + 1: {d0 r0, d0 r1, d1 r0, d1 r1}
};

// Row g's queries as they are in memory, then as fragments. Rows of this (request, KV head) are counted from tile0, n_rows of them.
template <int D, int NT>
struct RawQueries {
  uint4 u[NT][D / 32];
};
template <int D, int NT>
__device__ __forceinline__ void ask_queries(RawQueries<D, NT>& raw, const AttnArgs& a, uint32_t kv_head, uint32_t tile0, uint32_t n_rows, uint32_t q0, uint32_t lane) {
#pragma unroll
  for (int e = 0; e < NT; e++) {
    const uint32_t r = min(tile0 + 8 * e + (lane >> 2), n_rows - 1);
    const uint16_t* p = a.q.data + static_cast<int64_t>(q0 + r / a.group) * a.q.tok + static_cast<int64_t>(kv_head * a.group + r % a.group) * a.q.head + 8 * (lane & 3);
    if (a.q_vec) {
#pragma unroll
      for (int b = 0; b < D / 32; b++) raw.u[e][b] = *reinterpret_cast<const uint4*>(p + 32 * b);
    } else {
#pragma unroll
      for (int b = 0; b < D / 32; b++) {
        uint32_t h[8];
#pragma unroll
        for (int i = 0; i < 8; i++) h[i] = p[32 * b + i];
        raw.u[e][b] = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
      }
    }
  }
}
template <int D, int NT>
__device__ __forceinline__ void set_queries(WarpState<D, NT>& w, RawQueries<D, NT>& raw, const AttnArgs& a, uint32_t tile0, uint32_t n_rows, uint32_t lane) {
  constexpr int NB = D / 32;
  const uint32_t g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int e = 0; e < NT; e++) {
    const uint32_t row = tile0 + 8 * e + g;
    float x[NB][8], big = 0.f;
    if (row >= n_rows) {
#pragma unroll
      for (int b = 0; b < NB; b++) raw.u[e][b] = make_uint4(0, 0, 0, 0);
    }
    if (a.bf) {
#pragma unroll
      for (int b = 0; b < NB; b++) unpack8<true>(raw.u[e][b], x[b]);
    } else {
#pragma unroll
      for (int b = 0; b < NB; b++) unpack8<false>(raw.u[e][b], x[b]);
    }
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int i = 0; i < 8; i++) big = fmaxf(big, fabsf(x[b][i]));
    big = fmaxf(big, __shfl_xor_sync(FULL, big, 1));
    big = fmaxf(big, __shfl_xor_sync(FULL, big, 2));
    const RowPower power = RowPower::of(big);
    const float down = power.down(), turn = copysignf(power.up(), a.scale_log2);
    float sum[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) {
      sum[b] = 0.f;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const __half2 h = __floats2half2_rn(x[b][2 * j] * turn, x[b][2 * j + 1] * turn);
        sum[b] += __low2float(h) + __high2float(h);
        w.q[e][b][j] = u2((j & 1) ? __hmul2(h, __float2half2_rn(0.0625f)) : h);
      }
      sum[b] += __shfl_xor_sync(FULL, sum[b], 1);
      sum[b] += __shfl_xor_sync(FULL, sum[b], 2);
      sum[b] *= a.mantissa;
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
    w.qsum[e] = t < lo_from ? u2(hi) : t < 2 * lo_from ? u2(lo) : 0u;
#pragma unroll
    for (int c = 0; c < 2; c++) {
      // (never 0: a masked score, -infinity, stays what it is)
      w.s_scale[e][c] = fmaxf(a.power * __shfl_sync(FULL, down, 4 * (2 * t + c)), 0x1p-122f);
      w.m[e][c] = NEG_BIG;
      w.l[e][c] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < 2 * NB; i++)
#pragma unroll
      for (int k = 0; k < 4; k++) w.o[e][i][k] = 0.f;
  }
}

// Where the k-th 16 tokens of a unit's K or V lie: `part` = the offset of a page's codes, d or m, `row` = bytes of a token of it.
template <int D, uint32_t PAGE>
__device__ constexpr uint32_t tile_at(int k, uint32_t row, uint32_t part) {
  return 16u * k / PAGE * (PAGE * (PoolLayout<D>::TOK / 2)) + part + 16u * k % PAGE * row;
}

// S^T of the k-th 16 tokens of a unit, times the softmax scale's mantissa.
template <int D, int NT, uint32_t PAGE>
__device__ __forceinline__ void scores16(const WarpState<D, NT>& w, const uint8_t* buf, uint32_t lane, float (&s)[NT][4][4], int k, float mantissa24) {
  using L = PoolLayout<D>;
  constexpr int NB = D / 32;
  const uint8_t *kc = buf + tile_at<D, PAGE>(k, L::ROW, 0), *kd = buf + tile_at<D, PAGE>(k, 2 * NB, L::kd(PAGE)), *km = buf + tile_at<D, PAGE>(k, 2 * NB, L::km(PAGE));
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
#pragma unroll
  for (int e = 0; e < NT; e++) {
    float acc[4] = {0.f, 0.f, 0.f, 0.f}, low[4];
    mma_1688_first(low, ma, mb, w.qsum[e]);
#pragma unroll
    for (int b = 0; b < NB; b++) {
      float p[4];
      mma_16816_first(p, wa[b] & 0x000f000fu, wb[b] & 0x000f000fu, wa[b] & 0x00f000f0u, wb[b] & 0x00f000f0u, w.q[e][b][0], w.q[e][b][1]);
      const uint32_t xa = wa[b] >> 8, xb = wb[b] >> 8;
      mma_16816(p, xa & 0x000f000fu, xb & 0x000f000fu, xa & 0x00f000f0u, xb & 0x00f000f0u, w.q[e][b][2], w.q[e][b][3]);
      acc[0] = fmaf(da[b], p[0], acc[0]);
      acc[1] = fmaf(da[b], p[1], acc[1]);
      acc[2] = fmaf(db[b], p[2], acc[2]);
      acc[3] = fmaf(db[b], p[3], acc[3]);
    }
#pragma unroll
    for (int c = 0; c < 4; c++) s[e][k][c] = fmaf(acc[c], mantissa24, low[c]);
  }
}

// O^T += V^T P^T of the k-th 16 tokens of a unit. s: P as S^T fragments.
template <int D, int NT, uint32_t PAGE>
__device__ __forceinline__ void values16(WarpState<D, NT>& w, const uint8_t* buf, uint32_t lane, const float (&s)[NT][4][4], int k, uint32_t bias) {
  using L = PoolLayout<D>;
  constexpr int NB = D / 32;
  const uint32_t g = lane >> 2, t = lane & 3;
  const uint8_t *vc = buf + tile_at<D, PAGE>(k, L::ROW, 0), *vd = buf + tile_at<D, PAGE>(k, 2 * NB, L::kd(PAGE)), *vm = buf + tile_at<D, PAGE>(k, 2 * NB, L::km(PAGE));
  // [pair 0: MMA columns 2 t, 2 t + 1; pair 1: 2 t + 8, 2 t + 9][first, second token]
  uint32_t codes[2][2][NB / 2], dw[2][2][NB / 2], mw[2][2][NB / 2];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t tok = tile_token(2 * t + (i & 1) + 8 * (i >> 1));
    uint32_t(&c)[NB / 2] = codes[i >> 1][i & 1], (&d)[NB / 2] = dw[i >> 1][i & 1], (&m)[NB / 2] = mw[i >> 1][i & 1];
    if constexpr (NB == 4) {
      const uint2 x = *reinterpret_cast<const uint2*>(vc + tok * L::ROW + L::v16(tok, g, 0)), e = *reinterpret_cast<const uint2*>(vd + tok * 8),
                  f = *reinterpret_cast<const uint2*>(vm + tok * 8);
      c[0] = x.x; c[1] = x.y;
      d[0] = e.x; d[1] = e.y;
      m[0] = f.x; m[1] = f.y;
    } else {
      c[0] = *reinterpret_cast<const uint32_t*>(vc + tok * L::ROW + L::v16(tok, g, 0));
      d[0] = *reinterpret_cast<const uint32_t*>(vd + tok * 4);
      m[0] = *reinterpret_cast<const uint32_t*>(vm + tok * 4);
    }
  }
  uint32_t p0[NT], p1[NT];
#pragma unroll
  for (int e = 0; e < NT; e++) {
    p0[e] = movmatrix(pack2<false>(s[e][k][0], s[e][k][1]));
    p1[e] = movmatrix(pack2<false>(s[e][k][2], s[e][k][3]));
  }
  const __half2 off = __float2half2_rn(-1024.f), off16 = __float2half2_rn(-64.f), sixteenth = __float2half2_rn(0.0625f);
#pragma unroll
  for (int bl = 0; bl < NB; bl++) {
    const uint32_t sel = (bl & 1) ? 0x7632u : 0x5410u;
    uint32_t av[2][4];
#pragma unroll
    for (int pr = 0; pr < 2; pr++) {
      const uint32_t x = prmt(codes[pr][0][bl >> 1], codes[pr][1][bl >> 1], sel), y = x >> 8;
      const __half2 d = h2(prmt(dw[pr][0][bl >> 1], dw[pr][1][bl >> 1], sel)), m = h2(prmt(mw[pr][0][bl >> 1], mw[pr][1][bl >> 1], sel));
      // 1024 + q and 1024 + 16 q as f16 numbers, then q
      av[pr][0] = u2(__hfma2(__hadd2(biased(x, 0x000f000fu, bias), off), d, m));
      av[pr][1] = u2(__hfma2(__hfma2(biased(x, 0x00f000f0u, bias), sixteenth, off16), d, m));
      av[pr][2] = u2(__hfma2(__hadd2(biased(y, 0x000f000fu, bias), off), d, m));
      av[pr][3] = u2(__hfma2(__hfma2(biased(y, 0x00f000f0u, bias), sixteenth, off16), d, m));
    }
#pragma unroll
    for (int e = 0; e < NT; e++) {
      mma_16816(w.o[e][2 * bl], av[0][0], av[0][1], av[1][0], av[1][1], p0[e], p1[e]);
      mma_16816(w.o[e][2 * bl + 1], av[0][2], av[0][3], av[1][2], av[1][3], p0[e], p1[e]);
    }
  }
}

// P, still as the S^T fragments of four tiles, from the scores: masks (cut: some row may not see all of the unit, of which `left` keys are there), maximum, exponentials, sums; O is rescaled.
template <int D, int NT>
__device__ __forceinline__ void softmax64(WarpState<D, NT>& w, float (&s)[NT][4][4], bool cut, int left, uint32_t tile0, int q_len, const AttnArgs& a, uint32_t lane) {
  constexpr int NB = D / 32;
  const uint32_t g = lane >> 2;
#pragma unroll
  for (int e = 0; e < NT; e++) {
    if (cut) {
#pragma unroll
      for (int c = 0; c < 2; c++) {
        // the keys of the unit that row 2 t + c sees are [lo, hi); columns behind the request's rows are left as they are, nobody reads them
        const int behind = q_len - 1 - static_cast<int>((tile0 + 8 * e + 2 * (lane & 3) + c) / a.group);  // queries behind this one
        const int hi = behind < 0 ? left : left - behind, lo = a.window && behind >= 0 ? hi - static_cast<int>(a.window) : 0;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int k = c; k < 4; k += 2) {
            const int key = 16 * i + static_cast<int>(tile_token(g + 8 * (k >> 1)));
            if (key < lo || key >= hi) s[e][i][k] = __int_as_float(0xff800000);
          }
      }
    }
    float mx[2];
#pragma unroll
    for (int c = 0; c < 2; c++) {
      mx[c] = fmaxf(s[e][0][c], s[e][0][c + 2]);
#pragma unroll
      for (int i = 1; i < 4; i++) mx[c] = fmaxf(mx[c], fmaxf(s[e][i][c], s[e][i][c + 2]));
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) mx[c] = fmaxf(mx[c], __shfl_xor_sync(FULL, mx[c], o));
      mx[c] *= w.s_scale[e][c];
    }
    if (__any_sync(FULL, mx[0] > w.m[e][0] || mx[1] > w.m[e][1])) {
      float corr[2];
#pragma unroll
      for (int c = 0; c < 2; c++) {
        const float m_new = fmaxf(w.m[e][c], mx[c]);
        corr[c] = ex2(w.m[e][c] - m_new);
        w.m[e][c] = m_new;
        w.l[e][c] *= corr[c];
      }
#pragma unroll
      for (int i = 0; i < 2 * NB; i++)
#pragma unroll
        for (int k = 0; k < 4; k++) w.o[e][i][k] *= corr[k & 1];
    }
    const float top[2] = {w.m[e][0] - P_UP, w.m[e][1] - P_UP};
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int k = 0; k < 4; k++) {
        s[e][i][k] = ex2(fmaf(s[e][i][k], w.s_scale[e][k & 1], -top[k & 1]));
        w.l[e][k & 1] += s[e][i][k];
      }
  }
}


// One CTA per SM. A warp fetches ahead into RING buffers, K and V of its units in turn: one is worked on, the others are on
// their way. Head_dim 128, eight rows: 12 warps with three buffers take 57 us for the batch above and 22.5 for 32768 keys; 16 warps
// (128 registers, spills) with two 58.6 and 24.6.
template <int D, int NT>
struct Shape {
  static constexpr uint32_t ROWS = 8 * NT;                               // rows of an item
  static constexpr uint32_t NWARP = D == 128 ? (NT == 1 ? 12 : 8) : (NT == 1 ? 16 : 12), THREADS = 32 * NWARP;
  static constexpr uint32_t RING = D == 128 && NT == 1 ? 3 : 4;
  static constexpr uint32_t PART = UNIT * PoolLayout<D>::TOK / 2;        // bytes of a unit's K (or V)
  static constexpr uint32_t STRIDE = D + 4;                              // floats of a row of a partial result: o, m, l
  static constexpr uint32_t PARTIAL = ROWS * STRIDE;                     // floats of one
  static constexpr uint32_t SMEM = NWARP * RING * PART;
  static_assert(PARTIAL * 4 <= RING * PART && 2 * NWARP <= 32, "a partial result goes over its warp's buffers; a lane per piece");
};

// What one request asks for.
struct Request {
  int q0, q_len, kv_len, low;  // low: no query sees a key before it
  uint32_t units, tiles;       // units of 64 keys of an item; items per KV head (none without keys: there are only zeros to write)
  __device__ int first() const { return low & ~static_cast<int>(UNIT - 1); }
};
template <int NT>
__device__ __forceinline__ Request request(const AttnArgs& a, uint32_t r, bool report) {
  Request q;
  const Lengths n = lengths_of(a, r, report);
  q.q0 = n.q0;
  q.q_len = n.q_len;
  q.kv_len = n.kv_len;
  q.low = min(first_seen(q.kv_len - q.q_len + 1, a.window), q.kv_len);
  q.units = (static_cast<uint32_t>(q.kv_len - q.first()) + UNIT - 1) / UNIT;
  q.tiles = q.kv_len ? (static_cast<uint32_t>(q.q_len) * a.group + 8 * NT - 1) / (8 * NT) : 0;
  return q;
}

// A place in the line of units.
struct Cursor {
  Request q;
  uint32_t r, head, tile, unit;
};
// The next item (a cursor lies in shared memory, one lane moves it). known: the requests, or null if there are too many.
template <int NT>
__device__ __forceinline__ void next_item(Cursor& c, const AttnArgs& a, const Request* known) {
  c.unit = 0;
  if (++c.tile < c.q.tiles) return;
  c.tile = 0;
  if (++c.head < a.pool.n_kv_head) return;
  c.head = 0;
  do {
    if (++c.r >= a.n_req) return;
    c.q = known ? known[c.r] : request<NT>(a, c.r, false);
  } while (c.q.tiles == 0);
}

// A piece of an item that one warp has worked on: the item's first unit in the line and its units; its rows.
struct Piece {
  uint32_t used, start, units, head, row0, rows;
  int q0;
};
// An item whose pieces lie in several CTAs: one of this CTA's pieces of it, where it begins, over how many CTAs it goes.
struct Join {
  uint32_t piece, first_cta, n, last;
};

// The unit that is fetched, one lane per page.
struct Fetch {
  int key0, kv_len, low;
  uint32_t rem;        // units of the item from this one on
  uint32_t ids, base;  // ids: lane l has the page id of page `base + l` of the request
  uint32_t pages;      // those that are fetched: they hold keys of [low, kv_len) and have a good id
  const uint8_t* src;  // this lane's page, K
};
// What the warp has to know of a unit when it works on it: keys from its first one to the last one, keys before the first that
// is looked at (both relative to the unit), the pages that were fetched, whether the item ends with it.
struct Unit {
  int left, low;
  uint32_t pages, ends;
};
__device__ __forceinline__ void copy_pages(uint32_t pages, const uint8_t* src, uint32_t bytes, uint32_t dst, uint32_t bar, uint32_t lane) {
  if (lane == 0) mbar_arrive_expect_tx(bar, __popc(pages) * bytes);
  __syncwarp();
  if (pages >> lane & 1)
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst + lane * bytes), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
template <uint32_t PAGE>
__device__ __forceinline__ void load_ids(Fetch& f, const AttnArgs& a, uint32_t r, uint32_t lane) {
  f.base = static_cast<uint32_t>(f.key0) / PAGE;
  f.ids = 0xffffffffu;
  if (f.base + lane < (static_cast<uint32_t>(f.kv_len) + PAGE - 1) / PAGE) f.ids = static_cast<uint32_t>(a.page_table[static_cast<size_t>(r) * a.table_stride + f.base + lane]);
}
template <uint32_t PAGE>
__device__ __forceinline__ void start_item(Fetch& f, const AttnArgs& a, const Cursor& c, uint32_t lane) {
  f.key0 = c.q.first() + static_cast<int>(c.unit * UNIT);
  f.kv_len = c.q.kv_len;
  f.low = c.q.low;
  f.rem = c.q.units - c.unit;
  load_ids<PAGE>(f, a, c.r, lane);
}
template <int D, uint32_t PAGE>
__device__ __forceinline__ void fetch_keys(Fetch& f, const AttnArgs& a, const Cursor& c, Unit& info, uint32_t dst, uint32_t bar, uint32_t lane) {
  constexpr uint32_t N = UNIT / PAGE, BYTES = PAGE * (PoolLayout<D>::TOK / 2);
  const uint32_t page0 = static_cast<uint32_t>(f.key0) / PAGE;
  if (page0 - f.base >= 32) load_ids<PAGE>(f, a, c.r, lane);
  const uint32_t id = __shfl_sync(FULL, f.ids, (page0 - f.base + lane) & 31);
  const int key = f.key0 + static_cast<int>(lane * PAGE);
  const bool there = lane < N && key < f.kv_len && key + static_cast<int>(PAGE) > f.low, good = there && id < a.pool.n_pages;
  if (there && !good) note_range(a.err);
  f.pages = __ballot_sync(FULL, good);
  if (lane == 0) info = Unit{f.kv_len - f.key0, f.low - f.key0, f.pages, f.rem == 1};
  f.src = a.pool.data + (static_cast<uint64_t>(id) * a.pool.n_kv_head + c.head) * (2 * BYTES);
  copy_pages(f.pages, f.src, BYTES, dst, bar, lane);
}

// Places of a unit's K or V that hold no key of the request may hold any bits: their d and m become 0, so that the values are
// numbers (P is 0 there). pages: those that have been fetched; tokens [from, to) are the request's.
template <int D, uint32_t PAGE>
__device__ __noinline__ void clear_scales(uint8_t* buf, uint32_t pages, int from, int to) {
  using L = PoolLayout<D>;
  for (uint32_t tok = threadIdx.x & 31; tok < UNIT; tok += 32) {
    if ((pages >> (tok / PAGE) & 1) && static_cast<int>(tok) >= from && static_cast<int>(tok) < to) continue;
    uint8_t* at = buf + tok / PAGE * (PAGE * (L::TOK / 2)) + L::kd(PAGE) + tok % PAGE * 2 * L::NB;
    for (uint32_t i = 0; i < L::NB / 2; i++) {
      reinterpret_cast<uint32_t*>(at)[i] = 0;
      reinterpret_cast<uint32_t*>(at + L::km(PAGE) - L::kd(PAGE))[i] = 0;
    }
  }
  fence_proxy_async();  // the next copy into the buffer comes behind these
  __syncwarp();
}

// A token's d's in a buffer with a unit's K or V; bits of its blocks that have a scale that is no finite number.
template <int D, uint32_t PAGE>
__device__ __forceinline__ uint16_t* scales_at(uint8_t* buf, uint32_t tok) {
  using L = PoolLayout<D>;
  return reinterpret_cast<uint16_t*>(buf + tok / PAGE * (PAGE * (L::TOK / 2)) + L::kd(PAGE) + tok % PAGE * 2 * L::NB);
}
template <int D, uint32_t PAGE>
__device__ __forceinline__ uint32_t blocks_without_numbers(uint8_t* buf, uint32_t tok) {
  using L = PoolLayout<D>;
  const uint32_t *d = reinterpret_cast<const uint32_t*>(scales_at<D, PAGE>(buf, tok)), *m = d + (L::km(PAGE) - L::kd(PAGE)) / 4;
  uint32_t bad = 0;
#pragma unroll
  for (uint32_t b = 0; b < L::NB / 2; b++) bad |= no_numbers(d[b], m[b]) << (2 * b);
  return bad;
}
// Values that are no numbers, in a unit of which an item's rows see different keys: 0 times such a value is not 0, so the blocks become zeros in the buffer
// and are counted here, for the rows that see them. Returns what to write over: bit 2 NB e + NB c + b is block b of row 2 t + c of tile e.
template <int D, int NT, uint32_t PAGE>
__device__ __noinline__ uint32_t take_no_numbers(uint8_t* buf, int left, uint32_t tile0, int q_len, uint32_t group, uint32_t window) {
  using L = PoolLayout<D>;
  constexpr uint32_t NB = L::NB;
  const uint32_t lane = threadIdx.x & 31;
  uint32_t found = 0;
#pragma unroll 1
  for (uint32_t k = 0; k < UNIT; k += 32) {
    const uint32_t tok = k + lane;
    uint16_t *d = scales_at<D, PAGE>(buf, tok), *m = d + (L::km(PAGE) - L::kd(PAGE)) / 2;
    const uint32_t bad = blocks_without_numbers<D, PAGE>(buf, tok);
#pragma unroll
    for (uint32_t b = 0; b < NB; b++)
      if (bad >> b & 1) d[b] = m[b] = 0;
    for (uint32_t who = __ballot_sync(FULL, bad != 0); who; who &= who - 1) {
      const int at = __ffs(who) - 1, key = static_cast<int>(k) + at;
      const uint32_t blocks = __shfl_sync(FULL, bad, at);
      for (uint32_t e = 0; e < NT; e++)
        for (uint32_t c = 0; c < 2; c++) {
          const int behind = q_len - 1 - static_cast<int>((tile0 + 8 * e + 2 * (lane & 3) + c) / group), hi = left - behind;
          if (behind >= 0 && key < hi && (window == 0 || key >= hi - static_cast<int>(window))) found |= blocks << (NB * (2 * e + c));
        }
    }
  }
  fence_proxy_async();  // the next copy into the buffer comes behind these
  __syncwarp();
  return found;
}

// A warp: row `row` of the `n` partial results at part(k) of an item, in order, becomes the output's row.
template <int D, int NT, typename Part>
__device__ __forceinline__ void join_row(const AttnArgs& a, const Piece& p, uint32_t row, uint32_t n, Part part, uint32_t lane) {
  using S = Shape<D, NT>;
  constexpr int V = D / 32;  // dims of a lane
  float m = NEG_BIG, l = 0.f, o[V] = {};
  for (uint32_t k0 = 0; k0 < n; k0 += 32) {
    const uint32_t some = min(n - k0, 32u);
    const float2 ml = lane < some ? *reinterpret_cast<const float2*>(part(k0 + lane) + row * S::STRIDE + D) : make_float2(NEG_BIG, 0.f);
    float top = ml.x;
#pragma unroll
    for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, x));
    top = fmaxf(top, m);
    const float before = ex2(m - top), weight = ex2(ml.x - top);
    float sum = weight * ml.y;
#pragma unroll
    for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(FULL, sum, x);
    l = l * before + sum;
    m = top;
#pragma unroll
    for (int x = 0; x < V; x++) o[x] *= before;
#pragma unroll 8
    for (uint32_t k = 0; k < some; k++) {
      const float* v = part(k0 + k) + row * S::STRIDE + V * lane;
      const float wk = __shfl_sync(FULL, weight, k);
      if constexpr (V == 4) {
        const float4 e = *reinterpret_cast<const float4*>(v);
        o[0] = fmaf(e.x, wk, o[0]);
        o[1] = fmaf(e.y, wk, o[1]);
        o[2] = fmaf(e.z, wk, o[2]);
        o[3] = fmaf(e.w, wk, o[3]);
      } else {
        const float2 e = *reinterpret_cast<const float2*>(v);
        o[0] = fmaf(e.x, wk, o[0]);
        o[1] = fmaf(e.y, wk, o[1]);
      }
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint16_t* out = out_row(a, p.q0, p.head, p.row0 + row) + V * lane;
  if constexpr (V == 4) {
    store4(a.bf, out, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
  } else {
    const uint32_t h = a.bf ? pack2<true>(o[0] * inv, o[1] * inv) : pack2<false>(o[0] * inv, o[1] * inv);
    out[0] = static_cast<uint16_t>(h);
    out[1] = static_cast<uint16_t>(h >> 16);
  }
}

// The same of four rows at a time, eight lanes each, for few partial results, one after the other; into the output (to == null) or the partial
// result `to`.
template <int D, int NT, typename Part>
__device__ __forceinline__ void join_rows4(const AttnArgs& a, const Piece& p, uint32_t row0, uint32_t n, Part part, float* to, uint32_t lane) {
  using S = Shape<D, NT>;
  constexpr int V = D / 32;  // fours of dims of a lane
  const uint32_t row = min(row0 + (lane >> 3), p.rows - 1), at = row * S::STRIDE, col = 4 * (lane & 7);
  float m = NEG_BIG, l = 0.f;
  float4 o[V];
#pragma unroll
  for (int x = 0; x < V; x++) o[x] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
  for (uint32_t k = 0; k < n; k++) {
    const float* v = part(k) + at;
    const float2 ml = *reinterpret_cast<const float2*>(v + D);
    float4 e[V];
#pragma unroll
    for (int x = 0; x < V; x++) e[x] = *reinterpret_cast<const float4*>(v + 32 * x + col);
    const float top = fmaxf(m, ml.x), w0 = ex2(m - top), w1 = ex2(ml.x - top);
    m = top;
    l = l * w0 + ml.y * w1;
#pragma unroll
    for (int x = 0; x < V; x++) o[x] = make_float4(o[x].x * w0 + e[x].x * w1, o[x].y * w0 + e[x].y * w1, o[x].z * w0 + e[x].z * w1, o[x].w * w0 + e[x].w * w1);
  }
  if (row0 + (lane >> 3) >= p.rows) return;
  if (to) {
#pragma unroll
    for (int x = 0; x < V; x++) *reinterpret_cast<float4*>(to + at + 32 * x + col) = o[x];
    if ((lane & 7) == 0) *reinterpret_cast<float2*>(to + at + D) = make_float2(m, l);
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint16_t* out = out_row(a, p.q0, p.head, p.row0 + row) + col;
#pragma unroll
  for (int x = 0; x < V; x++) store4(a.bf, out + 32 * x, o[x].x * inv, o[x].y * inv, o[x].z * inv, o[x].w * inv);
}

// Zeros for the `n_tok` tokens of a request without keys, by a CTA. (Their values can be more than 32 bits count.)
template <int D>
__device__ __noinline__ void zero_rows(const AttnArgs& a, int q0, uint32_t n_tok) {
  const uint32_t step = blockDim.x / (D / 4), dt = step / a.n_head, dh = step % a.n_head;  // rows that the CTA writes at a time
  const uint32_t row = threadIdx.x / (D / 4);
  for (uint32_t t = row / a.n_head, h = row % a.n_head; t < n_tok;) {
    store4(false, a.out.data + static_cast<int64_t>(q0 + t) * a.out.tok + static_cast<int64_t>(h) * a.out.head + threadIdx.x % (D / 4) * 4, 0.f, 0.f, 0.f, 0.f);
    t += dt;
    h += dh;
    if (h >= a.n_head) {
      h -= a.n_head;
      t++;
    }
  }
}

template <int D, int NT, uint32_t PAGE>
__global__ void __launch_bounds__(Shape<D, NT>::THREADS, 1) kv4_attention_kernel(const __grid_constant__ AttnArgs a, float* __restrict__ scratch, uint32_t* __restrict__ counters) {
  using S = Shape<D, NT>;
  using L = PoolLayout<D>;
  constexpr int NB = D / 32;
  constexpr uint32_t NWARP = S::NWARP, THREADS = S::THREADS, RING = S::RING, HALF = PAGE * (L::TOK / 2), ALL_PAGES = (1u << UNIT / PAGE) - 1;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t bars[NWARP][RING];
  __shared__ uint32_t line[THREADS + 1];     // units before the requests of thread t's part
  __shared__ Request requests[THREADS];      // all of them if there are no more than threads
  __shared__ Cursor cursors[NWARP][2];       // the item that is worked on, the item that is fetched
  __shared__ Unit infos[NWARP][4];
  __shared__ Piece pieces[2 * NWARP];        // of a warp: where an item ended that had begun before its stretch; what its stretch ended with
  __shared__ Join joins[2];
  __shared__ uint32_t items_s, most_s, plan[3];  // plan: the CTA's stretch [0, 1) of the line; units of a stretch
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  uint8_t* const buf = smem + warp * RING * S::PART;
  const uint32_t buf_at = smem_u32(buf), bar = smem_u32(&bars[warp][0]);
  if (lane < RING) {
    mbar_init(bar + 8 * lane, 1);
    fence_barrier_init();  // (by whoever made one)
  }
  if (lane < 2) pieces[2 * warp + lane].used = 0;
  if (threadIdx.x == 0) items_s = most_s = 0;
  __syncthreads();
  pdl_launch_dependents();
  pdl_wait();

  // ---- the line of units ----
  const uint32_t per = (a.n_req + THREADS - 1) / THREADS;
  const Request* known = per == 1 ? requests : nullptr;
  {
    uint32_t units = 0, items = 0, most = 0;
    for (uint32_t r = threadIdx.x * per; r < min((threadIdx.x + 1) * per, a.n_req); r++) {
      const Request q = request<NT>(a, r, blockIdx.x == 0);
      if (known) requests[r] = q;
      items += q.tiles * a.pool.n_kv_head;
      if (q.tiles) most = max(most, q.units);
      units += q.tiles * a.pool.n_kv_head * q.units;
    }
    uint32_t up = units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(FULL, up, o);
      if (lane >= o) up += x;
    }
    line[threadIdx.x + 1] = up;  // within the warp
    items = __reduce_add_sync(FULL, items);
    most = __reduce_max_sync(FULL, most);
    if (lane == 0 && items) {
      atomicAdd(&items_s, items);
      atomicMax(&most_s, most);
    }
  }
  __syncthreads();
  if (a.n_req > 32) {
    uint32_t before = 0;
    for (uint32_t w = 0; w < warp; w++) before += line[32 * (w + 1)];
    __syncthreads();
    line[threadIdx.x + 1] += before;
    __syncthreads();
  }
  // (with 32 requests or fewer the first warp's part is the line)
  const uint32_t total = line[a.n_req > 32 ? THREADS : 32], n_cta = gridDim.x;
  auto locate = [&](uint32_t x, Cursor& c) {  // the warp: unit x < total
    uint32_t at = 0;                          // the last part that begins at x or before it
    for (uint32_t i = 0; i < (a.n_req > 32 ? THREADS : 32u); i += 32) {
      const uint32_t n = __popc(__ballot_sync(FULL, line[i + lane + 1] <= x));
      at += n;
      if (n < 32) break;
    }
    if (lane == 0) {
      uint32_t left = at ? x - line[at] : x;
      for (uint32_t r = at * per; r < a.n_req; r++) {
        const Request q = known ? known[r] : request<NT>(a, r, false);
        const uint32_t n = q.tiles * a.pool.n_kv_head * q.units;
        if (left >= n) {
          left -= n;
          continue;
        }
        const uint32_t item = left / q.units;
        c.q = q;
        c.r = r;
        c.unit = left - item * q.units;
        c.head = item / q.tiles;
        c.tile = item - c.head * q.tiles;
        break;
      }
    }
    __syncwarp();
  };
  for (uint32_t r = blockIdx.x; r < a.n_req; r += n_cta) {
    const Request q = known ? known[r] : request<NT>(a, r, false);
    if (q.kv_len == 0) zero_rows<D>(a, q.q0, q.q_len);
  }
  // One item per CTA where that takes at most one round of the warps more than equal stretches, which need their pieces
  // joined; else equal stretches, of one unit per warp at least.
  uint32_t c0, c1;
  const uint32_t share = max((total + n_cta - 1) / n_cta, NWARP);
  if (items_s <= n_cta && (most_s + NWARP - 1) / NWARP <= (share + NWARP - 1) / NWARP + 1) {
    c0 = c1 = 0;
    if (blockIdx.x < items_s) {
      uint32_t left = blockIdx.x;
      for (uint32_t r = 0; r < a.n_req; r++) {
        const Request q = known ? known[r] : request<NT>(a, r, false);
        const uint32_t n = q.tiles * a.pool.n_kv_head;
        if (left < n) {
          c0 += left * q.units;
          c1 = c0 + q.units;
          break;
        }
        left -= n;
        c0 += n * q.units;
      }
    }
  } else {
    c0 = min(static_cast<uint64_t>(blockIdx.x) * share, static_cast<uint64_t>(total));
    c1 = c0 + min(share, total - c0);
  }
  if (c0 >= c1) return;  // (all threads)
  if (threadIdx.x == 0) {
    plan[0] = c0;
    plan[1] = c1;
    plan[2] = share;
  }
  const uint32_t begin = static_cast<uint64_t>(c1 - c0) * warp / NWARP, n = static_cast<uint64_t>(c1 - c0) * (warp + 1) / NWARP - begin;
  __syncthreads();

  if (n > 0) {
    Cursor &cur = cursors[warp][0], &next = cursors[warp][1];
    locate(plan[0] + begin, cur);
    if (lane == 0) next = cur;
    __syncwarp();
    Fetch f;
    uint32_t asked = 1, nb = 0, flying = 0;  // units asked for; the buffer (and its barrier) that is filled next; filled ones
    auto fetch_k = [&]() {       // of unit asked - 1
      fetch_keys<D, PAGE>(f, a, next, infos[warp][(asked - 1) & 3], buf_at + nb * S::PART, bar + 8 * nb, lane);
      if (++nb == RING) nb = 0;
      flying++;
    };
    auto fetch_v = [&]() {
      copy_pages(f.pages, f.src + HALF, HALF, buf_at + nb * S::PART, bar + 8 * nb, lane);
      if (++nb == RING) nb = 0;
      flying++;
    };
    auto next_unit = [&]() {
      asked++;
      if (f.rem > 1) {
        f.rem--;
        f.key0 += UNIT;
      } else {
        if (lane == 0) next_item<NT>(next, a, known);
        __syncwarp();
        start_item<PAGE>(f, a, next, lane);
      }
    };
    RawQueries<D, NT> raw;
    ask_queries<D, NT>(raw, a, cur.head, cur.tile * S::ROWS, cur.q.q_len * a.group, cur.q.q0, lane);
    start_item<PAGE>(f, a, next, lane);
    fetch_k();
    fetch_v();
    if (n > 1) {
      next_unit();
      fetch_k();
      if (RING == 4) fetch_v();
    }
    WarpState<D, NT> w;
    bool fresh = true, from_start = false, ok = true;
    uint32_t first = 0;          // of this piece; cur.unit is its place in the item
    uint32_t b = 0, phase = 0;   // the buffer that is worked on, the phases of the barriers' next use
    // (the lanes decide together: what follows shuffles and multiplies with the whole warp, and one lane may see the phase that another one gave up on)
    auto wait = [&]() { return __all_sync(FULL, wait_phase(bar + 8 * b, phase >> b & 1)); };
    auto done = [&]() {
      phase ^= 1u << b;
      if (++b == RING) b = 0;
      flying--;
      __syncwarp();
    };
    for (uint32_t i = 0; i < n; i++) {
      if (fresh) {
        if (i) ask_queries<D, NT>(raw, a, cur.head, cur.tile * S::ROWS, cur.q.q_len * a.group, cur.q.q0, lane);
        set_queries<D, NT>(w, raw, a, cur.tile * S::ROWS, cur.q.q_len * a.group, lane);
        from_start = cur.unit == 0;
        first = i;
        fresh = false;
      }
      float s[NT][4][4];
      ok = ok && wait();
      if (!ok) break;
      const Unit u = infos[warp][i & 3];
      const bool part = u.pages != ALL_PAGES || u.low > 0 || u.left < static_cast<int>(UNIT);
      {
        uint8_t* kb = buf + b * S::PART;
        if (part) clear_scales<D, PAGE>(kb, u.pages, 0, UNIT);
#pragma unroll
        for (int k = 0; k < 4; k++) scores16<D, NT, PAGE>(w, kb, lane, s, k, a.mantissa24);
      }
      done();
      if (RING == 3 && i + 1 < n) fetch_v();  // of unit i + 1
      if (RING == 4 && i + 2 < n) {
        next_unit();
        fetch_k();
      }
      const int q_len = cur.q.q_len;
      const bool cut = u.left - static_cast<int>(UNIT) < q_len - 1 || (a.window && u.left > static_cast<int>(a.window));
      softmax64<D, NT>(w, s, cut, u.left, cur.tile * S::ROWS, q_len, a, lane);
      ok = wait();
      if (!ok) break;
      {
        uint8_t* vb = buf + b * S::PART;
        if (part) clear_scales<D, PAGE>(vb, u.pages, u.low, u.left);
        if (cut && q_len > 1 && __any_sync(FULL, (blocks_without_numbers<D, PAGE>(vb, lane) | blocks_without_numbers<D, PAGE>(vb, lane + 32)) != 0)) {
          const uint32_t spoiled = take_no_numbers<D, NT, PAGE>(vb, u.left, cur.tile * S::ROWS, q_len, a.group, a.window);
#pragma unroll
          for (int e = 0; e < NT; e++)
#pragma unroll
            for (int i = 0; i < 2 * NB; i++)
#pragma unroll
              for (int c = 0; c < 4; c++)
                if (spoiled >> (NB * (2 * e + (c & 1)) + i / 2) & 1) w.o[e][i][c] = __int_as_float(0x7fffffff);
        }
#pragma unroll
        for (int k = 0; k < 4; k++) values16<D, NT, PAGE>(w, vb, lane, s, k, a.bias);
      }
      done();
      if (RING == 3 && i + 2 < n) {
        next_unit();
        fetch_k();
      }
      if (RING == 4 && i + 2 < n) fetch_v();

      if (u.ends || i + 1 == n) {
        // sums over the lanes of a row
#pragma unroll
        for (int e = 0; e < NT; e++)
#pragma unroll
          for (int c = 0; c < 2; c++)
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) w.l[e][c] += __shfl_xor_sync(FULL, w.l[e][c], o);
        const uint32_t row0 = cur.tile * S::ROWS, n_rows = static_cast<uint32_t>(q_len) * a.group;
        if (u.ends && from_start) {
#pragma unroll
          for (int e = 0; e < NT; e++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
              const uint32_t row = row0 + 8 * e + 2 * t + c;
              if (row >= n_rows) continue;
              const float inv = w.l[e][c] == 0.f ? 0.f : 1.f / w.l[e][c];
              uint16_t* out = out_row(a, cur.q.q0, cur.head, row);
#pragma unroll
              for (int x = 0; x < NB; x++)
                store4(a.bf, out + 32 * x + 4 * g, w.o[e][2 * x][c] * inv, w.o[e][2 * x][c + 2] * inv, w.o[e][2 * x + 1][c] * inv, w.o[e][2 * x + 1][c + 2] * inv);
            }
        } else {
          // an item's end goes to memory (the buffers are in use), the stretch's end over the buffers
          const bool last = i + 1 == n;
          float* to = last ? reinterpret_cast<float*>(buf) : scratch + (static_cast<size_t>(blockIdx.x) * NWARP + warp) * S::PARTIAL;
#pragma unroll
          for (int e = 0; e < NT; e++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
              float* p = to + (8 * e + 2 * t + c) * S::STRIDE;
#pragma unroll
              for (int x = 0; x < NB; x++)
                *reinterpret_cast<float4*>(p + 32 * x + 4 * g) = make_float4(w.o[e][2 * x][c], w.o[e][2 * x][c + 2], w.o[e][2 * x + 1][c], w.o[e][2 * x + 1][c + 2]);
              if (g == 0) *reinterpret_cast<float2*>(p + D) = make_float2(w.m[e][c], w.l[e][c]);
            }
          if (lane == 0)
            pieces[2 * warp + (last ? 1 : 0)] = Piece{1, plan[0] + begin + first - cur.unit, cur.q.units, cur.head, row0, min(S::ROWS, n_rows - row0), cur.q.q0};
        }
        fresh = true;
        if (i + 1 < n) {
          __syncwarp();  // (every lane has read the item that ends)
          if (lane == 0) next_item<NT>(cur, a, known);
          __syncwarp();
        }
      }
    }
    if (!ok) {  // the wait gave up: what is on its way comes before the buffers are given back
      if (lane == 0) reinterpret_cast<volatile uint32_t*>(a.err)[1] = 1;
      for (; flying > 0; flying--) {
        (void)wait_phase(bar + 8 * b, phase >> b & 1);
        if (++b == RING) b = 0;
      }
    }
  }
  __syncthreads();

  // ---- the CTA's pieces: joined; items that lie in this CTA alone are written ----
  float* exchange = scratch + static_cast<size_t>(n_cta) * NWARP * S::PARTIAL;
  const bool used = lane < 2 * NWARP && pieces[lane].used;
  const uint32_t start = used ? pieces[lane].start : 0, all_used = __ballot_sync(FULL, used), under = all_used & ((1u << lane) - 1);
  const uint32_t prev = __shfl_sync(FULL, start, under ? 31 - __clz(under) : 0);
  uint32_t heads = __ballot_sync(FULL, used && (!under || prev != start)), n_joins = 0, turn = 0;  // the first piece of every item
  while (heads) {
    const uint32_t i = __ffs(heads) - 1;
    heads &= heads - 1;
    const uint32_t run = all_used & ~((1u << i) - 1) & (heads ? (1u << (__ffs(heads) - 1)) - 1 : FULL), n_run = __popc(run);
    const Piece& p = pieces[i];
    const bool all = p.start >= plan[0] && p.start + p.units <= plan[1];
    const uint32_t first_cta = all ? 0 : p.start / plan[2];
    float* to = all ? nullptr : exchange + static_cast<size_t>(2 * blockIdx.x + (blockIdx.x == first_cta)) * S::PARTIAL;
    for (uint32_t row = 0; row < p.rows; row += 4) {  // the warps take the rows of all items in turn
      if (turn == warp)
        join_rows4<D, NT>(a, p, row, n_run, [&](uint32_t k) {
          const uint32_t x = __fns(run, 0, k + 1);
          return (x & 1) ? reinterpret_cast<const float*>(smem + (x >> 1) * (RING * S::PART)) : scratch + (static_cast<size_t>(blockIdx.x) * NWARP + (x >> 1)) * S::PARTIAL;
        }, to, lane);
      if (++turn == NWARP) turn = 0;
    }
    if (!all) {  // an item that began before the stretch, one that goes on behind it
      if (threadIdx.x == 0) joins[n_joins] = Join{i, first_cta, (p.start + p.units - 1) / plan[2] - first_cta + 1, 0};
      n_joins++;
    }
  }
  if (n_joins == 0) return;  // (all threads)

  // ---- items of several CTAs: the one that comes last joins them ----
  __syncthreads();
  if (threadIdx.x < n_joins) {
    Join& j = joins[threadIdx.x];
    j.last = arrive(&counters[j.first_cta]) == j.n - 1;
    if (j.last) counters[j.first_cta] = 0;  // for the next launch
  }
  __syncthreads();
  turn = 0;
  for (uint32_t q = 0; q < n_joins; q++) {
    const Join j = joins[q];
    if (!j.last) continue;
    const float* from = exchange + static_cast<size_t>(2 * j.first_cta) * S::PARTIAL;
    const Piece& p = pieces[j.piece];
    auto part = [&](uint32_t k) { return from + (2 * k + (k == 0)) * S::PARTIAL; };
    const uint32_t step = j.n <= 4 ? 4 : 1;
    for (uint32_t row = 0; row < p.rows; row += step) {
      if (turn == warp) {
        if (step == 4) join_rows4<D, NT>(a, p, row, j.n, part, nullptr, lane);
        else join_row<D, NT>(a, p, row, j.n, part, lane);
      }
      if (++turn == NWARP) turn = 0;
    }
  }
}

// f(kernel, shape) for the instance of (head_dim, rows of an item, page).
template <typename F>
cudaError_t with_kernel(uint32_t head_dim, bool two, uint32_t page, F f) {
  auto by_page = [&](auto d, auto nt) {
    constexpr int D = decltype(d)::value, NT = decltype(nt)::value;
    return page == 16 ? f(kv4_attention_kernel<D, NT, 16>, Shape<D, NT>()) : page == 32 ? f(kv4_attention_kernel<D, NT, 32>, Shape<D, NT>()) : f(kv4_attention_kernel<D, NT, 64>, Shape<D, NT>());
  };
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  if (head_dim == 128) return two ? by_page(std::integral_constant<int, 128>(), I2()) : by_page(std::integral_constant<int, 128>(), I1());
  return two ? by_page(std::integral_constant<int, 64>(), I2()) : by_page(std::integral_constant<int, 64>(), I1());
}

}  // namespace

cudaError_t bp_kv4_attention_init(bp_paged_ctx* c) {
  cudaError_t e = cudaSuccess;
  for (uint32_t i = 0; i < 12 && e == cudaSuccess; i++)
    e = with_kernel(i & 1 ? 128 : 64, i & 2, 16u << (i >> 2), [](auto kernel, auto shape) {
      return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(shape.SMEM));
    });
  if (e != cudaSuccess) return e;
  // a piece per warp and two per CTA, of the instance that needs most
  size_t floats = 0;
  for (uint32_t i = 0; i < 4; i++)
    (void)with_kernel(i & 1 ? 128 : 64, i & 2, 16, [&](auto, auto shape) {
      const size_t need = static_cast<size_t>(c->sm_count) * (shape.NWARP + 2) * shape.PARTIAL;
      if (need > floats) floats = need;
      return cudaSuccess;
    });
  e = cudaMalloc(&c->partials, floats * sizeof(float));
  if (e != cudaSuccess) return e;
  e = cudaMalloc(&c->counters, static_cast<size_t>(c->sm_count) * sizeof(uint32_t));
  if (e != cudaSuccess) return e;
  return cudaMemset(c->counters, 0, static_cast<size_t>(c->sm_count) * sizeof(uint32_t));
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
  a.table_stride = in.table_stride;
  a.table_pages = in.table_stride < (0x7fffffffu >> pool.log_page) ? in.table_stride : (0x7fffffffu >> pool.log_page);
  a.window = in.window < in.max_kv ? in.window : 0;  // (nobody has more keys)
  a.scale_log2 = in.scale * 1.4426950408889634f;
  int exponent = 0;
  const float fraction = frexpf(fabsf(a.scale_log2), &exponent);
  const bool split = fraction > 0.f && fraction < 1.f;  // (not of 0 and infinity)
  a.mantissa = split ? 2.f * fraction : 1.f;
  a.mantissa24 = a.mantissa * 0x1p24f;
  a.power = split ? ldexpf(1.f, exponent - 1) : fraction;
  a.bias = 0x64006400u;
  a.bf = bf;
  a.q_vec = reinterpret_cast<uintptr_t>(in.q.data) % 16 == 0 && in.q.tok_stride % 8 == 0 && in.q.head_stride % 8 == 0;
  // Which kernel. Here the codes are expanded once per 16 rows (tokens x query heads per KV head) of a request, there once for up to 128, with some 14 us
  // for an item's beginning and end. us, this kernel / the other one:
  //   head_dim 128, 32 / 8 heads         16 rows  32 rows  48 rows     head_dim 64, 40 / 8 heads    15 rows  30 rows  40 rows  50 rows
  //   16 requests of 4096 keys           41/75    68/75    97/76                                    28/60    47/61    60/61    78/61
  //   the same, window 1024              19/36    31/36    38/36                                    15/28    24/29    26/29    30/29
  //   64 requests of 1000 keys           46/85    78/87    113/88                                   29/70    50/70    65/71    85/72
  //   1 request of 30000 keys            33/64    48/63    62/64                                    27/45    36/45    42/45    50/45
  // and as much apart with 2, 4 and 8 requests of 4096 keys and with 2 KV heads; so 32 rows is the line for both.
  const uint64_t rows = static_cast<uint64_t>(a.max_q) * a.group;
  // (Without any key there are only zeros to write, and there may be no pool: this kernel looks at none.)
  if (a.max_kv != 0 && rows > 32) return bp_launch_kv4_prefill(c, s, head_dim, a);
  return with_kernel(head_dim, a.max_q * a.group > 8, pool.page, [&](auto kernel, auto shape) {
    return bp_launch(true, kernel, dim3(c->sm_count), dim3(shape.THREADS), shape.SMEM, s, a, c->partials, c->counters);
  });
}
