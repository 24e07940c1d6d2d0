// Attention of many queries per request over a paged 4-bit cache, on the 5th-generation tensor cores (include/bonsai_paged.h;
// few queries: bp_kv4_attention.cu).
//
// An item is one KV head of one request and NQ query tiles of 128 rows (a row is a query head of a token). Keys come in tiles of
// 64. Roles of a CTA, one CTA per SM:
//   expanders (8 warps)     codes -> f16 operand tiles in shared memory, K and V, once for all query tiles of the item. Every
//                           value is an f16 number (the format's choice of m and d): nothing rounds. The next tile's codes are
//                           on their way in registers meanwhile. Places that hold no key of the request become zeros.
//   S issuer X (1 thread)   S_X = Q_X K^T (tcgen05.mma kind::f16, M 128, N 64) into one of two 64-column buffers in TMEM
//   softmax X (4 warps)     thread = row = TMEM lane: masks, running maximum and sum, P as f16 over the tile's S buffer; O_X is
//                           rescaled in TMEM only when a row's maximum grew by more than 2^5 (P stays below 2^15 meanwhile)
//   O issuer X (1 thread)   O_X += P_X V (P from TMEM as the A operand, V as the MN-major B operand)
// The key tiles of all items lie in one line, of which every CTA takes an equal stretch; an item that lies in several CTAs is joined by the
// one that comes last, in the order of its keys (as in bp_kv4_attention.cu). In PARTS (prefixes that several requests have in common, and keys behind them) nobody joins: rows and
// pieces of rows go to memory as 32-bit records, through the dead Q tile, and bp_kv4_shared.cu joins them. Every wait is bounded; a timeout sets the context's error word and
// the CTA winds down and frees its TMEM.
//
// P is f16 because V is (see bp_kv4_attention.cu).
//
// Bound by the softmax warps: of the some 2340 cycles of a tile of 64 keys and 256 rows (clocks read in a copy of the kernel) they wait 250 for S, while the S issuers wait
// 1600 for a free buffer, the O issuers 1770 for P, and the expanders 490 for free slots. The row exponentials alone take 1024 cycles at 16 per cycle and SM, the MMAs
// would take about 1450 at the measured rate of a library product. 2048 queries behind 32768 keys, 32 / 8 heads of 128: 1.21 ms, 881 TFLOP/s, 54 % of that rate
// (floor 0.65 ms). Four expander warps whose page ids were waited for took 1.39 ms; eight of them, with two softmax threads per row, 1.38; with one softmax
// thread per row 1.25; with whole lines read and one barrier per slot 1.23. 4 requests of up to 512 queries behind up to 4099 keys: 98 us (floor 32): a tile costs the
// same, beginning and ending an item about 14 us; before the line weighted items and the partial results had whole-warp accesses it was 216. 4 chunks of up to 512 queries with
// 16384 keys in common and up to 1030 of their own: 434 us, 836 TFLOP/s (BEHIND; in PARTS, with 20 to join them, 444). One query tile of 128 rows (64 tokens behind 8191 keys in common, 90 CTAs): 33 us, 1.0 to 1.15
// per key tile (2000 cycles: an expander warp takes 1900 for it, nearly all of them one instruction waiting for another, the softmax 1300), 1.3 before the first item is
// found, 1.8 for the queries, 2 from there to the first scores, 2.4 to write the rows. (Tried: two key tiles per turn of the expanders, 280 bytes of registers spilled: 45 us; K and V of a tile
// behind one fence: the same; every 2nd or 4th pair of exponentials by a polynomial on the FMA units: chunks 536 and 487 us instead of 450.)
#include <type_traits>

#include "bp_kv4_attention.cuh"

namespace {

using namespace bp;
using namespace bp::kv4;

constexpr uint32_t BM = 128, BN = 64;  // query rows of a tile, keys of a tile
constexpr uint32_t SLOTS = 4;          // K and V tiles in shared memory
// Tiles of which some rows of an item see only a part: its rows are 256 tokens at most, so these are 5 tiles at each end of the keys that they see; where a
// window is so short that no tile lies between the two ends, the two overlap or are less than two tiles apart: 11 tiles.
constexpr uint32_t MIXED = 11;
// What beginning and ending an item costs, in key tiles. (In parts its rows are 32-bit records.) us in parts, 32 / 8 heads of 128 and 40 / 8 of 64; no number is the best for all, 10 is never
// more than 16 % from it:
//   requests x tokens, prefix, own   16 x 16, 8192, 600   16 x 40, 4096, 400   8 x 64, 16384, 700   32 x 40, 1000, 1000   32 x 8, 4096, 500 (64 dims)
//   cost 4                           86 / 79              110 / 106            238 / 231            139 / 120             69
//   6                                86 / 81              102 / 99             215 / 210            137 / 119             72
//   10                               90 / 85              103 / 100            192 / 208            137 / 121             80
//   14                               96 / 90              111 / 102            196 / 215            134 / 120             89
//   20                               103 / 96             115 / 108            201 / 224            132 / 120             93
template <int MODE>
constexpr uint32_t ITEM_COST = MODE == PARTS ? BP_KV4_ITEM_COST_IN_PARTS : 6;
constexpr float GROW = 5.f;            // log2 by which a maximum may grow before O is rescaled; P_UP + GROW stays below 16

template <int D, uint32_t NQ>
struct Shape {
  static constexpr uint32_t ROWS = BM * NQ;
  static constexpr uint32_t Q_B = BM * D * 2, KV_B = BN * D * 2;          // operand tiles: D / 64 chunks of rows of 128 bytes
  static constexpr uint32_t OFF_K = NQ * Q_B, OFF_V = OFF_K + SLOTS * KV_B, SMEM = OFF_V + SLOTS * KV_B + 1024;
  static constexpr uint32_t TM_O = 128 * NQ, TMEM_COLS = 256 * NQ;        // S_X at 128 X, O_X at TM_O + 128 X
  static constexpr uint32_t FIRST_EXPANDER = 4, FIRST_SOFTMAX = 12;       // warps 0, 1: O issuers, 2, 3: S issuers
  static constexpr uint32_t NWARP = FIRST_SOFTMAX + 4 * NQ, THREADS = 32 * NWARP;
  static constexpr uint32_t PARTIAL = ROWS * (D + 2);                     // floats of a partial result: o as fours [dims / 4][row], (m, l) [row]
  static constexpr uint32_t PIECE = ROWS * RECORD<D>;                     // the same in PARTS: a record per row
};

struct Request {
  int q0, q_len, kv_len;
  uint32_t rows, causal;
  int before;       // BEHIND: keys of its prefix, which come before its own kv_len
  uint32_t prefix;
};
template <int MODE>
__device__ __forceinline__ Request request(const AttnArgs& a, uint32_t r, bool report) {
  Request q;
  const Lengths n = lengths_of<MODE>(a, r, report);
  q.q0 = n.q0;
  q.q_len = n.q_len;
  q.kv_len = n.kv_len;
  q.rows = static_cast<uint32_t>(q.q_len) * a.group;
  q.causal = is_causal<MODE>(a, r);
  q.before = 0;
  q.prefix = 0;
  if (MODE == BEHIND && a.n_prefix) {
    uint32_t lo = 0, hi = a.n_prefix + 1;  // the last one that has begun is lo, if any has
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) >> 1;
      if (a.prefix_start[mid] <= static_cast<int>(r)) lo = mid;
      else hi = mid;
    }
    if (lo < a.n_prefix && a.prefix_start[lo] <= static_cast<int>(r)) {
      q.prefix = lo;
      q.before = min(max(a.prefix_len[lo], 0), static_cast<int>(min(a.max_prefix, a.prefix_pages << a.pool.log_page)));
    }
  }
  return q;
}
// Keys [low, high) that the rows [row0, row0 + rows) of a request see, of all of them together; key tiles from low's on, one at least (its
// rows have zeros to write).
struct Keys {
  int low, high;
  int all_from, all_to;  // every row sees the keys in between
  uint32_t tiles;
  __device__ int first() const { return low & ~static_cast<int>(BN - 1); }
};
template <int MODE>
__device__ __forceinline__ Keys keys_of(const AttnArgs& a, const Request& q, uint32_t row0, uint32_t rows) {
  Keys k;
  if (MODE == PARTS && !q.causal) {
    k.low = k.all_from = 0;
    k.high = k.all_to = q.kv_len;
    k.tiles = max((static_cast<uint32_t>(q.kv_len) + BN - 1) / BN, 1u);
    return k;
  }
  const int t0 = static_cast<int>(row0 / a.group), t1 = static_cast<int>((min(row0 + rows, q.rows) - 1) / a.group), past = q.kv_len - q.q_len;
  k.high = max(past + t1 + 1, 0);
  k.low = first_seen(past + t0 + 1, a.window);
  k.all_from = first_seen(past + t1 + 1, a.window);
  k.all_to = past + t0 + 1;
  if (MODE == BEHIND) {
    k.low = k.all_from = 0;
    k.high += q.before;
    k.all_to = q.before + max(k.all_to, 0);
  }
  k.tiles = max((static_cast<uint32_t>(k.high - k.first()) + BN - 1) / BN, 1u);
  return k;
}

// A place in the line, in which an item takes ITEM_COST places before those of its tiles: item (r, x, head) of `keys.tiles` tiles, tile
// `at` of it, the item's first tile lying at place `start`.
struct Cursor {
  Request q;
  Keys keys;
  uint32_t r, x, head, at, start;
};

// Byte offset of 16-byte unit u of row r in an operand tile of `rows` rows: chunks of 64 dims, 128-byte swizzle.
__device__ __forceinline__ uint32_t oper_off(uint32_t rows, uint32_t r, uint32_t u) { return (u >> 3) * (rows * 128) + r * 128 + (((u & 7) ^ (r & 7)) << 4); }

// A quarter of the codes of one token's K and V and their scales; `id` is a page of the
// pool.
template <int D>
struct Raw {
  static constexpr int NB = D / 32;
  uint32_t k[NB], v[NB], kd[NB / 2], km[NB / 2], vd[NB / 2], vm[NB / 2];
};
template <int D>
__device__ __forceinline__ void ask(Raw<D>& w, const AttnArgs& a, uint32_t id, int key, uint32_t head, uint32_t quarter) {
  using L = PoolLayout<D>;
  constexpr int NB = D / 32;
  const uint32_t page = a.pool.page, tok = static_cast<uint32_t>(key) & (page - 1);
  const uint8_t* k = a.pool.data + (static_cast<uint64_t>(id) * a.pool.n_kv_head + head) * (page * L::TOK);
  const uint8_t* v = k + L::v(page);
  const uint32_t scales = L::kd(page) + tok * 2 * NB, kv = tok * L::ROW, gap = page * 2 * NB;
  if constexpr (NB == 4) {
    const uint4 x = *reinterpret_cast<const uint4*>(k + kv + 16 * quarter), y = *reinterpret_cast<const uint4*>(v + kv + L::v16(tok, 2 * quarter, 0));
    w.k[0] = x.x, w.k[1] = x.y, w.k[2] = x.z, w.k[3] = x.w;
    w.v[0] = y.x, w.v[1] = y.y, w.v[2] = y.z, w.v[3] = y.w;
    const uint2 e = *reinterpret_cast<const uint2*>(k + scales), f = *reinterpret_cast<const uint2*>(k + scales + gap);
    const uint2 g = *reinterpret_cast<const uint2*>(v + scales), h = *reinterpret_cast<const uint2*>(v + scales + gap);
    w.kd[0] = e.x, w.kd[1] = e.y, w.km[0] = f.x, w.km[1] = f.y;
    w.vd[0] = g.x, w.vd[1] = g.y, w.vm[0] = h.x, w.vm[1] = h.y;
  } else {
    const uint2 x = *reinterpret_cast<const uint2*>(k + kv + 8 * quarter), y = *reinterpret_cast<const uint2*>(v + kv + 8 * quarter);
    w.k[0] = x.x, w.k[1] = x.y;
    w.v[0] = y.x, w.v[1] = y.y;
    w.kd[0] = *reinterpret_cast<const uint32_t*>(k + scales), w.km[0] = *reinterpret_cast<const uint32_t*>(k + scales + gap);
    w.vd[0] = *reinterpret_cast<const uint32_t*>(v + scales), w.vm[0] = *reinterpret_cast<const uint32_t*>(v + scales + gap);
  }
}
// What a thread of the expanders has asked for: the codes of the tile that `key` lies in, the next two page ids. TWO: the first `before` keys lie in other pages, of `first`.
template <int D, bool TWO>
struct Ahead {
  Raw<D> raw;
  int key;
  uint32_t id, id_next;
  bool there;
  // Page ids are asked for two tiles ahead and looked at one tile ahead, when the codes are asked for: nothing here waits for memory.
  // A token that holds no key of the request (or lies in a page outside the pool) gets page 0's codes, and zeros for its scales.
  static __device__ __forceinline__ bool has_key(const Keys& keys, int key) { return key >= keys.low && key < keys.high; }
  static __device__ __forceinline__ uint32_t ask_id(const AttnArgs& a, const Keys& keys, const int32_t* table, const int32_t* first, int before, int key) {
    return !has_key(keys, key) ? 0u : static_cast<uint32_t>(TWO && key < before ? first[key >> a.pool.log_page] : table[(TWO ? key - before : key) >> a.pool.log_page]);
  }
  __device__ __forceinline__ void ask_codes(const AttnArgs& a, const Keys& keys, int before, uint32_t head, uint32_t quarter) {
    there = has_key(keys, key) && id < a.pool.n_pages;
    if (has_key(keys, key) && !there) note_range(a.err);
    ask<D>(raw, a, there ? id : 0u, TWO && key >= before ? key - before : key, head, quarter);
  }
};
// Eight codes at bits 4 i of both halves -> four words of two f16 values m + d q.
__device__ __forceinline__ uint4 expand8(uint32_t w, __half2 d, __half2 m, uint32_t bias) {
  const __half2 off = __float2half2_rn(-1024.f), off16 = __float2half2_rn(-64.f), sixteenth = __float2half2_rn(0.0625f);
  const uint32_t y = w >> 8;
  return make_uint4(u2(__hfma2(__hadd2(biased(w, 0x000f000fu, bias), off), d, m)), u2(__hfma2(__hfma2(biased(w, 0x00f000f0u, bias), sixteenth, off16), d, m)),
                    u2(__hfma2(__hadd2(biased(y, 0x000f000fu, bias), off), d, m)), u2(__hfma2(__hfma2(biased(y, 0x00f000f0u, bias), sixteenth, off16), d, m)));
}
// One token's quarter into the K or V operand tile. A V word's halves are dims i and i + 4 of a group of eight: that order stays, and
// the end of an item puts it right.
template <int D, bool V>
__device__ __forceinline__ void put(const Raw<D>& w, uint8_t* tile, uint32_t row, uint32_t quarter, uint32_t bias) {
  constexpr int NB = D / 32;
#pragma unroll
  for (int b = 0; b < NB; b++) {
    const uint32_t sel = b & 1 ? 0x3232u : 0x1010u;
    const __half2 d = h2(prmt(V ? w.vd[b >> 1] : w.kd[b >> 1], 0, sel)), m = h2(prmt(V ? w.vm[b >> 1] : w.km[b >> 1], 0, sel));
    const uint32_t codes = V ? prmt(w.v[b >> 1], w.v[NB / 2 + (b >> 1)], b & 1 ? 0x7632u : 0x5410u) : w.k[b];
    *reinterpret_cast<uint4*>(tile + oper_off(BN, row, 4 * b + quarter)) = expand8(codes, d, m, bias);
  }
}
// Column of O that holds dim i of a group of eight.
__host__ __device__ constexpr int column_of(int i) { return i < 4 ? 2 * i : 2 * (i - 4) + 1; }

// What several CTAs have of one item: the first of them, how many.
struct Join {
  uint32_t first_cta, n, last;
};

// `rows` staged output rows (16-byte chunks xor-ed with the row) from row0 of a request on to memory, by `n` threads.
template <int D>
__device__ __forceinline__ void store_rows(const AttnArgs& a, int q0, uint32_t head, uint32_t row0, uint32_t rows, const uint8_t* stage, uint32_t me, uint32_t n) {
  constexpr uint32_t U = D / 8;
#pragma unroll 4
  for (uint32_t k = me; k < rows * U; k += n) {
    const uint32_t r = k / U, u = k % U;
    const uint4 v = *reinterpret_cast<const uint4*>(stage + r * (D * 2) + ((u ^ (r & (U - 1))) << 4));
    uint16_t* out = out_row(a, q0, head, row0 + r) + 8 * u;
    if ((reinterpret_cast<uintptr_t>(out) & 15) == 0) {
      *reinterpret_cast<uint4*>(out) = v;
    } else {
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 8; e++) out[e] = static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1)));
    }
  }
}

template <int D, uint32_t NQ, int MODE>
__global__ void __launch_bounds__(Shape<D, NQ>::THREADS, 1) kv4_prefill_kernel(const __grid_constant__ AttnArgs a, float* __restrict__ scratch, uint32_t* __restrict__ counters) {
  using S = Shape<D, NQ>;
  constexpr uint32_t THREADS = S::THREADS;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t k_full[SLOTS], v_full[SLOTS], k_empty[SLOTS], v_empty[SLOTS], pv_done[NQ][SLOTS];
  __shared__ __align__(8) uint64_t s_ready[NQ][2], p_ready[NQ][2], p_free[NQ][2], o_done[NQ], drained;
  // Values that are no numbers, in tiles of which the item's rows see different keys (0 times such a value is not 0): such blocks become zeros in
  // V, `bad` has them by key (a bit per block), and a piece's end writes them over in the rows that see them.
  __shared__ __align__(16) uint8_t bad[MIXED][BN];
  __shared__ float row_scale[S::ROWS];  // the softmax scale in log2 units over the power of two of a row's queries
  __shared__ uint32_t line[THREADS + 1];
  __shared__ Request requests[THREADS];  // all of them if there are no more than threads
  __shared__ float* records[S::ROWS];    // PARTS: where the rows go
  __shared__ Cursor cur;
  __shared__ Join join_s;
  __shared__ uint32_t tmem_base_s;
  __shared__ volatile uint32_t abort_s;

  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < SLOTS; i++) {
      mbar_init(smem_u32(&k_full[i]), 8);
      mbar_init(smem_u32(&v_full[i]), 8);
      mbar_init(smem_u32(&k_empty[i]), NQ);
      mbar_init(smem_u32(&v_empty[i]), NQ);
      for (uint32_t x = 0; x < NQ; x++) mbar_init(smem_u32(&pv_done[x][i]), 1);
    }
    for (uint32_t x = 0; x < NQ; x++) {
      for (uint32_t b = 0; b < 2; b++) {
        mbar_init(smem_u32(&s_ready[x][b]), 1);
        mbar_init(smem_u32(&p_ready[x][b]), 4);
        mbar_init(smem_u32(&p_free[x][b]), 1);
      }
      mbar_init(smem_u32(&o_done[x]), 1);
    }
    abort_s = 0;
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(smem_u32(&tmem_base_s), S::TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_s;
  if (!(MODE == PARTS && a.first)) pdl_launch_dependents();
  pdl_wait();
  if (MODE == PARTS && a.first) pdl_launch_dependents();

  // After one wait has given up no other one waits.
  auto waitx = [&](uint64_t* bar, uint32_t parity) {
    if (mbar_test(smem_u32(bar), parity)) return true;
    if (!abort_s && wait_phase(smem_u32(bar), parity, &abort_s)) return true;
    if (!abort_s) {
      abort_s = 1;
      reinterpret_cast<volatile uint32_t*>(a.err)[1] = 1;
    }
    return false;
  };

  if (MODE == BEHIND && blockIdx.x == 0) {  // what is wrong with the prefixes is reported
    for (uint32_t g = threadIdx.x; g < a.n_prefix; g += THREADS) {
      const int from = a.prefix_start[g], to = a.prefix_start[g + 1];
      if (from < 0 || to < from || to > static_cast<int>(a.n_own) || a.prefix_len[g] > static_cast<int>(min(a.max_prefix, a.prefix_pages << a.pool.log_page))) note_range(a.err);
    }
  }
  // ---- the line of key tiles, and this CTA's stretch [c0, c1) of it ----
  const uint32_t per = (a.n_req + THREADS - 1) / THREADS;
  auto tiles_of = [&](const Request& q) {  // of all items of a request
    uint32_t n = 0;
    for (uint32_t row0 = 0; row0 < q.rows; row0 += S::ROWS) n += keys_of<MODE>(a, q, row0, S::ROWS).tiles + ITEM_COST<MODE>;
    return n * a.pool.n_kv_head;
  };
  {
    uint32_t units = 0;
    for (uint32_t r = threadIdx.x * per; r < min((threadIdx.x + 1) * per, a.n_req); r++) {
      const Request q = request<MODE>(a, r, blockIdx.x == 0);
      if (per == 1) requests[r] = q;
      units += tiles_of(q);
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(FULL, units, o);
      if (lane >= o) units += x;
    }
    line[threadIdx.x + 1] = units;  // within the warp
    __syncthreads();
    uint32_t before = 0;
    for (uint32_t w = 0; w < warp; w++) before += line[32 * (w + 1)];
    __syncthreads();
    line[threadIdx.x + 1] += before;
    if (threadIdx.x == 0) line[0] = 0;
    __syncthreads();
  }
  const uint32_t total = line[THREADS], share = (total + gridDim.x - 1) / gridDim.x;
  const uint32_t c0 = min(static_cast<uint64_t>(blockIdx.x) * share, static_cast<uint64_t>(total)), c1 = c0 + min(share, total - c0);
  auto request_of = [&](uint32_t r) { return per == 1 ? requests[r] : request<MODE>(a, r, false); };
  uint32_t at = 0;  // (warp 0)
  if (warp == 0 && c0 < c1) {
    for (uint32_t i = 0; i < THREADS; i += 32) {
      const uint32_t n = __popc(__ballot_sync(FULL, line[i + lane + 1] <= c0));
      at += n;
      if (n < 32) break;
    }
  }
  if (threadIdx.x == 0 && c0 < c1) {
    uint32_t left = c0 - line[at];
    bool found = false;
    for (uint32_t r = at * per; r < a.n_req && !found; r++) {
      const Request q = request_of(r);
      for (uint32_t x = 0; x * S::ROWS < q.rows; x++) {
        const Keys k = keys_of<MODE>(a, q, x * S::ROWS, S::ROWS);
        const uint32_t places = k.tiles + ITEM_COST<MODE>, n = places * a.pool.n_kv_head;
        if (left < n) {
          const uint32_t head = left / places, in = left - head * places;
          cur = Cursor{q, k, r, x, head, in > ITEM_COST<MODE> ? in - ITEM_COST<MODE> : 0, c0 - in + ITEM_COST<MODE>};
          found = true;
          break;
        }
        left -= n;
      }
    }
  }
  __syncthreads();

  // Barrier phases count on across items: done = key tiles so far, pieces = pieces so far.
  uint32_t done = 0, pieces = 0;
  for (uint32_t pos = c0; pos < c1;) {
    pos = max(pos, cur.start);
    if (pos >= c1) break;  // (the stretch ends before the item's first tile)
    const Request q = cur.q;
    const Keys keys = cur.keys;
    const uint32_t head = cur.head, row0 = cur.x * S::ROWS, first = cur.at, n = min(keys.tiles - first, c1 - pos);
    const uint32_t start = cur.start;
    const int key_first = keys.first() + static_cast<int>(first * BN);
    // the piece's tiles [plain0, plain0 + plain_n) are seen whole by every row
    const uint32_t plain0 = static_cast<uint32_t>(max(keys.all_from - key_first + static_cast<int>(BN) - 1, 0)) / BN;
    const uint32_t plain_n = static_cast<uint32_t>(max((keys.all_to - key_first) / static_cast<int>(BN) - static_cast<int>(plain0), 0));
    // the expanders' first codes are on their way while the queries come (where there are registers for both)
    Ahead<D, MODE == BEHIND> ahead;
    const bool expands = warp >= S::FIRST_EXPANDER && warp < S::FIRST_SOFTMAX;
    const int before = MODE == BEHIND ? q.before : 0;
    const int32_t* first_table = MODE == BEHIND ? a.prefix_table + static_cast<size_t>(q.prefix) * a.prefix_stride : nullptr;
    auto ask_first = [&]() {
      const int32_t* table = pages_of<MODE>(a, cur.r, head);
      ahead.key = key_first + static_cast<int>(8 * (warp - S::FIRST_EXPANDER) + (lane & 7));
      ahead.id = ahead.ask_id(a, keys, table, first_table, before, ahead.key);
      ahead.id_next = n > 1 ? ahead.ask_id(a, keys, table, first_table, before, ahead.key + static_cast<int>(BN)) : 0u;
      ahead.ask_codes(a, keys, before, head, lane >> 3);
    };
    if (NQ == 1 && expands) ask_first();
    // ---- queries -> f16, each row times its power of two ----
    {
      constexpr uint32_t U = D / 8, ITERS = (S::ROWS * U + THREADS - 1) / THREADS;
      static_assert(THREADS % U == 0 && (S::ROWS * U) % 32 == 0, "rows are groups of U lanes");
      uint4 raw[ITERS];  // every load is on its way before the first is used
#pragma unroll
      for (uint32_t k = 0; k < ITERS; k++) {
        const uint32_t i = threadIdx.x + k * THREADS, r = min(row0 + min(i / U, S::ROWS - 1), q.rows - 1), u = i % U;
        const uint16_t* p = a.q.data + static_cast<int64_t>(q.q0 + r / a.group) * a.q.tok + static_cast<int64_t>(head * a.group + r % a.group) * a.q.head + 8 * u;
        if (a.q_vec) {
          raw[k] = *reinterpret_cast<const uint4*>(p);
        } else {
          uint32_t h[8];
#pragma unroll
          for (int e = 0; e < 8; e++) h[e] = p[e];
          raw[k] = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
        }
      }
#pragma unroll
      for (uint32_t k = 0; k < ITERS; k++) {
        const uint32_t i = threadIdx.x + k * THREADS, r = i / U, u = i % U;
        if (i >= S::ROWS * U) break;  // (whole warps)
        if (row0 + r >= q.rows) raw[k] = make_uint4(0, 0, 0, 0);
        float x[8], big = 0.f;
        if (a.bf) unpack8<true>(raw[k], x);
        else unpack8<false>(raw[k], x);
#pragma unroll
        for (int e = 0; e < 8; e++) big = fmaxf(big, fabsf(x[e]));
#pragma unroll
        for (uint32_t o = 1; o < U; o <<= 1) big = fmaxf(big, __shfl_xor_sync(FULL, big, o));
        const RowPower power = RowPower::of(big);
        const float up = copysignf(power.up(), a.scale_log2);
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] *= up;
        *reinterpret_cast<uint4*>(smem + (r / BM) * S::Q_B + oper_off(BM, r % BM, u)) = pack8<false>(x);
        // (never 0: a masked score, -infinity, stays what it is)
        if (u == 0) row_scale[r] = fmaxf(fabsf(a.scale_log2) * power.down(), 1e-37f);
      }
    }
    fence_proxy_async();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();

    if (warp < 2) {
      // ---------------- O_X += P_X V ----------------
      const uint32_t x = warp;
      if (x < NQ && elect_one()) {
        constexpr uint32_t IDESC = umma_idesc(1, 0, 0, 0, 1, BM, D);              // f32 += f16 (TMEM) x f16 (MN-major)
        const uint64_t dmn = umma_desc_sw128(0, BN * 128, 1024);                  // the next 64 dims a chunk on, 8 keys 1 KB
        const uint32_t s_col = tmem + x * 128, o_col = tmem + S::TM_O + x * 128;
        for (uint32_t i = 0; i < n; i++) {
          const uint32_t c = done + i, s = c % SLOTS, b = c & 1;
          if (!waitx(&p_ready[x][b], (c >> 1) & 1) || !waitx(&v_full[s], (c / SLOTS) & 1)) break;
          tc_fence_after();
          const uint64_t vb = dmn + ((smem_base + S::OFF_V + s * S::KV_B) >> 4);
#pragma unroll
          for (uint32_t ks = 0; ks < BN / 16; ks++) umma_f16_ts(o_col, s_col + 64 * b + 8 * ks, vb + ks * (16 * 128 >> 4), IDESC, (i | ks) ? 1u : 0u);
          umma_commit(smem_u32(&p_free[x][b]));
          umma_commit(smem_u32(&pv_done[x][s]));
          umma_commit(smem_u32(&v_empty[s]));
        }
        umma_commit(smem_u32(&o_done[x]));
      }
    } else if (warp < S::FIRST_EXPANDER) {
      // ---------------- S_X = Q_X K^T, up to two tiles ahead of P V ----------------
      const uint32_t x = warp - 2;
      if (x < NQ && elect_one()) {
        constexpr uint32_t IDESC = umma_idesc(1, 0, 0, 0, 0, BM, BN);
        const uint64_t dk = umma_desc_sw128(0, 16, 1024);
        const uint64_t qa = dk + ((smem_base + x * S::Q_B) >> 4);
        for (uint32_t i = 0; i < n; i++) {
          const uint32_t c = done + i, s = c % SLOTS, b = c & 1;
          if (!waitx(&k_full[s], (c / SLOTS) & 1) || (c >= 2 && !waitx(&p_free[x][b], ((c >> 1) - 1) & 1))) break;
          tc_fence_after();
          const uint64_t kb = dk + ((smem_base + S::OFF_K + s * S::KV_B) >> 4);
#pragma unroll
          for (uint32_t ks = 0; ks < D / 16; ks++)  // chunk ks / 4, 32 bytes per step inside it
            umma_f16(tmem + x * 128 + 64 * b, qa + (ks >> 2) * (BM * 128 >> 4) + (ks & 3) * 2, kb + (ks >> 2) * (BN * 128 >> 4) + (ks & 3) * 2, IDESC, ks);
          umma_commit(smem_u32(&s_ready[x][b]));
        }
      }
    } else if (warp < S::FIRST_SOFTMAX) {
      // ---------------- codes -> operand tiles ----------------
      const uint32_t quarter = lane >> 3, row = 8 * (warp - S::FIRST_EXPANDER) + (lane & 7);  // a warp: all of eight tokens, eight rows per 16-byte phase
      const int32_t* table = pages_of<MODE>(a, cur.r, head);
      if (NQ != 1) ask_first();
      for (uint32_t i = 0; i < n; i++) {
        const uint32_t c = done + i, s = c % SLOTS;
        const bool mixed = i - plain0 >= plain_n;
        Raw<D> mine = ahead.raw;
        const bool there = ahead.there;
        if (!there || mixed) {
          uint32_t found = 0;
#pragma unroll
          for (int e = 0; e < D / 64; e++) {
            const uint32_t two = no_numbers(mine.vd[e], mine.vm[e]), keep = (two & 1 ? 0u : 0xffffu) | (two & 2 ? 0u : 0xffff0000u);
            if (!there) mine.kd[e] = mine.km[e] = 0;
            mine.vd[e] &= there ? keep : 0u;
            mine.vm[e] &= there ? keep : 0u;
            found |= two << (2 * e);
          }
          if (mixed && quarter == 0) bad[i < plain0 ? i : i - plain_n][row] = there ? static_cast<uint8_t>(found) : 0;
        }
        ahead.key += BN;
        ahead.id = ahead.id_next;
        if (i + 1 < n) ahead.ask_codes(a, keys, before, head, quarter);
        if (i + 2 < n) ahead.id_next = ahead.ask_id(a, keys, table, first_table, before, ahead.key + static_cast<int>(BN));
        if (c >= SLOTS && !__all_sync(FULL, waitx(&k_empty[s], (c / SLOTS - 1) & 1))) break;
        put<D, false>(mine, smem + S::OFF_K + s * S::KV_B, row, quarter, a.bias);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&k_full[s]));
        if (c >= SLOTS && !__all_sync(FULL, waitx(&v_empty[s], (c / SLOTS - 1) & 1))) break;
        put<D, true>(mine, smem + S::OFF_V + s * S::KV_B, row, quarter, a.bias);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&v_full[s]));
      }
    } else {
      // ---------------- softmax X ----------------
      // (after a wait that gave up the warps go on to the end without waiting: they meet at a named barrier)
      const uint32_t x = (warp - S::FIRST_SOFTMAX) >> 2, quad = warp & 3, r = quad * 32 + lane;
      const uint32_t lane_addr = (quad * 32) << 16, s_addr = tmem + lane_addr + x * 128, o_addr = tmem + lane_addr + S::TM_O + x * 128;
      const uint32_t tile_row = row0 + x * BM, row = tile_row + r;
      const float scale = row_scale[x * BM + r];
      // this row sees the keys [lo, hi)
      const int past = q.kv_len - q.q_len;
      const int own = past + static_cast<int>(row / a.group) + 1;
      const int hi = row >= q.rows ? 0 : MODE == PARTS && !q.causal ? q.kv_len : MODE == BEHIND ? before + max(own, 0) : own, lo = MODE == PLAIN ? first_seen(hi, a.window) : 0;
      float m_run = NEG_BIG, l_run = 0.f;
      for (uint32_t i = 0; i < n; i++) {
        const uint32_t c = done + i, b = c & 1, s = c % SLOTS;
        const bool mixed = i - plain0 >= plain_n;
        (void)waitx(&s_ready[x][b], (c >> 1) & 1);
        __syncwarp();
        tc_fence_after();
        if (quad == 0 && lane == 0) mbar_arrive(smem_u32(&k_empty[s]));  // Q K^T of the tile is complete
        uint32_t raw[BN];
#pragma unroll
        for (uint32_t k = 0; k < BN; k += 32) tmem_ld32(s_addr + 64 * b + k, raw + k);
        tmem_ld_wait();
        const int key0 = key_first + static_cast<int>(i * BN);
        if (mixed) {
          const int from = lo - key0, to = hi - key0;
#pragma unroll
          for (int k = 0; k < static_cast<int>(BN); k++)
            if (k >= to || k < from) raw[k] = 0xff800000u;
        }
        float mx[4] = {__uint_as_float(raw[0]), __uint_as_float(raw[1]), __uint_as_float(raw[2]), __uint_as_float(raw[3])};
#pragma unroll
        for (uint32_t k = 4; k < BN - 4; k += 8)
#pragma unroll
          for (uint32_t e = 0; e < 4; e++) mx[e] = max3(mx[e], __uint_as_float(raw[k + e]), __uint_as_float(raw[k + 4 + e]));
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) mx[e] = fmaxf(mx[e], __uint_as_float(raw[BN - 4 + e]));
        const float m_tile = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) ;
        // (The maximum is kept as it comes and taken off before the scale: scores may be of any size. A scaled one would be rounded, from 2^24 on by
        // more than f16 has room for. One packed addition per two scores, 2 % of a prompt.)
        const bool grow = (m_tile - m_run) * scale > GROW;
        const float m_new = grow ? m_tile : m_run, corr = grow ? ex2((m_run - m_new) * scale) : 1.f;
        m_run = m_new;
        if (i > 0 && __any_sync(FULL, grow)) {
          // O_X may be rescaled only between two P V: the previous tile's must be complete
          (void)waitx(&pv_done[x][(c - 1) % SLOTS], ((c - 1) / SLOTS) & 1);
          __syncwarp();
          tc_fence_after();
#pragma unroll 1
          for (uint32_t k = 0; k < D / 16; k++) {
            uint32_t o[16];
            tmem_ld16(o_addr + 16 * k, o);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * corr);
            tmem_st16(o_addr + 16 * k, o);
          }
        }
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        const float down = -m_new;
#pragma unroll
        for (uint32_t k0 = 0; k0 < BN; k0 += 32) {
          uint32_t ph[16];
#pragma unroll
          for (uint32_t k = 0; k < 16; k++) {
            float e0 = down, e1 = down;
            add2(e0, e1, __uint_as_float(raw[k0 + 2 * k]), __uint_as_float(raw[k0 + 2 * k + 1]));
            fma2(e0, e1, e0, e1, scale, P_UP);
            const float p0 = ex2(e0), p1 = ex2(e1);
            add2(sum[2 * (k & 1)], sum[2 * (k & 1) + 1], p0, p1);
            ph[k] = pack2<false>(p0, p1);
          }
          tmem_st16(s_addr + 64 * b + k0 / 2, ph);  // (every S value of this row is in registers)
        }
        l_run = l_run * corr + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&p_ready[x][b]));
      }
      (void)waitx(&v_full[(done + n - 1) % SLOTS], ((done + n - 1) / SLOTS) & 1);  // (`bad` is complete)
      uint32_t over = 0;
#pragma unroll 1
      for (uint32_t at = 0, i; (i = at < plain0 ? at : at + plain_n) < n; at++) {
        const uint4* look = reinterpret_cast<const uint4*>(bad[at]);
        uint32_t any = 0;
#pragma unroll
        for (uint32_t k = 0; k < BN / 16; k++) any |= look[k].x | look[k].y | look[k].z | look[k].w;
        const int key0 = key_first + static_cast<int>(i * BN);
        if (any) {
#pragma unroll 1
          for (int k = max(lo - key0, 0); k < min(hi - key0, static_cast<int>(BN)); k++) over |= bad[at][k];
        }
      }
      (void)waitx(&o_done[x], pieces & 1);
      __syncwarp();
      tc_fence_after();
      if constexpr (MODE == PARTS) {
        // ---- a record per row: in its own place, or as a piece of an item that several CTAs have, whose first one says where they are ----
        const uint32_t first_cta = start / share, parts = (start + keys.tiles - 1) / share - first_cta + 1;
        const bool all = first == 0 && n == keys.tiles;
        float* record = row < q.rows ? record_of<D>(a, !q.causal, q.q0, head, row) : nullptr;
        float* to = all ? record : scratch + static_cast<size_t>(2 * blockIdx.x + (blockIdx.x == first_cta)) * S::PIECE + (x * BM + r) * RECORD<D>;
        const bool there = record && !abort_s;
        // half the dims at a time through the dead Q tile, so that a row's 2 D bytes go to memory together
        constexpr uint32_t U = D / 8;
        uint8_t* stage = smem + x * S::Q_B;
        const uint32_t rows = min(BM, q.rows - min(tile_row, q.rows));
        records[x * BM + r] = to;
        // What is summed refers to the maximum: without P_UP, which a large maximum would swallow. The maximum's product with the scale is rounded; what it lost goes into the sums where
        // both parts are this kernel's (beside it are the other kernel's scores, each rounded the same way). From 2^31 on what is lost no longer fits.
        const float m = m_run * scale, lost = a.first ? 0.f : fmaf(m_run, scale, -m);
        const float down_by = ex2(fminf(fmaxf(lost, -60.f), 60.f) - P_UP);
#pragma unroll 1
        for (uint32_t half = 0; half < 2; half++) {
          if (half) named_bar_sync(1 + x, 128);  // (what was staged before has gone)
#pragma unroll 1
          for (uint32_t k = 0; k < D / 32; k++) {
            uint32_t o[16];
            tmem_ld16(o_addr + D / 2 * half + 16 * k, o);
            tmem_ld_wait();
            const bool none = over >> (D / 64 * half + (k >> 1)) & 1;
#pragma unroll
            for (int e = 0; e < 4; e++) {
              float v[4];
#pragma unroll
              for (int j = 0; j < 4; j++) v[j] = none ? __int_as_float(0x7fffffff) : __uint_as_float(o[8 * (e >> 1) + column_of(4 * (e & 1) + j)]) * down_by;
              *reinterpret_cast<float4*>(stage + r * (2 * D) + (((4 * k + e) ^ (r & (U - 1))) << 4)) = make_float4(v[0], v[1], v[2], v[3]);
            }
          }
          named_bar_sync(1 + x, 128);
          if (!abort_s) {
#pragma unroll 4
            for (uint32_t k = r; k < rows * U; k += 128) {
              const uint32_t row_in = k / U, u = k % U;
              *reinterpret_cast<float4*>(records[x * BM + row_in] + D / 2 * half + 4 * u) = *reinterpret_cast<const float4*>(stage + row_in * (2 * D) + ((u ^ (row_in & (U - 1))) << 4));
            }
          }
        }
        if (there) {
          end_record<D>(to, l_run == 0.f ? NEG_BIG : m, l_run * down_by);
          if (!all && blockIdx.x == first_cta) end_record<D>(record, NEG_BIG, 0.f, first_cta, parts, x * BM + r);
        }
      } else if (first == 0 && n == keys.tiles) {
        // ---- the whole item: O / l through the dead Q tile, whole rows of it to memory ----
        const float inv_l = l_run == 0.f ? 0.f : 1.f / l_run;
        uint8_t* stage = smem + x * S::Q_B;
#pragma unroll 1
        for (uint32_t k = 0; k < D / 16; k++) {
          uint32_t o[16];
          tmem_ld16(o_addr + 16 * k, o);
          tmem_ld_wait();
          const float inv = over >> (k >> 1) & 1 ? __int_as_float(0x7fffffff) : inv_l;
#pragma unroll
          for (int e = 0; e < 2; e++) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = __uint_as_float(o[8 * e + column_of(j)]) * inv;
            const uint32_t u = 2 * k + e;
            *reinterpret_cast<uint4*>(stage + r * (D * 2) + ((u ^ (r & (D / 8 - 1))) << 4)) = a.bf ? pack8<true>(v) : pack8<false>(v);
          }
        }
        named_bar_sync(1 + x, 128);
        if (tile_row < q.rows && !abort_s) store_rows<D>(a, q.q0, head, tile_row, min(BM, q.rows - tile_row), stage, r, 128);
      } else {
        // ---- a part of an item: as it is, to be joined ----
        const uint32_t first_cta = start / share;
        float* mine = scratch + static_cast<size_t>(2 * blockIdx.x + (blockIdx.x == first_cta)) * S::PARTIAL;
        float4* to = reinterpret_cast<float4*>(mine) + x * BM + r;
#pragma unroll 1
        for (uint32_t k = 0; k < D / 16; k++) {
          uint32_t o[16];
          tmem_ld16(o_addr + 16 * k, o);
          tmem_ld_wait();
          if (over >> (k >> 1) & 1) {
#pragma unroll
            for (int e = 0; e < 16; e++) o[e] = 0x7fffffffu;
          }
#pragma unroll
          for (int e = 0; e < 4; e++) {
            float v[4];
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = __uint_as_float(o[8 * (e >> 1) + column_of(4 * (e & 1) + j)]);
            to[(4 * k + e) * S::ROWS] = make_float4(v[0], v[1], v[2], v[3]);  // (a warp's 32 rows are 512 bytes)
          }
        }
        reinterpret_cast<float2*>(mine + D * S::ROWS)[x * BM + r] = make_float2(l_run == 0.f ? NEG_BIG : m_run, l_run);
      }
    }
    done += n;
    pieces++;
    pos += n;
    tc_fence_before();
    __syncthreads();  // the piece is finished by every role: Q, S and O can be reused
    tc_fence_after();
    if (abort_s) break;

    // ---- an item of several CTAs is joined by the one that comes last ----
    const bool whole = MODE == PARTS || (first == 0 && n == keys.tiles);  // (parts are joined by another kernel)
    if (threadIdx.x == 0) {
      if (!whole) {
        const uint32_t first_cta = start / share, parts = (start + keys.tiles - 1) / share - first_cta + 1;
        const bool last = arrive(&counters[first_cta]) == parts - 1;
        if (last) counters[first_cta] = 0;  // for the next launch
        join_s = Join{first_cta, parts, last};
      }
      if (pos < c1) {
        Cursor c = cur;
        c.at = 0;
        c.start = pos + ITEM_COST<MODE>;
        if (++c.head == a.pool.n_kv_head) {
          c.head = 0;
          if (++c.x * S::ROWS >= c.q.rows) {
            c.x = 0;
            do c.q = request_of(++c.r);  // (there is a further item in the line)
            while (c.q.rows == 0);
          }
          c.keys = keys_of<MODE>(a, c.q, c.x * S::ROWS, S::ROWS);
        }
        cur = c;
      }
    }
    __syncthreads();
    if (!whole && join_s.last) {
      const Join j = join_s;
      const float* from = scratch + static_cast<size_t>(2 * j.first_cta) * S::PARTIAL;
      const uint32_t rows = min(S::ROWS, q.rows - row0);
      auto piece = [&](uint32_t k) { return from + static_cast<size_t>(2 * k + (k == 0)) * S::PARTIAL; };
      auto ml = [&](uint32_t k, uint32_t r) { return reinterpret_cast<const float2*>(piece(k) + D * S::ROWS)[r]; };
      // the rows' maxima (before the scale, as in the tiles: scaled ones would be rounded) and 1 / sums, in the dead K tiles; then a thread per four dims of a row, the rows of a warp side by side
      float2* joined = reinterpret_cast<float2*>(smem + S::OFF_K);
      for (uint32_t r = threadIdx.x; r < S::ROWS; r += THREADS) {
        float m = NEG_BIG, l = 0.f;
        const float scale = row_scale[r];
#pragma unroll 4
        for (uint32_t k = 0; k < j.n; k++) {
          const float2 e = ml(k, r);
          const float top = fmaxf(m, e.x);
          l = l * ex2((m - top) * scale) + e.y * ex2((e.x - top) * scale);
          m = top;
        }
        joined[r] = make_float2(m, l == 0.f ? 0.f : 1.f / l);
      }
      __syncthreads();
#pragma unroll 4
      for (uint32_t i = threadIdx.x; i < S::ROWS * (D / 4); i += THREADS) {
        const uint32_t r = i % S::ROWS, c = i / S::ROWS;
        const float2 all = joined[r];
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
        for (uint32_t k = 0; k < j.n; k++) {
          const float4 v = reinterpret_cast<const float4*>(piece(k))[c * S::ROWS + r];
          const float w = ex2((ml(k, r).x - all.x) * row_scale[r]) * all.y;
          o = make_float4(fmaf(v.x, w, o.x), fmaf(v.y, w, o.y), fmaf(v.z, w, o.z), fmaf(v.w, w, o.w));
        }
        // staged in the dead Q tiles: whole rows go to memory
        const uint32_t lo = a.bf ? pack2<true>(o.x, o.y) : pack2<false>(o.x, o.y), hi = a.bf ? pack2<true>(o.z, o.w) : pack2<false>(o.z, o.w);
        *reinterpret_cast<uint2*>(smem + r * (D * 2) + (((c >> 1) ^ (r & (D / 8 - 1))) << 4) + 8 * (c & 1)) = make_uint2(lo, hi);
      }
      __syncthreads();
      store_rows<D>(a, q.q0, head, row0, rows, smem, threadIdx.x, THREADS);
    }
    __syncthreads();
  }

  if (abort_s) {  // (all threads) the MMAs on their way are complete before TMEM and shared memory are given back
    if (threadIdx.x == 0) {
      mbar_init(smem_u32(&drained), 4);
      fence_barrier_init();
    }
    __syncthreads();
    if (warp < 4 && elect_one()) umma_commit(smem_u32(&drained));  // (the threads that issued them)
    if (threadIdx.x == 0) (void)wait_phase(smem_u32(&drained), 0);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, S::TMEM_COLS);
}

template <int MODE, typename F>
cudaError_t with_kernel(uint32_t head_dim, bool two, F f) {
  if (head_dim == 128) return two ? f(kv4_prefill_kernel<128, 2, MODE>, Shape<128, 2>()) : f(kv4_prefill_kernel<128, 1, MODE>, Shape<128, 1>());
  return two ? f(kv4_prefill_kernel<64, 2, MODE>, Shape<64, 2>()) : f(kv4_prefill_kernel<64, 1, MODE>, Shape<64, 1>());
}

}  // namespace

cudaError_t bp_kv4_prefill_init(bp_paged_ctx* c) {
  size_t floats = 0;
  cudaError_t e = cudaSuccess;
  auto allow = [&](auto kernel, auto shape) {
    const size_t need = 2 * static_cast<size_t>(c->sm_count) * shape.PIECE;  // two pieces per CTA
    if (need > floats) floats = need;
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(shape.SMEM));
  };
  for (uint32_t i = 0; i < 4 && e == cudaSuccess; i++) {
    e = with_kernel<PLAIN>(i & 1 ? 128 : 64, i & 2, allow);
    if (e == cudaSuccess) e = with_kernel<PARTS>(i & 1 ? 128 : 64, i & 2, allow);
    if (e == cudaSuccess) e = with_kernel<BEHIND>(i & 1 ? 128 : 64, i & 2, allow);
  }
  return e != cudaSuccess ? e : cudaMalloc(&c->prefill_partials, floats * sizeof(float));
}

cudaError_t bp_launch_kv4_prefill(bp_paged_ctx* c, cudaStream_t s, uint32_t head_dim, int mode, uint64_t rows, uint32_t ctas, const AttnArgs& a, const float** slots, uint32_t* piece) {
  auto launch = [&](auto kernel, auto shape) {
    using S = decltype(shape);
    if (slots) *slots = c->prefill_partials;
    if (piece) *piece = S::PIECE;
    return bp_launch(true, kernel, dim3(ctas ? ctas : c->sm_count), dim3(S::THREADS), S::SMEM, s, a, c->prefill_partials, c->counters);
  };
  return mode == PLAIN   ? with_kernel<PLAIN>(head_dim, rows > BM, launch)
         : mode == PARTS ? with_kernel<PARTS>(head_dim, rows > BM, launch)
                         : with_kernel<BEHIND>(head_dim, rows > BM, launch);
}
