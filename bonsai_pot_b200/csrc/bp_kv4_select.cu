// Attention over chosen pages of a 4-bit cache (include/bonsai_pages.h): the pages' summaries, the choice, and the call of the attention
// kernel (bp_kv4_attention.cu) over a list of pages per token and KV head.
#include "bp_kv4_attention.cuh"
#include "bp_paged_host.cuh"

namespace {

using namespace bp;
using namespace bp::kv4;
using namespace bp::paged;

// ---- summaries -------------------------------------------------------------------------------------------------------

struct SummaryArgs {
  Pool pool;
  int8_t* codes;
  float* scales;
  const int32_t *pages, *n_tok;
  uint32_t n;
  uint32_t* err;
  uint32_t bias;
};
constexpr uint32_t SUMMARY_WARPS = 4;

// Latency again: 31 pages of 64 tokens and 8 heads 2.3 us (5.7 with a warp per page). A warp per 16 tokens of a page and KV head, all of whose loads are on their way at once: a lane has eight dims (a 32-bit word) of every 32 / (D / 8)-th token. The
// page's first warp goes on. Every value m + d q is an f16 number, so f16 maxima are exact.
template <int D>
__global__ void __launch_bounds__(32 * SUMMARY_WARPS) kv4_summary_kernel(const __grid_constant__ SummaryArgs a) {
  using L = PoolLayout<D>;
  constexpr uint32_t NB = L::NB, LANES = D / 8, STEP = 32 / LANES, N = 16 / STEP;
  __shared__ __half2 found[SUMMARY_WARPS][8][LANES];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, log_warps = a.pool.log_page - 4;
  const uint32_t item = blockIdx.x * (SUMMARY_WARPS >> log_warps) + (warp >> log_warps), at = item / a.pool.n_kv_head, head = item - at * a.pool.n_kv_head;
  const uint32_t part = warp & ((1u << log_warps) - 1);
  pdl_launch_dependents();
  pdl_wait();
  const int32_t page = at < a.n ? a.pages[at] : -1;
  const int32_t given = page < 0 || !a.n_tok ? static_cast<int32_t>(a.pool.page) : a.n_tok[at];
  const bool good = page >= 0 && static_cast<uint32_t>(page) < a.pool.n_pages && given > 0 && given <= static_cast<int32_t>(a.pool.page);
  if (page >= 0 && !good && lane == 0 && part == 0) note_range(a.err);
  const uint32_t n = good ? given : 0, c = lane % LANES / NB, b = lane % NB;
  const size_t record = good ? static_cast<size_t>(page) * a.pool.n_kv_head + head : 0;
  const uint8_t* k = a.pool.data + record * (a.pool.page * L::TOK);
  const uint8_t *words = k + (c * NB + b) * 4, *ds = k + L::kd(a.pool.page) + 2 * b, *ms = k + L::km(a.pool.page) + 2 * b;
  const __half2 none_hi = __float2half2_rn(-INFINITY), none_lo = __float2half2_rn(INFINITY);
  __half2 hi[4] = {none_hi, none_hi, none_hi, none_hi}, lo[4] = {none_lo, none_lo, none_lo, none_lo};
  const __half2 off = __float2half2_rn(-1024.f), off16 = __float2half2_rn(-64.f), sixteenth = __float2half2_rn(0.0625f);
  const uint32_t t0 = 16 * part + lane / LANES;
  uint32_t w[N];
  uint16_t d16[N], m16[N];
#pragma unroll
  for (uint32_t i = 0; i < N; i++) {
    const uint32_t t = t0 + i * STEP;
    if (t >= n) continue;
    w[i] = *reinterpret_cast<const uint32_t*>(words + t * L::ROW);
    d16[i] = *reinterpret_cast<const uint16_t*>(ds + t * 2 * NB);
    m16[i] = *reinterpret_cast<const uint16_t*>(ms + t * 2 * NB);
  }
#pragma unroll
  for (uint32_t i = 0; i < N; i++) {
    if (t0 + i * STEP >= n) continue;
    const uint32_t x = w[i], y = x >> 8;
    const __half2 d = __half2half2(__ushort_as_half(d16[i])), m = __half2half2(__ushort_as_half(m16[i]));
    const __half2 v[4] = {__hfma2(__hadd2(biased(x, 0x000f000fu, a.bias), off), d, m), __hfma2(__hfma2(biased(x, 0x00f000f0u, a.bias), sixteenth, off16), d, m),
                          __hfma2(__hadd2(biased(y, 0x000f000fu, a.bias), off), d, m), __hfma2(__hfma2(biased(y, 0x00f000f0u, a.bias), sixteenth, off16), d, m)};
#pragma unroll
    for (int e = 0; e < 4; e++) {
      hi[e] = __hmax2(hi[e], v[e]);
      lo[e] = __hmin2(lo[e], v[e]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
#pragma unroll
    for (uint32_t o = LANES; o < 32; o <<= 1) {
      hi[i] = __hmax2(hi[i], h2(__shfl_xor_sync(FULL, u2(hi[i]), o)));
      lo[i] = __hmin2(lo[i], h2(__shfl_xor_sync(FULL, u2(lo[i]), o)));
    }
  }
  if (log_warps > 0) {
    if (part != 0 && lane < LANES) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        found[warp][i][lane] = hi[i];
        found[warp][4 + i][lane] = lo[i];
      }
    }
    __syncthreads();
    for (uint32_t p = 1; p < 1u << log_warps; p++) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        hi[i] = __hmax2(hi[i], found[(warp + p) % SUMMARY_WARPS][i][lane % LANES]);
        lo[i] = __hmin2(lo[i], found[(warp + p) % SUMMARY_WARPS][4 + i][lane % LANES]);
      }
    }
  }
  if (!good || part != 0) return;
  float ends[2][8], top = 0.f;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 x = __half22float2(hi[i]), z = __half22float2(lo[i]);
    const bool some0 = z.x <= x.x, some1 = z.y <= x.y;
    ends[0][2 * i] = some0 ? x.x : 0.f;
    ends[0][2 * i + 1] = some1 ? x.y : 0.f;
    ends[1][2 * i] = some0 ? -z.x : 0.f;
    ends[1][2 * i + 1] = some1 ? -z.y : 0.f;
  }
#pragma unroll
  for (int i = 0; i < 8; i++) top = fmaxf(top, fmaxf(fabsf(ends[0][i]), fabsf(ends[1][i])));
#pragma unroll
  for (uint32_t o = 1; o < LANES; o <<= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, o));
  // 2^(e - 6), e limited to -24 .. 16
  const uint32_t e = min(max(__float_as_uint(top) & 0x7f800000u, (127u - 24u) << 23), (127u + 16u) << 23);
  const bool twice = top > 127.f * __uint_as_float(e - (6u << 23));
  const float scale = __uint_as_float(e - (twice ? 5u << 23 : 6u << 23)), inv = __uint_as_float((254u << 23) - __float_as_uint(scale));
  if (lane < LANES) {
#pragma unroll
    for (int s = 0; s < 2; s++) {
      uint32_t word[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int code = static_cast<int>(fminf(fmaxf(ceilf(ends[s][i] * inv), -127.f), 127.f));
        word[i >> 2] |= (static_cast<uint32_t>(code) & 255u) << (8 * (i & 3));
      }
      *reinterpret_cast<uint2*>(a.codes + (record * 2 + s) * D + 32 * b + 8 * c) = make_uint2(word[0], word[1]);
    }
    if (lane == 0) a.scales[record] = scale;
  }
}

// ---- the choice ------------------------------------------------------------------------------------------------------

struct ChoiceArgs {
  AttnArgs a;
  const int8_t* codes;
  const float* scales;
  int32_t *pages, *keys;
  uint32_t chosen, first, last;
  uint32_t split;  // CTAs of a cluster, which share a token's pages
};
constexpr uint32_t CHOICE_THREADS = 256, MAX_BLOCKS = 49152;
template <int D>
constexpr uint32_t AT_A_TIME = 512 / D;  // pages that eight lanes ask for together, 128 bytes each

// Sum of u8 x s8 products of four bytes each, added to c.
__device__ __forceinline__ int dot4(uint32_t u, uint32_t s, int c) {
  int d;
  asm("dp4a.u32.s32 %0, %1, %2, %3;" : "=r"(d) : "r"(u), "r"(s), "r"(c));
  return d;
}
// A number whose order as an unsigned one is that of x (no NaN).
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// Stores into the shared memory of the cluster's first CTA, at the same place as `at` here.
__device__ __forceinline__ void store_to_first(uint32_t* at, uint32_t x) {
  uint32_t there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(there) : "r"(smem_u32(at)));
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(there), "r"(x) : "memory");
}

// A cluster of `split` CTAs per token and KV head. Every CTA scores its part of the pages, eight lanes per page with 2 D / 8 bytes of its summary each; the scores
// go to the first CTA, which looks for the want-th highest of them: the range in which it lies is cut into up to 256 parts of equal width and counted until one part
// holds no others than are wanted. Bound by latency: what follows the launch is one chain of accesses to memory (the token's request 0.4 us, its lengths, page ids and summaries
// 1.6 to 2 for as many pages as are asked for at a time) and of barriers (range and counts 2, the list 1.5). One token of 1024 pages 6.9 us in clusters of eight (0.3 of memory; 23 with a CTA per head that
// asked for four pages at a time per warp), 53 tokens of up to 512 pages 10.3, 32 tokens of up to 512 pages of twice the bytes 9.3 (4749 pages of 8 heads: 1.5 of memory).
template <int D>
__global__ void __launch_bounds__(CHOICE_THREADS) kv4_select_kernel(const __grid_constant__ ChoiceArgs s) {
  constexpr uint32_t WARPS = CHOICE_THREADS / 32;
  extern __shared__ uint32_t order[];  // scores of the token's pages as ordered numbers
  __shared__ __align__(16) uint8_t query[2 * D];
  __shared__ float tops[WARPS];
  __shared__ uint32_t hist[256], sums[WARPS], lows[WARPS], highs[WARPS], pick[3];
  const AttnArgs& a = s.a;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, token = blockIdx.x / s.split, rank = blockIdx.x - token * s.split, head = blockIdx.y;
  pdl_launch_dependents();
  if (s.split > 1) cluster_arrive();  // (nobody stores into a CTA that has not begun)
  pdl_wait();
  // ---- the sums of the queries' positive and negative parts, in the order of the heads ----
  float up = 0.f, down = 0.f;
  if (threadIdx.x < D) {
    const uint16_t* q = a.q.data + static_cast<int64_t>(token) * a.q.tok + static_cast<int64_t>(head * a.group) * a.q.head + threadIdx.x;
#pragma unroll 4
    for (uint32_t g = 0; g < a.group; g++) {
      const float x = a.bf ? to_f32<true>(q[g * a.q.head]) : to_f32<false>(q[g * a.q.head]);
      up += fmaxf(x, 0.f);
      down += fmaxf(-x, 0.f);
    }
  }
  // ---- what the token sees ----
  const int r = last_begun(a.q_start, a.n_req + 1, static_cast<int>(token), lane);
  int sees = -1;
  if (r >= 0 && r < static_cast<int>(a.n_req)) {
    const Lengths n = lengths_of<PLAIN>(a, r, head == 0 && threadIdx.x == 0);
    const int i = static_cast<int>(token) - n.q0;
    if (i < n.q_len) sees = max(n.kv_len - n.q_len + i + 1, 0);
  }
  const uint32_t blocks = sees > 0 ? (static_cast<uint32_t>(sees) + a.pool.page - 1) >> a.pool.log_page : 0, n = min(blocks, s.chosen);
  int32_t* out = s.pages + (static_cast<size_t>(token) * a.pool.n_kv_head + head) * s.chosen;
  const int32_t* table = a.page_table + static_cast<size_t>(max(r, 0)) * a.table_stride;
  if (rank == 0) {
    if (head == 0 && threadIdx.x == 0) s.keys[token] = sees < 0 ? -1 : sees - static_cast<int>((blocks - n) << a.pool.log_page);
    for (uint32_t i = n + threadIdx.x; i < s.chosen; i += CHOICE_THREADS) out[i] = -1;
    if (n == blocks)
      for (uint32_t i = threadIdx.x; i < n; i += CHOICE_THREADS) out[i] = table[i];
  }
  if (n == blocks) {  // (the whole cluster)
    if (s.split > 1) cluster_wait();
    return;
  }
  // ---- the query in 8 bits ----
  float top = fmaxf(up, down);
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, o));
  if (lane == 0) tops[warp] = top;
  __syncthreads();
#pragma unroll
  for (uint32_t w = 0; w < WARPS; w++) top = fmaxf(top, tops[w]);
  const uint32_t e = min(max(__float_as_uint(top) & 0x7f800000u, 27u << 23), 254u << 23);  // 2^-100 .. 2^127
  const float inv = __uint_as_float((261u << 23) - e);                                      // 2^(7 - e)
  if (threadIdx.x < D) {
    query[threadIdx.x] = static_cast<uint8_t>(fminf(rintf(up * inv), 255.f));
    query[D + threadIdx.x] = static_cast<uint8_t>(fminf(rintf(down * inv), 255.f));
  }
  __syncthreads();
  // ---- scores ----
  constexpr uint32_t W = 2 * D / 32;  // words of a lane
  uint32_t mine[W];
#pragma unroll
  for (uint32_t i = 0; i < W; i++) mine[i] = reinterpret_cast<const uint32_t*>(query)[(lane & 7) * 4 + (i >> 2) * 32 + (i & 3)];
  const uint32_t per = (blocks + s.split - 1) / s.split, from = min(rank * per, blocks), to = min(from + per, blocks);
  if (s.split > 1) cluster_wait();
  constexpr uint32_t STEP = CHOICE_THREADS / 8;
  uint32_t ids[AT_A_TIME<D>];
  auto ask_ids = [&](uint32_t b0) {
#pragma unroll
    for (uint32_t k = 0; k < AT_A_TIME<D>; k++) ids[k] = b0 + k * STEP < to ? static_cast<uint32_t>(table[b0 + k * STEP]) : 0xffffffffu;
  };
  ask_ids(from + (threadIdx.x >> 3));
  for (uint32_t b0 = from + (threadIdx.x >> 3); __any_sync(FULL, b0 < to); b0 += AT_A_TIME<D> * STEP) {
    uint4 v[AT_A_TIME<D>][W / 4];
    float scale[AT_A_TIME<D>];
    bool good[AT_A_TIME<D>];
#pragma unroll
    for (uint32_t k = 0; k < AT_A_TIME<D>; k++) {
      good[k] = ids[k] < a.pool.n_pages;
      const size_t record = good[k] ? static_cast<size_t>(ids[k]) * a.pool.n_kv_head + head : 0;
      const uint4* codes = reinterpret_cast<const uint4*>(s.codes + record * 2 * D) + (lane & 7);
      scale[k] = s.scales[record];
#pragma unroll
      for (uint32_t i = 0; i < W / 4; i++) v[k][i] = codes[8 * i];
    }
    ask_ids(b0 + AT_A_TIME<D> * STEP);
#pragma unroll
    for (uint32_t k = 0; k < AT_A_TIME<D>; k++) {
      int sum = 0;
#pragma unroll
      for (uint32_t i = 0; i < W / 4; i++) {
        sum = dot4(mine[4 * i], v[k][i].x, sum);
        sum = dot4(mine[4 * i + 1], v[k][i].y, sum);
        sum = dot4(mine[4 * i + 2], v[k][i].z, sum);
        sum = dot4(mine[4 * i + 3], v[k][i].w, sum);
      }
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(FULL, sum, o);
      const uint32_t b = b0 + k * STEP;
      if (b < to && (lane & 7) == k % 8) {
        if (!good[k]) note_range(a.err);
        const uint32_t x = good[k] ? ordered(static_cast<float>(sum) * scale[k]) : 0u;
        if (s.split > 1) store_to_first(&order[b], x);
        else order[b] = x;
      }
    }
  }
  if (s.split > 1) {
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    if (rank) return;
  } else {
    __syncthreads();
  }
  // ---- the want-th highest of those that are not chosen anyway ----
  const uint32_t begin = s.first, end = blocks - s.last;
  uint32_t want = n - s.first - s.last, least = 0xffffffffu, ties = 0;  // chosen are those above `least` and the first `ties` of those equal to it
  if (want > 0) {
    uint32_t low = 0xffffffffu, high = 0;
    for (uint32_t i = begin + threadIdx.x; i < end; i += CHOICE_THREADS) {
      low = min(low, order[i]);
      high = max(high, order[i]);
    }
    low = __reduce_min_sync(FULL, low);
    high = __reduce_max_sync(FULL, high);
    if (lane == 0) {
      lows[warp] = low;
      highs[warp] = high;
    }
    hist[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < WARPS; w++) {
      low = min(low, lows[w]);
      high = max(high, highs[w]);
    }
    while (true) {
      const uint32_t range = high - low, bits = 32 - __clz(range), shift = bits > 8 ? bits - 8 : 0;
      for (uint32_t i = begin + threadIdx.x; i < end; i += CHOICE_THREADS) {
        const uint32_t x = order[i] - low;
        if (x <= range) atomicAdd(&hist[x >> shift], 1);
      }
      __syncthreads();
      // thread t: those in part 255 - t or a higher one
      const uint32_t count = hist[255 - threadIdx.x];
      uint32_t run = count;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(FULL, run, o);
        if (lane >= o) run += x;
      }
      if (lane == 31) sums[warp] = run;
      __syncthreads();
      for (uint32_t w = 0; w < warp; w++) run += sums[w];
      if (run >= want && run - count < want) {
        pick[0] = 255 - threadIdx.x;
        pick[1] = want - (run - count);
        pick[2] = count;
      }
      hist[255 - threadIdx.x] = 0;
      __syncthreads();
      low += pick[0] << shift;
      want = pick[1];
      if (shift == 0 || pick[2] == want) {
        least = low;
        ties = shift == 0 ? want : 0xffffffffu;  // (the whole part)
        break;
      }
      high = low + ((1u << shift) - 1);
    }
  }
  // ---- in the order of the keys: a thread has `each` pages side by side ----
  const uint32_t each = (blocks + CHOICE_THREADS - 1) / CHOICE_THREADS, b0 = min(threadIdx.x * each, blocks), b1 = min(b0 + each, blocks);
  auto kind = [&](uint32_t b) -> uint32_t {  // 1: chosen, 1 << 16: equal to the last one
    if (b < begin || b >= end) return 1;
    return order[b] > least ? 1u : ties && order[b] == least ? 1u << 16 : 0u;
  };
  uint32_t mine_of = 0;
  for (uint32_t b = b0; b < b1; b++) mine_of += kind(b);
  uint32_t upto = mine_of;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t x = __shfl_up_sync(FULL, upto, o);
    if (lane >= o) upto += x;
  }
  if (lane == 31) sums[warp] = upto;
  __syncthreads();
  for (uint32_t w = 0; w < warp; w++) upto += sums[w];
  uint32_t above = (upto - mine_of) & 0xffff, equal = (upto - mine_of) >> 16;
  for (uint32_t b = b0; b < b1; b++) {
    const uint32_t k = kind(b);
    if (k == 1 || (k && equal < ties)) out[above + min(equal, ties)] = table[b];
    above += k & 0xffff;
    equal += k >> 16;
  }
}

}  // namespace

cudaError_t bp_kv4_select_init(bp_paged_ctx* c) {
  (void)c;
  cudaError_t e = cudaFuncSetAttribute(kv4_select_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_BLOCKS * 4);
  return e != cudaSuccess ? e : cudaFuncSetAttribute(kv4_select_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_BLOCKS * 4);
}

extern "C" {

int bp_kv4_summarise(bp_paged_ctx* c, void* stream, const bp_kv4_pool* pool, const bp_block_summary* summary, const void* pages, const void* n_tok, uint32_t n) {
  if (int s = enter(c)) return s;
  if (!pool || !summary) return fail(c, BP_ERR_NULL, "null pointer argument");
  Pool p;
  BP_CHECK(c, check_pool(pool, &p));
  if (!aligned_to(summary->codes, 16) || !aligned_to(summary->scales, 4)) return fail_config(c, "codes must be 16-byte, scales 4-byte aligned");
  if (!aligned_to(pages, 4) || !aligned_to(n_tok, 4)) return fail_config(c, "pages and n_tok must be 4-byte aligned");
  if (static_cast<uint64_t>(n) * p.n_kv_head > 0x7fffffffull) return fail_config(c, "n * n_kv_head must be < 2^31");
  if (n == 0) return BP_OK;
  if (!p.data || !summary->codes || !summary->scales || !pages) return fail(c, BP_ERR_NULL, "null pointer argument");
  OnDevice on(c->device);
  BP_TRY(c, on.err);
  const SummaryArgs a{p, static_cast<int8_t*>(summary->codes), static_cast<float*>(summary->scales), static_cast<const int32_t*>(pages), static_cast<const int32_t*>(n_tok), n,
                      c->err_dev, 0x64006400u};
  const uint32_t of_cta = SUMMARY_WARPS * 16 / p.page;
  const dim3 grid((n * p.n_kv_head + of_cta - 1) / of_cta);
  BP_TRY(c, bp_launch(true, pool->head_dim == 128 ? kv4_summary_kernel<128> : kv4_summary_kernel<64>, grid, dim3(32 * SUMMARY_WARPS), 0, static_cast<cudaStream_t>(stream), a));
  return BP_OK;
}

int bp_kv4_select(bp_paged_ctx* c, void* stream, uint32_t dtype, const bp_kv4_pool* pool, const bp_block_summary* summary, const bp_kv4_choice* in) {
  if (int s = enter(c)) return s;
  if (!pool || !summary || !in) return fail(c, BP_ERR_NULL, "null pointer argument");
  if (dtype > BP_DTYPE_BF16) return fail_config(c, "the activation type must be BP_DTYPE_F16 or BP_DTYPE_BF16");
  Rows rq;
  Pool p;
  BP_CHECK(c, check_pool(pool, &p));
  BP_CHECK(c, check_rows(&in->q, &rq));
  if (in->n_head == 0 || in->n_head % p.n_kv_head) return fail_config(c, "n_head must be a multiple of n_kv_head");
  if (in->last == 0 || static_cast<uint64_t>(in->first) + in->last > in->chosen) return fail_config(c, "last must be > 0 and first + last <= chosen");
  if (!aligned_to(in->q_start, 4) || !aligned_to(in->kv_len, 4) || !aligned_to(in->page_table, 4) || !aligned_to(in->pages, 4) || !aligned_to(in->keys, 4))
    return fail_config(c, "q_start, kv_len, page_table, pages and keys must be 4-byte aligned");
  if (!aligned_to(summary->codes, 16) || !aligned_to(summary->scales, 4)) return fail_config(c, "codes must be 16-byte, scales 4-byte aligned");
  if (in->n_req > 65535) return fail_config(c, "at most 65535 requests");
  if (static_cast<uint64_t>(in->total_q) * in->n_head > 0x7fffffffull || in->chosen > 0x7fffffffu) return fail_config(c, "total_q * n_head and chosen must be < 2^31");
  const uint32_t cap = bp_kv4_table_pages(p, in->table_stride);
  const uint64_t asked = (static_cast<uint64_t>(in->max_kv) + p.page - 1) / p.page, blocks = asked < cap ? asked : cap;
  if (blocks > MAX_BLOCKS) return fail_config(c, "at most 49152 pages per request");
  if (in->total_q == 0) return BP_OK;
  if (!in->q_start || !in->pages || !in->keys || !rq.data || (in->n_req != 0 && !in->kv_len) || (blocks != 0 && in->n_req != 0 && (!in->page_table || !p.data || !summary->codes || !summary->scales)))
    return fail(c, BP_ERR_NULL, "null pointer argument");
  OnDevice on(c->device);
  BP_TRY(c, on.err);
  ChoiceArgs s = {};
  bp_kv4_attention_args(c, dtype == BP_DTYPE_BF16, p, in->q, in->q, in->n_head, 1.f, &s.a);
  s.a.q_start = static_cast<const int32_t*>(in->q_start);
  s.a.kv_len = static_cast<const int32_t*>(in->kv_len);
  s.a.page_table = static_cast<const int32_t*>(in->page_table);
  s.a.n_req = in->n_req;
  s.a.total_q = in->total_q;
  s.a.max_q = in->max_q < in->total_q ? in->max_q : in->total_q;
  s.a.max_kv = in->max_kv < 0x7fffff00u ? in->max_kv : 0x7fffff00u;
  s.a.table_stride = in->table_stride;
  s.a.table_pages = cap;
  s.codes = static_cast<const int8_t*>(summary->codes);
  s.scales = static_cast<const float*>(summary->scales);
  s.pages = static_cast<int32_t*>(in->pages);
  s.keys = static_cast<int32_t*>(in->keys);
  s.chosen = in->chosen;
  s.first = in->first;
  s.last = in->last;
  // CTAs per token and head: as many as the SMs hold at once (four each), each of more pages than it asks for at a time. (One token of 1024 pages 7 us instead of
  // 23, 32 tokens of up to 512 pages in twos 9.3 instead of 10.8.)
  s.split = 1;
  while (s.split < 8 && 2 * static_cast<uint64_t>(in->total_q) * p.n_kv_head * s.split <= 4 * static_cast<uint64_t>(c->sm_count) && blocks > (pool->head_dim == 128 ? 128u : 256u) * s.split) s.split *= 2;
  if (static_cast<uint64_t>(in->total_q) * s.split > 0x7fffffffull) return fail_config(c, "total_q is too large for one call");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(in->total_q * s.split, p.n_kv_head);
  cfg.blockDim = dim3(CHOICE_THREADS);
  cfg.dynamicSmemBytes = blocks * 4;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = s.split;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = s.split > 1 ? 2 : 1;
  BP_TRY(c, cudaLaunchKernelEx(&cfg, pool->head_dim == 128 ? kv4_select_kernel<128> : kv4_select_kernel<64>, s));
  return BP_OK;
}

int bp_kv4_attention_selected(bp_paged_ctx* c, void* stream, uint32_t dtype, const bp_kv4_pool* pool, const bp_kv4_chosen* in) {
  if (int s = enter(c)) return s;
  if (!pool || !in) return fail(c, BP_ERR_NULL, "null pointer argument");
  if (dtype > BP_DTYPE_BF16) return fail_config(c, "the activation type must be BP_DTYPE_F16 or BP_DTYPE_BF16");
  Rows rq, ro;
  Pool p;
  BP_CHECK(c, check_pool(pool, &p));
  BP_CHECK(c, check_rows(&in->q, &rq));
  BP_CHECK(c, check_rows(&in->out, &ro));
  if (in->n_head == 0 || in->n_head % p.n_kv_head) return fail_config(c, "n_head must be a multiple of n_kv_head");
  if (in->scale != in->scale) return fail_config(c, "scale must be a number");
  if (!aligned_to(in->pages, 4) || !aligned_to(in->keys, 4)) return fail_config(c, "pages and keys must be 4-byte aligned");
  if (in->total_q > 65535) return fail_config(c, "at most 65535 tokens");
  if (in->total_q == 0) return BP_OK;
  if (static_cast<uint64_t>(in->total_q) * in->n_head > 0x7fffffffull || in->chosen > 0x7fffff00u / p.page) return fail_config(c, "total_q * n_head and the chosen keys must be < 2^31");
  const uint64_t tiles = (static_cast<uint64_t>(in->n_head / p.n_kv_head) + 7) / 8 * in->total_q;
  if (tiles * p.n_kv_head > 0xffffffffull / (static_cast<uint64_t>(in->chosen) * p.page / 64 + 8)) return fail_config(c, "total_q * n_head * chosen is too large for one call");
  if (!rq.data || !ro.data || !in->keys || (in->chosen != 0 && (!p.data || !in->pages))) return fail(c, BP_ERR_NULL, "null pointer argument");
  OnDevice on(c->device);
  BP_TRY(c, on.err);
  AttnArgs a;
  bp_kv4_attention_args(c, dtype == BP_DTYPE_BF16, p, in->q, in->out, in->n_head, in->scale, &a);
  a.kv_len = static_cast<const int32_t*>(in->keys);
  a.page_table = static_cast<const int32_t*>(in->pages);
  a.n_req = a.total_q = in->total_q;
  a.max_q = 1;
  a.max_kv = in->chosen * p.page;
  a.table_stride = a.table_pages = in->chosen;
  BP_TRY(c, bp_launch_kv4_few_rows(c, static_cast<cudaStream_t>(stream), pool->head_dim, CHOSEN, a.group, 0, a));
  return BP_OK;
}

}  // extern "C"
