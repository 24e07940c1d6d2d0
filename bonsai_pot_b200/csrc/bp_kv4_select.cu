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

// A warp per page and KV head: a lane has eight dims (a 32-bit word) of every 32 / (D / 8)-th token. Every value m + d q is an f16 number, so f16 maxima are exact.
template <int D>
__global__ void __launch_bounds__(32 * SUMMARY_WARPS) kv4_summary_kernel(const __grid_constant__ SummaryArgs a) {
  using L = PoolLayout<D>;
  constexpr uint32_t NB = L::NB, LANES = D / 8, STEP = 32 / LANES;
  const uint32_t lane = threadIdx.x & 31, item = blockIdx.x * SUMMARY_WARPS + (threadIdx.x >> 5), at = item / a.pool.n_kv_head, head = item - at * a.pool.n_kv_head;
  pdl_launch_dependents();
  pdl_wait();
  if (at >= a.n) return;
  const int32_t page = a.pages[at];
  if (page < 0) return;
  const int32_t given = a.n_tok ? a.n_tok[at] : static_cast<int32_t>(a.pool.page);
  if (static_cast<uint32_t>(page) >= a.pool.n_pages || given <= 0 || given > static_cast<int32_t>(a.pool.page)) {
    if (lane == 0) note_range(a.err);
    return;
  }
  const uint32_t n = given, c = lane % LANES / NB, b = lane % NB;
  const size_t record = static_cast<size_t>(page) * a.pool.n_kv_head + head;
  const uint8_t* k = a.pool.data + record * (a.pool.page * L::TOK);
  const uint8_t *words = k + (c * NB + b) * 4, *ds = k + L::kd(a.pool.page) + 2 * b, *ms = k + L::km(a.pool.page) + 2 * b;
  const __half2 none_hi = __float2half2_rn(-INFINITY), none_lo = __float2half2_rn(INFINITY);
  __half2 hi[4] = {none_hi, none_hi, none_hi, none_hi}, lo[4] = {none_lo, none_lo, none_lo, none_lo};
  const __half2 off = __float2half2_rn(-1024.f), off16 = __float2half2_rn(-64.f), sixteenth = __float2half2_rn(0.0625f);
#pragma unroll 4
  for (uint32_t t = lane / LANES; t < n; t += STEP) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(words + t * L::ROW), y = w >> 8;
    const __half2 d = __half2half2(__ushort_as_half(*reinterpret_cast<const uint16_t*>(ds + t * 2 * NB)));
    const __half2 m = __half2half2(__ushort_as_half(*reinterpret_cast<const uint16_t*>(ms + t * 2 * NB)));
    const __half2 v[4] = {__hfma2(__hadd2(biased(w, 0x000f000fu, a.bias), off), d, m), __hfma2(__hfma2(biased(w, 0x00f000f0u, a.bias), sixteenth, off16), d, m),
                          __hfma2(__hadd2(biased(y, 0x000f000fu, a.bias), off), d, m), __hfma2(__hfma2(biased(y, 0x00f000f0u, a.bias), sixteenth, off16), d, m)};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      hi[i] = __hmax2(hi[i], v[i]);
      lo[i] = __hmin2(lo[i], v[i]);
    }
  }
  float ends[2][8], top = 0.f;
#pragma unroll
  for (int i = 0; i < 4; i++) {
#pragma unroll
    for (uint32_t o = LANES; o < 32; o <<= 1) {
      hi[i] = __hmax2(hi[i], h2(__shfl_xor_sync(FULL, u2(hi[i]), o)));
      lo[i] = __hmin2(lo[i], h2(__shfl_xor_sync(FULL, u2(lo[i]), o)));
    }
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
};
constexpr uint32_t CHOICE_THREADS = 256, MAX_BLOCKS = 49152;

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

// A CTA per token and KV head.
template <int D>
__global__ void __launch_bounds__(CHOICE_THREADS) kv4_select_kernel(const __grid_constant__ ChoiceArgs s) {
  extern __shared__ uint32_t order[];  // scores of the token's pages as ordered numbers
  __shared__ __align__(16) uint8_t query[2 * D];
  __shared__ float tops[CHOICE_THREADS / 32];
  __shared__ uint32_t hist[256], sums[CHOICE_THREADS / 32], pick[2];
  const AttnArgs& a = s.a;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, token = blockIdx.x, head = blockIdx.y;
  pdl_launch_dependents();
  pdl_wait();
  // the token's request
  uint32_t lo = 0, hi = a.n_req + 1;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) >> 1;
    if (a.q_start[mid] <= static_cast<int>(token)) lo = mid;
    else hi = mid;
  }
  int sees = -1;
  if (lo < a.n_req && a.q_start[lo] <= static_cast<int>(token)) {
    const Lengths n = lengths_of<PLAIN>(a, lo, head == 0 && threadIdx.x == 0);
    const int i = static_cast<int>(token) - n.q0;
    if (i >= 0 && i < n.q_len) sees = max(n.kv_len - n.q_len + i + 1, 0);
  }
  const uint32_t blocks = sees > 0 ? (static_cast<uint32_t>(sees) + a.pool.page - 1) >> a.pool.log_page : 0, n = min(blocks, s.chosen);
  if (head == 0 && threadIdx.x == 0) s.keys[token] = sees < 0 ? -1 : sees - static_cast<int>((blocks - n) << a.pool.log_page);
  int32_t* out = s.pages + (static_cast<size_t>(token) * a.pool.n_kv_head + head) * s.chosen;
  const int32_t* table = a.page_table + static_cast<size_t>(lo) * a.table_stride;
  for (uint32_t i = n + threadIdx.x; i < s.chosen; i += CHOICE_THREADS) out[i] = -1;
  if (n == blocks) {
    for (uint32_t i = threadIdx.x; i < n; i += CHOICE_THREADS) out[i] = table[i];
    return;
  }
  // ---- the query in 8 bits ----
  float up = 0.f, down = 0.f;
  if (threadIdx.x < D) {
    const uint16_t* q = a.q.data + static_cast<int64_t>(token) * a.q.tok + static_cast<int64_t>(head * a.group) * a.q.head + threadIdx.x;
    for (uint32_t g = 0; g < a.group; g++) {
      const float x = a.bf ? to_f32<true>(q[g * a.q.head]) : to_f32<false>(q[g * a.q.head]);
      up += fmaxf(x, 0.f);
      down += fmaxf(-x, 0.f);
    }
  }
  float top = fmaxf(up, down);
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, o));
  if (lane == 0) tops[warp] = top;
  __syncthreads();
#pragma unroll
  for (uint32_t w = 0; w < CHOICE_THREADS / 32; w++) top = fmaxf(top, tops[w]);
  const uint32_t e = min(max(__float_as_uint(top) & 0x7f800000u, 27u << 23), 254u << 23);  // 2^-100 .. 2^127
  const float inv = __uint_as_float((261u << 23) - e);                                      // 2^(7 - e)
  if (threadIdx.x < D) {
    query[threadIdx.x] = static_cast<uint8_t>(fminf(rintf(up * inv), 255.f));
    query[D + threadIdx.x] = static_cast<uint8_t>(fminf(rintf(down * inv), 255.f));
  }
  __syncthreads();
  // ---- scores: eight lanes per page, 2 D / 8 bytes each ----
  constexpr uint32_t W = 2 * D / 32;  // words of a lane
  uint32_t mine[W];
#pragma unroll
  for (uint32_t i = 0; i < W; i++) mine[i] = reinterpret_cast<const uint32_t*>(query)[(lane & 7) * 4 + (i >> 2) * 32 + (i & 3)];
  for (uint32_t b0 = warp * 4; b0 < blocks; b0 += CHOICE_THREADS / 8) {
    const uint32_t b = b0 + (lane >> 3);
    const bool there = b < blocks;
    const uint32_t page = there ? static_cast<uint32_t>(table[b]) : 0u;
    const bool good = page < a.pool.n_pages;
    int sum = 0;
    float scale = 0.f;
    if (there && good) {
      const size_t record = static_cast<size_t>(page) * a.pool.n_kv_head + head;
      const uint4* codes = reinterpret_cast<const uint4*>(s.codes + record * 2 * D);
      scale = s.scales[record];
#pragma unroll
      for (uint32_t i = 0; i < W / 4; i++) {
        const uint4 v = codes[(lane & 7) + 8 * i];
        sum = dot4(mine[4 * i], v.x, sum);
        sum = dot4(mine[4 * i + 1], v.y, sum);
        sum = dot4(mine[4 * i + 2], v.z, sum);
        sum = dot4(mine[4 * i + 3], v.w, sum);
      }
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(FULL, sum, o);
    if (there && (lane & 7) == 0) {
      if (!good) note_range(a.err);
      order[b] = b < s.first || b >= blocks - s.last ? 0xffffffffu : good ? ordered(static_cast<float>(sum) * scale) : 0u;
    }
  }
  __syncthreads();
  // ---- the n-th highest: digit by digit ----
  uint32_t prefix = 0, mask = 0, want = n;  // of those whose bits under mask are prefix, the want-th is looked for
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (uint32_t i = threadIdx.x; i < 256; i += CHOICE_THREADS) hist[i] = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < blocks; i += CHOICE_THREADS) {
      const uint32_t x = order[i];
      if ((x & mask) == prefix) atomicAdd(&hist[x >> shift & 255], 1);
    }
    __syncthreads();
    // thread t: those with the digit 255 - t or a higher one
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
    }
    __syncthreads();
    prefix |= pick[0] << shift;
    mask |= 255u << shift;
    want = pick[1];
    __syncthreads();
  }
  // ---- in the order of the keys: those above, and the first `want` of those equal ----
  uint32_t done_above = 0, done_equal = 0;
  for (uint32_t b0 = 0; b0 < blocks; b0 += CHOICE_THREADS) {
    const uint32_t b = b0 + threadIdx.x, x = b < blocks ? order[b] : 0u;
    const bool above = b < blocks && x > prefix, equal = b < blocks && x == prefix;
    const uint32_t am = __ballot_sync(FULL, above), em = __ballot_sync(FULL, equal), under = (1u << lane) - 1;
    if (lane == 0) sums[warp] = __popc(am) | __popc(em) << 16;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (uint32_t w = 0; w < CHOICE_THREADS / 32; w++) {
      if (w == warp) before = all;
      all += sums[w];
    }
    const uint32_t a_at = done_above + (before & 0xffff) + __popc(am & under), e_at = done_equal + (before >> 16) + __popc(em & under);
    if (above || (equal && e_at < want)) out[a_at + min(e_at, want)] = table[b];
    done_above += all & 0xffff;
    done_equal += all >> 16;
    __syncthreads();
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
  const dim3 grid((n * p.n_kv_head + SUMMARY_WARPS - 1) / SUMMARY_WARPS);
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
  BP_TRY(c, bp_launch(true, pool->head_dim == 128 ? kv4_select_kernel<128> : kv4_select_kernel<64>, dim3(in->total_q, p.n_kv_head), dim3(CHOICE_THREADS), blocks * 4,
                      static_cast<cudaStream_t>(stream), s));
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
