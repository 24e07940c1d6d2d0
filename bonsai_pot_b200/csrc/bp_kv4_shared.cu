// Attention of requests behind prefixes that several of them have in common (include/bonsai_pages.h).
//
// The keys that a query sees are those of its prefix and its request's own. With o_i = sum of 2^(s - m_i) v, l_i = sum of 2^(s - m_i) and m_i near the
// largest score s (log2 units) over part i of the keys, the output is sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i, m = the largest m_i. Prefixes are items whose rows
// are those of all their requests, so that their codes are read and expanded once for all of them; own keys are items of each request. Both are the attention
// kernels' (bp_kv4_attention.cu, bp_kv4_prefill.cu), which leave (o, m, l) of whole items in the caller's work memory and of pieces of items in the context's, in 32 bits;
// the kernel here joins them all, in the order of the keys.
//
// Floors: prefix and own keys once, 6.2 us for 64 tokens behind two prefixes of up to 8191 keys (32 / 8 heads of 128, up to 1000 keys of their own), the products, 220 us for 4 chunks of up to 512
// behind 16384. Measured 43.5 and 434 us, 16.9 for 8 tokens behind 2048 keys (bp_kv4_attention over the same keys in rows of pages for each request: 116, 403 and 19.1).
// Bound by the attention kernels' beginnings and ends and, of chunks, by their softmax. One launch after the other, each joining its items by the CTA that comes last, took 92, 513 and 31; chunks
// in parts 444.
#include "bp_kv4_attention.cuh"
#include "bp_paged_host.cuh"

namespace {

using namespace bp;
using namespace bp::kv4;
using namespace bp::paged;

struct JoinArgs {
  AttnArgs a;  // lengths of both parts, outputs
  const float* slots[2];             // pieces of prefixes, of own keys
  uint32_t piece[2], ctas[2], rows[2];  // floats of a piece, CTAs that have some, rows of one
};
// Rows of a request (on the average) times head_dim above which it has no need to share the expansion of its prefix's codes: its own rows fill a CTA's query tiles, and its keys are its prefix's
// and its own in one item, without parts. us, in one item / in parts:
//   head_dim 128, 32 / 8 heads        128 rows  256      512      1024         head_dim 64, 40 / 8 heads  160 rows  320      640      1280
//   4 requests behind 16384 keys      76/58     101/95   149/154  218/216                                 84/66     114/87   163/139  290/311
//   16 behind 4096                    76/64     100/93   143/155  212/247                                 86/72     107/86   130/124  175/190
//   4 behind 1000                     23/24     34/29    35/38    47/63                                   24/21     27/30    32/38    36/51
constexpr uint64_t BEHIND_VALUES = 57344;
constexpr uint32_t JOIN_THREADS = 256;

// A warp per row, N pieces of it on their way.
template <int D, int N>
__global__ void __launch_bounds__(JOIN_THREADS, N > 4 ? 3 : 6) kv4_join_kernel(const __grid_constant__ JoinArgs j) {
  const AttnArgs& a = j.a;
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t row = static_cast<uint64_t>(blockIdx.x) * (JOIN_THREADS / 32) + (threadIdx.x >> 5);
  pdl_launch_dependents();
  pdl_wait();
  if (row >= static_cast<uint64_t>(a.total_q) * a.n_head) return;
  const uint32_t token = static_cast<uint32_t>(row / a.n_head), head = static_cast<uint32_t>(row) - token * a.n_head;
  // where the pieces of either part are (asked for before it is known whether there is anything)
  const float* record[2] = {a.part + row * RECORD<D>, a.part + (static_cast<size_t>(a.total_q) * a.n_head + row) * RECORD<D>};
  const uint4 ends[2] = {*reinterpret_cast<const uint4*>(record[0] + D), *reinterpret_cast<const uint4*>(record[1] + D)};
  const int r = last_begun(a.q_start, a.n_own + 1, static_cast<int>(token), lane);
  if (r < 0 || r >= static_cast<int>(a.n_own)) return;  // a row of no request
  const int g = a.n_prefix ? last_begun(a.prefix_start, a.n_prefix + 1, r, lane) : -1;  // (without prefixes there may be no list of them)
  const Lengths own = lengths_of<PARTS>(a, a.n_prefix + r, false);
  if (static_cast<int>(token) >= own.q0 + own.q_len) return;  // (cut, and reported)
  const bool some = g >= 0 && g < static_cast<int>(a.n_prefix);
  uint32_t n[2], c[2], at[2];
  float2 first[2];
#pragma unroll
  for (int p = 0; p < 2; p++) {
    const bool none = p == 0 && !some;
    first[p] = none ? make_float2(NEG_BIG, 0.f) : make_float2(__uint_as_float(ends[p].x), __uint_as_float(ends[p].y));
    c[p] = ends[p].z;
    n[p] = none ? 0 : ends[p].w >> 16;
    at[p] = ends[p].w & 0xffff;
    // (after a wait that gave up nobody may have written this)
    if (n[p] != 0 && (n[p] > j.ctas[p] || c[p] > j.ctas[p] - n[p] || at[p] >= j.rows[p])) return;
  }
  const uint32_t n0 = max(n[0], 1u), all = n0 + max(n[1], 1u);
  auto piece = [&](uint32_t k) -> const float* {
    const int p = k >= n0;
    if (n[p] == 0) return record[p];
    return j.slots[p] + static_cast<size_t>(piece_at(c[p], k - (p ? n0 : 0))) * j.piece[p] + at[p] * RECORD<D>;
  };
  RowJoin<D> join;
  for (uint32_t k0 = 0; k0 < all; k0 += 32) {
    const uint32_t k = k0 + lane;
    // (a record without weights may not have been written, pieces have)
    const bool there = k < all && !(n[k >= n0] == 0 && first[k >= n0].y == 0.f);
    join.template add<N>(__ballot_sync(FULL, there), piece(min(k, all - 1)), lane);
  }
  join.put(a.bf, a.out.data + static_cast<int64_t>(token) * a.out.tok + static_cast<int64_t>(head) * a.out.head, lane);
}

}  // namespace

extern "C" {

uint64_t bp_kv4_shared_work(uint32_t total_q, uint32_t n_head, uint32_t head_dim) {
  return 2 * static_cast<uint64_t>(total_q) * n_head * (static_cast<uint64_t>(head_dim) + 4);
}

int bp_kv4_attention_shared(bp_paged_ctx* c, void* stream, uint32_t dtype, const bp_kv4_pool* pool, const bp_kv4_shared* in) {
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
  if (!aligned_to(in->q_start, 4) || !aligned_to(in->kv_len, 4) || !aligned_to(in->page_table, 4) || !aligned_to(in->prefix_start, 4) || !aligned_to(in->prefix_len, 4) ||
      !aligned_to(in->prefix_table, 4))
    return fail_config(c, "q_start, kv_len, page_table and the same of the prefixes must be 4-byte aligned");
  if (!aligned_to(in->work, 16)) return fail_config(c, "work must be 16-byte aligned");
  if (in->n_req == 0 || in->total_q == 0 || in->max_q == 0) return BP_OK;
  if (in->n_req > 65535 || in->n_prefix > 65535) return fail_config(c, "at most 65535 requests and prefixes");
  if (static_cast<uint64_t>(in->total_q) * in->n_head > 0x7fffffffull || in->max_kv > 0x7fffff00u || in->max_prefix > 0x7fffff00u)
    return fail_config(c, "total_q * n_head, max_kv and max_prefix must be < 2^31");
  // Units of 64 keys of 8 rows, and what an item of the kernel for many queries costs besides, are counted in 32 bits, those of both parts together. (Prefix and own keys in one
  // item are no more: that is for hundreds of rows per request, of which an item has 128 or 256.)
  const uint64_t rows8 = static_cast<uint64_t>(in->total_q) * (in->n_head / p.n_kv_head) / 8, cost = 1 + BP_KV4_ITEM_COST_IN_PARTS;
  if ((rows8 + in->n_req) * p.n_kv_head * (in->max_kv / 64 + cost) + (rows8 + in->n_prefix) * p.n_kv_head * (in->max_prefix / 64 + cost) > 0xffffffffull)  // (no more than 2^59 each)
    return fail_config(c, "total_q * n_head * max_kv or max_prefix is too large for one call");
  if (!rq.data || !ro.data || !in->q_start || !in->kv_len || !in->work || (in->max_kv != 0 && (!p.data || !in->page_table)) ||
      (in->n_prefix != 0 && (!in->prefix_start || !in->prefix_len || (in->max_prefix != 0 && (!p.data || !in->prefix_table)))))
    return fail(c, BP_ERR_NULL, "null pointer argument");
  OnDevice on(c->device);
  BP_TRY(c, on.err);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  JoinArgs j = {};
  AttnArgs& a = j.a;
  bp_kv4_attention_args(c, dtype == BP_DTYPE_BF16, p, in->q, in->out, in->n_head, in->scale, &a);
  a.q_start = static_cast<const int32_t*>(in->q_start);
  a.kv_len = static_cast<const int32_t*>(in->kv_len);
  a.page_table = static_cast<const int32_t*>(in->page_table);
  a.total_q = in->total_q;
  a.max_q = in->max_q < in->total_q ? in->max_q : in->total_q;
  a.max_kv = in->max_kv;
  a.table_stride = in->table_stride;
  a.table_pages = bp_kv4_table_pages(p, in->table_stride);
  a.prefix_start = static_cast<const int32_t*>(in->prefix_start);
  a.prefix_len = static_cast<const int32_t*>(in->prefix_len);
  a.prefix_table = static_cast<const int32_t*>(in->prefix_table);
  a.n_prefix = in->n_prefix;
  a.n_own = in->n_req;
  a.n_req = in->n_prefix + in->n_req;
  a.max_prefix = in->max_prefix;
  a.prefix_stride = in->prefix_stride;
  a.prefix_pages = bp_kv4_table_pages(p, in->prefix_stride);
  a.part = static_cast<float*>(in->work);
  // rows of a prefix (on the average) and of a request, by which either part goes to the kernel for few rows or the one for many; without any key there are only zeros
  const uint64_t own_rows = static_cast<uint64_t>(a.max_q) * a.group, prefix_rows = in->n_prefix ? (static_cast<uint64_t>(in->total_q) * a.group + in->n_prefix - 1) / in->n_prefix : 0;
  const bool own_many = in->max_kv != 0 && own_rows > BP_KV4_FEW_ROWS, prefix_many = in->max_prefix != 0 && prefix_rows > BP_KV4_FEW_ROWS;
  const uint32_t D = pool->head_dim;
  const uint64_t more = own_rows > prefix_rows ? own_rows : prefix_rows;
  const uint64_t average = static_cast<uint64_t>(in->total_q) * a.group / in->n_req;
  if (own_many && average * D > BEHIND_VALUES && static_cast<uint64_t>(in->max_prefix) + in->max_kv <= 0x7fffff00u) {
    a.n_req = a.n_own;
    BP_TRY(c, bp_launch_kv4_prefill(c, s, D, BEHIND, own_rows, 0, a));
    return BP_OK;
  }
  if (own_many || !prefix_many) {  // one launch for both
    BP_TRY(c, own_many ? bp_launch_kv4_prefill(c, s, D, PARTS, more, 0, a, &j.slots[0], &j.piece[0]) : bp_launch_kv4_few_rows(c, s, D, PARTS, more, 0, a, &j.slots[0], &j.piece[0]));
    j.slots[1] = j.slots[0];
    j.piece[1] = j.piece[0];
    j.ctas[0] = j.ctas[1] = c->sm_count;
  } else {
    // Side by side, each on its share of the SMs: what a tile of 64 keys takes there (1.2 us of 256 rows, 0.9 of 128) against 0.15 us for a unit of 64 keys of 128 dims here
    // (0.18, but requests are shorter than the longest), by the lengths that the caller says; a unit counts once, whatever a request's rows. 64 tokens, own keys up to 1000, behind 8191 and 5000:
    // 61 us with max_kv 1000, 98 with 8192, 122 with 32768; 16 requests of 5 tokens (20 rows) behind 8191: 123, most of it the own keys'.
    const float prefix_tiles = static_cast<float>(in->n_prefix) * p.n_kv_head * ((prefix_rows + 255) / 256) * (in->max_prefix / 64 + 6);
    const float prefix_cost = prefix_tiles * (prefix_rows > 128 ? 1.2f : 0.9f), own_cost = static_cast<float>(in->n_req) * p.n_kv_head * (in->max_kv / 64 + 1) * (0.15f / 128) * D;
    const float part = prefix_cost / (prefix_cost + own_cost);
    const int sms = c->sm_count, most = sms - sms / 8;
    int here = static_cast<int>(part * sms + 0.5f);
    here = here < sms / 8 ? sms / 8 : here > most ? most : here;
    AttnArgs x = a;
    x.first = 1;
    x.n_req = x.n_prefix;
    BP_TRY(c, bp_launch_kv4_prefill(c, s, D, PARTS, prefix_rows, here, x, &j.slots[0], &j.piece[0]));
    x = a;
    x.beside = 1;
    x.n_req = x.n_own;
    x.n_prefix = 0;
    BP_TRY(c, bp_launch_kv4_few_rows(c, s, D, PARTS, own_rows, sms - here, x, &j.slots[1], &j.piece[1]));
    j.ctas[0] = here;
    j.ctas[1] = sms - here;
  }
  j.rows[0] = j.piece[0] / (D + 4);
  j.rows[1] = j.piece[1] / (D + 4);
  const uint64_t rows = static_cast<uint64_t>(in->total_q) * in->n_head;
  const dim3 grid(static_cast<uint32_t>((rows + JOIN_THREADS / 32 - 1) / (JOIN_THREADS / 32)));
  // Many rows want many warps per SM (42400 of them: 25 us with 40 registers, 32 with 70), few rows many loads per warp (2048 behind prefixes: 41.6 us in all, 46.9).
  const bool many = rows > 48ull * c->sm_count;
  auto* kernel = D == 128 ? (many ? kv4_join_kernel<128, 4> : kv4_join_kernel<128, 8>) : many ? kv4_join_kernel<64, 4> : kv4_join_kernel<64, 8>;
  BP_TRY(c, bp_launch(true, kernel, grid, dim3(JOIN_THREADS), 0, s, j));
  return BP_OK;
}

}  // extern "C"
