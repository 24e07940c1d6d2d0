// Attention of requests behind prefixes that several of them have in common (include/bonsai_pages.h).
//
// The keys that a query sees are those of its prefix and its request's own. With o_i = sum of 2^(s - m_i) v, l_i = sum of 2^(s - m_i) and m_i = the
// largest score (log2 units) over part i of the keys, the output is sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i, m = max(m_1, m_2). The first part is
// a prefix whose rows are those of all its requests, so that its codes are read and expanded once for all of them; the second is each request's own. Both are the attention
// kernels' (bp_kv4_attention.cu, bp_kv4_prefill.cu), which leave (o, m, l) in the caller's work memory in 32 bits; the kernel here joins them.
#include "bp_kv4_attention.cuh"
#include "bp_paged_host.cuh"

namespace {

using namespace bp;
using namespace bp::kv4;
using namespace bp::paged;

struct JoinArgs {
  const float *prefix, *own;
  const float2 *prefix_ml, *own_ml;
  const int32_t *q_start, *prefix_start;
  uint32_t n_prefix;
  AttnArgs a;  // of the own keys' launch: where the outputs go, what the lengths are cut to
};
constexpr uint32_t JOIN_THREADS = 256;

// The last i of n with begin[i] <= x, or -1.
__device__ __forceinline__ int last_begun(const int32_t* begin, uint32_t n, int x) {
  int lo = -1, hi = static_cast<int>(n);
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (begin[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// A warp per row.
template <int D>
__global__ void __launch_bounds__(JOIN_THREADS) kv4_join_kernel(const __grid_constant__ JoinArgs j) {
  constexpr int V = D / 32;  // dims of a lane
  const AttnArgs& a = j.a;
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t row = static_cast<uint64_t>(blockIdx.x) * (JOIN_THREADS / 32) + (threadIdx.x >> 5);
  pdl_launch_dependents();
  pdl_wait();
  if (row >= static_cast<uint64_t>(a.total_q) * a.n_head) return;
  const uint32_t token = static_cast<uint32_t>(row / a.n_head), head = static_cast<uint32_t>(row) - token * a.n_head;
  const int r = last_begun(j.q_start, a.n_req + 1, static_cast<int>(token));
  if (r < 0 || r >= static_cast<int>(a.n_req)) return;  // a row of no request
  const Lengths n = lengths_of<OWN>(a, r, false);
  if (static_cast<int>(token) >= n.q0 + n.q_len) return;  // (cut, and reported)
  const int g = last_begun(j.prefix_start, j.n_prefix + 1, r);
  const float2 none = make_float2(NEG_BIG, 0.f);
  const float2 x = g >= 0 && g < static_cast<int>(j.n_prefix) ? j.prefix_ml[row] : none, y = j.own_ml[row];
  const float m = fmaxf(x.x, y.x), wx = x.y == 0.f ? 0.f : ex2(x.x - m), wy = y.y == 0.f ? 0.f : ex2(y.x - m), l = wx * x.y + wy * y.y;
  float o[V] = {};
  // (a part without weights has not been written)
  if (x.y != 0.f) {
#pragma unroll
    for (int i = 0; i < V; i++) o[i] = wx * j.prefix[row * D + V * lane + i];
  }
  if (y.y != 0.f) {
#pragma unroll
    for (int i = 0; i < V; i++) o[i] = fmaf(wy, j.own[row * D + V * lane + i], o[i]);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint16_t* out = a.out.data + static_cast<int64_t>(token) * a.out.tok + static_cast<int64_t>(head) * a.out.head + V * lane;
  if constexpr (V == 4) {
    store4(a.bf, out, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
  } else {
    const uint32_t h = a.bf ? pack2<true>(o[0] * inv, o[1] * inv) : pack2<false>(o[0] * inv, o[1] * inv);
    out[0] = static_cast<uint16_t>(h);
    out[1] = static_cast<uint16_t>(h >> 16);
  }
}

}  // namespace

extern "C" {

uint64_t bp_kv4_shared_work(uint32_t total_q, uint32_t n_head, uint32_t head_dim) {
  return 2 * static_cast<uint64_t>(total_q) * n_head * (static_cast<uint64_t>(head_dim) + 2);
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
  // units of 64 keys of 8 rows, and what an item of the kernel for many queries costs besides, are counted in 32 bits
  const uint64_t rows8 = static_cast<uint64_t>(in->total_q) * (in->n_head / p.n_kv_head) / 8;
  if ((rows8 + in->n_req) * p.n_kv_head > 0xffffffffull / (in->max_kv / 64 + 8) || (rows8 + in->n_prefix) * p.n_kv_head > 0xffffffffull / (in->max_prefix / 64 + 8))
    return fail_config(c, "total_q * n_head * max_kv or max_prefix is too large for one call");
  if (!rq.data || !ro.data || !in->q_start || !in->kv_len || !in->work || (in->max_kv != 0 && (!p.data || !in->page_table)) ||
      (in->n_prefix != 0 && (!in->prefix_start || !in->prefix_len || (in->max_prefix != 0 && (!p.data || !in->prefix_table)))))
    return fail(c, BP_ERR_NULL, "null pointer argument");
  OnDevice on(c->device);
  BP_TRY(c, on.err);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const size_t rows = static_cast<size_t>(in->total_q) * in->n_head;
  float* work = static_cast<float*>(in->work);
  AttnArgs a;
  bp_kv4_attention_args(c, dtype == BP_DTYPE_BF16, p, in->q, in->out, in->n_head, in->scale, &a);
  a.q_start = static_cast<const int32_t*>(in->q_start);
  a.total_q = in->total_q;
  JoinArgs j = {};
  j.prefix = work;
  j.own = work + rows * pool->head_dim;
  j.prefix_ml = reinterpret_cast<float2*>(work + 2 * rows * pool->head_dim);
  j.own_ml = j.prefix_ml + rows;
  j.q_start = a.q_start;
  j.prefix_start = static_cast<const int32_t*>(in->prefix_start);
  j.n_prefix = in->n_prefix;
  if (in->n_prefix != 0) {
    AttnArgs x = a;
    x.kv_len = static_cast<const int32_t*>(in->prefix_len);
    x.page_table = static_cast<const int32_t*>(in->prefix_table);
    x.prefix_start = j.prefix_start;
    x.n_all = in->n_req;
    x.n_req = in->n_prefix;
    x.max_q = in->total_q;
    x.max_kv = in->max_prefix;
    x.table_stride = in->prefix_stride;
    x.table_pages = bp_kv4_table_pages(p, in->prefix_stride);
    x.part = const_cast<float*>(j.prefix);
    x.part_ml = const_cast<float2*>(j.prefix_ml);
    BP_TRY(c, bp_launch_kv4_rows(c, s, pool->head_dim, PREFIX, (static_cast<uint64_t>(in->total_q) * a.group + in->n_prefix - 1) / in->n_prefix, x));
  }
  a.kv_len = static_cast<const int32_t*>(in->kv_len);
  a.page_table = static_cast<const int32_t*>(in->page_table);
  a.n_req = in->n_req;
  a.max_q = in->max_q < in->total_q ? in->max_q : in->total_q;
  a.max_kv = in->max_kv;
  a.table_stride = in->table_stride;
  a.table_pages = bp_kv4_table_pages(p, in->table_stride);
  a.part = const_cast<float*>(j.own);
  a.part_ml = const_cast<float2*>(j.own_ml);
  BP_TRY(c, bp_launch_kv4_rows(c, s, pool->head_dim, OWN, static_cast<uint64_t>(a.max_q) * a.group, a));
  j.a = a;
  const dim3 grid(static_cast<uint32_t>((rows + JOIN_THREADS / 32 - 1) / (JOIN_THREADS / 32)));
  BP_TRY(c, bp_launch(true, pool->head_dim == 128 ? kv4_join_kernel<128> : kv4_join_kernel<64>, grid, dim3(JOIN_THREADS), 0, s, j));
  return BP_OK;
}

}  // extern "C"
