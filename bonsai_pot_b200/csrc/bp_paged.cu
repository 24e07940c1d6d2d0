// Host side of the paged 4-bit cache operators (include/bonsai_paged.h): the context, the checks of the arguments, errors.
#include <string.h>

#include <new>

#include "bp_kv4_attention.cuh"
#include "bp_paged_host.cuh"

using namespace bp;
using namespace bp::paged;

extern "C" {

int bp_paged_create(int32_t device, bp_paged_ctx** out) {
  if (!out) return BP_ERR_NULL;
  *out = nullptr;
  bp_paged_ctx* c = new (std::nothrow) bp_paged_ctx();
  if (!c) return BP_ERR_CUDA;
  memset(c, 0, sizeof *c);
  *out = c;
  int n_dev = 0;
  cudaError_t e = cudaGetDeviceCount(&n_dev);
  if (e != cudaSuccess || n_dev == 0) return fail(c, BP_ERR_CUDA, "no CUDA device: this library has no CPU path");
  if (device < 0 || device >= n_dev) return fail_config(c, "device ordinal out of range");
  c->device = device;
  OnDevice on(device);
  BP_TRY(c, on.err);
  int major = 0;
  BP_TRY(c, cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device));
  if (major != 10) return fail(c, BP_ERR_CUDA, "this library is built for sm_100a (B200) only");
  BP_TRY(c, cudaDeviceGetAttribute(&c->sm_count, cudaDevAttrMultiProcessorCount, device));
  BP_TRY(c, bp_kv4_attention_init(c));
  BP_TRY(c, bp_kv4_prefill_init(c));
  BP_TRY(c, bp_pages_init(c));
  BP_TRY(c, bp_kv4_select_init(c));
  BP_TRY(c, cudaHostAlloc(&c->err_host, 2 * sizeof(uint32_t), cudaHostAllocMapped));
  c->err_host[0] = c->err_host[1] = 0;
  void* dev = nullptr;
  BP_TRY(c, cudaHostGetDevicePointer(&dev, c->err_host, 0));
  // the counters' zeros are written on the legacy stream, for which a first call's stream need not wait
  BP_TRY(c, cudaStreamSynchronize(cudaStreamLegacy));
  c->err_dev = static_cast<uint32_t*>(dev);
  return BP_OK;
}

void bp_paged_destroy(bp_paged_ctx* c) {
  if (!c) return;
  {
    OnDevice on(c->device);
    if (on.err == cudaSuccess) {
      if (c->partials) (void)cudaFree(c->partials);  // waits for launches that still use it
      if (c->prefill_partials) (void)cudaFree(c->prefill_partials);
      if (c->counters) (void)cudaFree(c->counters);
      if (c->page_counter) (void)cudaFree(c->page_counter);
      if (c->err_host) (void)cudaFreeHost(c->err_host);
    }
  }
  delete c;
}

const char* bp_paged_last_error(const bp_paged_ctx* c) { return c ? c->msg : ""; }

int bp_paged_status(bp_paged_ctx* c, void* stream) {
  if (int s = enter(c)) return s;
  OnDevice on(c->device);
  BP_TRY(c, on.err);
  BP_TRY(c, cudaStreamSynchronize(static_cast<cudaStream_t>(stream)));
  if (int s = enter(c)) return s;
  volatile uint32_t* word = c->err_host;
  if (word[0] != 0) {
    word[0] = 0;
    return fail(c, BP_ERR_CONTEXT_OVERFLOW, "context overflow: a position, slot, page id or number of keys lay outside its table or pool");
  }
  return BP_OK;
}

int bp_rope_fill(bp_paged_ctx* c, void* stream, const bp_rope_config* cfg, void* table_out) {
  if (int s = enter(c)) return s;
  if (!cfg || !table_out) return fail(c, BP_ERR_NULL, "null pointer argument");
  if (cfg->rot_dim < 2 || cfg->rot_dim % 2 || cfg->rot_dim > 256) return fail_config(c, "rot_dim must be even, 2 .. 256");
  if (cfg->n_pos == 0) return fail_config(c, "n_pos must be > 0");
  if (!(cfg->freq_base > 0.0f)) return fail_config(c, "freq_base must be > 0");
  if (cfg->scaling > BP_ROPE_SCALE_YARN) return fail_config(c, "unknown RoPE scaling");
  if (cfg->scaling != BP_ROPE_SCALE_NONE && !(cfg->factor >= 1.0f)) return fail_config(c, "a RoPE scaling factor must be >= 1");
  if (cfg->scaling == BP_ROPE_SCALE_NTK && cfg->rot_dim == 2) return fail_config(c, "BP_ROPE_SCALE_NTK needs rot_dim > 2");
  if (cfg->scaling == BP_ROPE_SCALE_YARN && (cfg->orig_ctx == 0 || !(cfg->beta_fast > cfg->beta_slow) || !(cfg->beta_slow > 0.0f) || !(cfg->freq_base > 1.0f)))
    return fail_config(c, "BP_ROPE_SCALE_YARN needs orig_ctx, freq_base > 1 and beta_fast > beta_slow > 0");
  if (!aligned_to(table_out, 8)) return fail_config(c, "a RoPE table must be 8-byte aligned");
  OnDevice on(c->device);
  BP_TRY(c, on.err);
  BP_TRY(c, bp_launch_rope_fill(static_cast<cudaStream_t>(stream), *cfg, static_cast<float2*>(table_out)));
  return BP_OK;
}

int bp_rope(bp_paged_ctx* c, void* stream, uint32_t dtype, const bp_rows* x, const bp_rows* out, uint32_t n_tok, uint32_t n_head,
            uint32_t head_dim, const void* positions, const bp_rope_table* table, const void* w_norm, float eps, uint32_t inverse) {
  if (int s = enter(c)) return s;
  if (!x || !out || !table) return fail(c, BP_ERR_NULL, "null pointer argument");
  if (dtype > BP_DTYPE_BF16) return fail_config(c, "the activation type must be BP_DTYPE_F16 or BP_DTYPE_BF16");
  if (head_dim < 2 || head_dim % 2 || head_dim > 256) return fail_config(c, "head_dim must be even, 2 .. 256");
  if (n_head == 0) return fail_config(c, "n_head must be > 0");
  if (w_norm && !(eps >= 0.0f)) return fail_config(c, "eps must be >= 0");
  Rows rx, ro;
  Rope rope;
  BP_CHECK(c, check_rows(x, &rx));
  BP_CHECK(c, check_rows(out, &ro));
  BP_CHECK(c, check_table(table, head_dim, &rope));
  if (!aligned_to(positions, 4) || !aligned_to(w_norm, 2)) return fail_config(c, "positions must be 4-byte, a norm weight 2-byte aligned");
  if (n_tok == 0) return BP_OK;
  if (!rx.data || !ro.data || !positions || !rope.table) return fail(c, BP_ERR_NULL, "null pointer argument");
  if (static_cast<uint64_t>(n_tok) * n_head > 1ull << 28) return fail_config(c, "n_tok * n_head must be <= 2^28");
  OnDevice on(c->device);
  BP_TRY(c, on.err);
  BP_TRY(c, bp_launch_rope(c, static_cast<cudaStream_t>(stream), dtype == BP_DTYPE_BF16, rx, ro, n_tok, n_head, head_dim,
                           static_cast<const int32_t*>(positions), rope, static_cast<const uint16_t*>(w_norm), eps, inverse != 0));
  return BP_OK;
}

uint64_t bp_kv4_pool_bytes(const bp_kv4_pool* pool) {
  Pool p;
  if (!pool) return 0;
  bp_kv4_pool shape = *pool;
  shape.data = nullptr;
  if (check_pool(&shape, &p)) return 0;
  return static_cast<uint64_t>(pool->n_pages) * pool->n_kv_head * pool->page_tokens * pool->head_dim * 5 / 4;
}

int bp_kv4_append(bp_paged_ctx* c, void* stream, uint32_t dtype, const bp_kv4_pool* pool, const bp_rows* k, const bp_rows* v,
                  uint32_t n_tok, const void* positions, const void* slots, const bp_rope_table* table, const void* w_k_norm, float eps) {
  if (int s = enter(c)) return s;
  if (!pool || !k || !v) return fail(c, BP_ERR_NULL, "null pointer argument");
  if (dtype > BP_DTYPE_BF16) return fail_config(c, "the activation type must be BP_DTYPE_F16 or BP_DTYPE_BF16");
  if (w_k_norm && !(eps >= 0.0f)) return fail_config(c, "eps must be >= 0");
  Rows rk, rv;
  Pool p;
  Rope rope = {};
  BP_CHECK(c, check_pool(pool, &p));
  BP_CHECK(c, check_rows(k, &rk));
  BP_CHECK(c, check_rows(v, &rv));
  if (table) BP_CHECK(c, check_table(table, pool->head_dim, &rope));
  if (!aligned_to(positions, 4) || !aligned_to(slots, 8) || !aligned_to(w_k_norm, 2))
    return fail_config(c, "positions must be 4-byte, slots 8-byte, a norm weight 2-byte aligned");
  if (n_tok == 0) return BP_OK;
  if (!p.data || !rk.data || !rv.data || !slots || (table && (!positions || !rope.table))) return fail(c, BP_ERR_NULL, "null pointer argument");
  if (static_cast<uint64_t>(n_tok) * p.n_kv_head > 0x7fffffffull) return fail_config(c, "n_tok * n_kv_head must be < 2^31");
  OnDevice on(c->device);
  BP_TRY(c, on.err);
  BP_TRY(c, bp_launch_kv4_append(c, static_cast<cudaStream_t>(stream), dtype == BP_DTYPE_BF16, p, pool->head_dim, rk, rv, n_tok,
                                 static_cast<const int32_t*>(positions), static_cast<const int64_t*>(slots), rope,
                                 static_cast<const uint16_t*>(w_k_norm), eps));
  return BP_OK;
}

int bp_kv4_read(bp_paged_ctx* c, void* stream, uint32_t dtype, const bp_kv4_pool* pool, const void* slots, uint32_t n_tok,
                const bp_rows* k, const bp_rows* v) {
  if (int s = enter(c)) return s;
  if (!pool || !k || !v) return fail(c, BP_ERR_NULL, "null pointer argument");
  if (dtype > BP_DTYPE_BF16) return fail_config(c, "the activation type must be BP_DTYPE_F16 or BP_DTYPE_BF16");
  Rows rk, rv;
  Pool p;
  BP_CHECK(c, check_pool(pool, &p));
  BP_CHECK(c, check_rows(k, &rk));
  BP_CHECK(c, check_rows(v, &rv));
  if (!aligned_to(slots, 8)) return fail_config(c, "slots must be 8-byte aligned");
  if (n_tok == 0) return BP_OK;
  if (!p.data || !rk.data || !rv.data || !slots) return fail(c, BP_ERR_NULL, "null pointer argument");
  if (static_cast<uint64_t>(n_tok) * p.n_kv_head > 0x7fffffffull) return fail_config(c, "n_tok * n_kv_head must be < 2^31");
  OnDevice on(c->device);
  BP_TRY(c, on.err);
  BP_TRY(c, bp_launch_kv4_read(c, static_cast<cudaStream_t>(stream), dtype == BP_DTYPE_BF16, p, pool->head_dim,
                               static_cast<const int64_t*>(slots), n_tok, rk, rv));
  return BP_OK;
}

int bp_kv4_attention(bp_paged_ctx* c, void* stream, uint32_t dtype, const bp_kv4_pool* pool, const bp_kv4_attn* a) {
  if (int s = enter(c)) return s;
  if (!pool || !a) return fail(c, BP_ERR_NULL, "null pointer argument");
  if (dtype > BP_DTYPE_BF16) return fail_config(c, "the activation type must be BP_DTYPE_F16 or BP_DTYPE_BF16");
  Rows rq, ro;
  Pool p;
  BP_CHECK(c, check_pool(pool, &p));
  BP_CHECK(c, check_rows(&a->q, &rq));
  BP_CHECK(c, check_rows(&a->out, &ro));
  if (a->n_head == 0 || a->n_head % p.n_kv_head) return fail_config(c, "n_head must be a multiple of n_kv_head");
  if (a->scale != a->scale) return fail_config(c, "scale must be a number");
  if (!aligned_to(a->q_start, 4) || !aligned_to(a->kv_len, 4) || !aligned_to(a->page_table, 4))
    return fail_config(c, "q_start, kv_len and page_table must be 4-byte aligned");
  if (a->n_req == 0 || a->total_q == 0 || a->max_q == 0) return BP_OK;
  if (a->n_req > 65535) return fail_config(c, "at most 65535 requests");
  if (static_cast<uint64_t>(a->total_q) * a->n_head > 0x7fffffffull || a->max_kv > 0x7fffff00u) return fail_config(c, "total_q * n_head and max_kv must be < 2^31");
  // units of 64 keys of 8 rows, and what an item of the kernel for many queries costs besides, are counted in 32 bits
  const uint64_t tiles = static_cast<uint64_t>(a->total_q) * (a->n_head / p.n_kv_head) / 8 + a->n_req;
  if (tiles * p.n_kv_head > 0xffffffffull / (a->max_kv / 64 + 8)) return fail_config(c, "total_q * n_head * max_kv is too large for one call");
  if (!rq.data || !ro.data || !a->q_start || !a->kv_len || (a->max_kv != 0 && (!p.data || !a->page_table))) return fail(c, BP_ERR_NULL, "null pointer argument");
  OnDevice on(c->device);
  BP_TRY(c, on.err);
  BP_TRY(c, bp_launch_kv4_attention(c, static_cast<cudaStream_t>(stream), dtype == BP_DTYPE_BF16, p, pool->head_dim, *a));
  return BP_OK;
}

}  // extern "C"
