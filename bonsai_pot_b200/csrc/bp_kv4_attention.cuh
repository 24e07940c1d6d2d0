// What the two attention kernels over 4-bit pages share (bp_kv4_attention.cu: few rows per request; bp_kv4_prefill.cu: many).
#pragma once

#include "bp_paged.cuh"

namespace bp {
namespace kv4 {

constexpr unsigned FULL = 0xffffffffu;
constexpr float NEG_BIG = -3e38f;  // the maximum of no score, below every score that 32 bits hold but the last few
constexpr float P_UP = 10.f;   // P is stored as f16 times 2^10: it keeps its bits down to 2^-24 of the maximum

// What a kernel's line of requests is.
enum Mode {
  PLAIN,   // requests, their outputs are written
  PARTS,   // prefixes that several requests have in common (their rows are those of all these requests, each sees every key), then requests behind
           // their prefixes: either sees a part of a row's keys only, and what comes out are partial results
  BEHIND,  // requests whose keys are their prefix's and then their own: two rows of pages; their outputs are written
  CHOSEN,  // tokens that see every key of pages chosen for each KV head; their outputs are written
};
// A partial result of a row: [0, D) the values' sum, [D] the score (log2 units) that its weights refer to, 2^(score - [D]), [D + 1] the sum of the weights, then as whole numbers [D + 2] c and
// [D + 3] n << 16 | r. n = 0: that is it. n > 0: n CTAs from c on have a piece of it each, at row r of their place for pieces (piece_at).
// bp_kv4_shared.cu puts them together.
template <int D>
constexpr uint32_t RECORD = D + 4;
// CTA c + k's place for pieces is the k-th of an item's: a CTA has at most two, of the item that ends in it and of the one that goes on behind it.
__host__ __device__ constexpr uint32_t piece_at(uint32_t c, uint32_t k) { return 2 * (c + k) + (k == 0); }

struct AttnArgs {
  Pool pool;
  Rows q, out;
  const int32_t *q_start, *kv_len, *page_table;
  uint32_t* err;
  uint32_t n_req, n_head, group, total_q, max_q, max_kv, table_stride, window;
  uint32_t table_pages;  // of a row of the page table that are looked at: what 31 bits of keys fill at most (rows may lie further apart)
  float scale_log2;
  float mantissa, power;  // their product: 1 <= mantissa < 2, power is one of two or 0
  float mantissa24;       // the mantissa times 2^24
  uint32_t bias;  // 0x64006400: two f16 numbers 1024
  uint32_t bf;    // activations are bfloat16
  uint32_t q_vec; // rows of q are 16-byte aligned
  // prefix g is that of the requests [prefix_start[g], prefix_start[g + 1]) of n_own. PARTS: in the line, requests [0, n_prefix) are the prefixes
  const int32_t *prefix_start, *prefix_len, *prefix_table;
  uint32_t n_prefix, n_own, max_prefix, prefix_stride, prefix_pages;
  float* part;  // [prefix, own][rows of q][n_head] records
  // The launch before this one has waited for what is read here and runs at the same time; it is waited for at the end. (first: this is that launch)
  uint32_t beside, first;
};
// Queries become f16 numbers, each row multiplied by the power of two that brings its largest element into [2^8, 2^9): the most for which 32 of them
// times a mantissa add up within f16, as bp_kv4_attention.cu wants. f16 and bf16 queries keep all their bits down to 2^-18 of the row's largest element,
// smaller ones are off by 2^-29 of it at most: f16 because the keys' values are f16 numbers, which a tensor core multiplies by nothing wider.
struct RowPower {
  uint32_t bits;  // exponent bits of the largest element; of zeros, tiny rows and infinities the nearest that leave 2^(8 - e) and 2^(e - 8) normal numbers
  static __device__ RowPower of(float largest) { return RowPower{min(max(__float_as_uint(largest) & 0x7f800000u, 9u << 23), 254u << 23)}; }
  __device__ float up() const { return __uint_as_float((262u << 23) - bits); }
  __device__ float down() const { return __uint_as_float(bits - (8u << 23)); }
};
// The first key that a query sees to which `keys` of its request are visible without a window (none or fewer: it lies before them all).
// Nothing here may pass 31 bits: windows are shorter than max_kv (a longer one is none).
__device__ __forceinline__ int first_seen(int keys, uint32_t window) { return window && keys > static_cast<int>(window) ? keys - static_cast<int>(window) : 0; }
// What a request has, cut to what there is: its first row of q, its queries, its keys. report: a cut is reported.
struct Lengths {
  int q0, q_len, kv_len;
};
template <int MODE>
__device__ __forceinline__ Lengths lengths_of(const AttnArgs& a, uint32_t r, bool report) {
  int keys, start, stop;
  uint32_t most = a.max_q, most_keys = min(a.max_kv, a.table_pages << a.pool.log_page);
  if (MODE == PARTS && r < a.n_prefix) {
    const int from = a.prefix_start[r], to = a.prefix_start[r + 1], last = static_cast<int>(a.n_own), f = min(max(from, 0), last), t = min(max(to, f), last);
    if (report && (f != from || t != to)) note_range(a.err);
    keys = a.prefix_len[r];
    start = a.q_start[f];
    stop = a.q_start[t];
    most = a.total_q;
    most_keys = min(a.max_prefix, a.prefix_pages << a.pool.log_page);
  } else if constexpr (MODE == CHOSEN) {  // (a negative number of keys: a token of no request)
    keys = a.kv_len[r];
    start = static_cast<int>(r);
    stop = start + (keys >= 0);
  } else {
    if (MODE == PARTS) r -= a.n_prefix;
    keys = a.kv_len[r];
    start = a.q_start[r];
    stop = a.q_start[r + 1];
  }
  const int q0 = max(start, 0);
  const int given_q = max(stop, q0) - q0, given_kv = max(keys, 0);
  const Lengths n{q0, min(min(given_q, static_cast<int>(most)), max(static_cast<int>(a.total_q) - q0, 0)), min(given_kv, static_cast<int>(most_keys))};
  if (report && (given_q > n.q_len || given_kv > n.kv_len || (start < 0 && stop > start))) note_range(a.err);
  return n;
}
// Whether the queries of request r see its keys up to their own (or all of them); its row of pages, for KV head `head`.
template <int MODE>
__device__ __forceinline__ bool is_causal(const AttnArgs& a, uint32_t r) {
  return MODE != PARTS || r >= a.n_prefix;
}
template <int MODE>
__device__ __forceinline__ const int32_t* pages_of(const AttnArgs& a, uint32_t r, uint32_t head) {
  if (MODE == PARTS && r < a.n_prefix) return a.prefix_table + static_cast<size_t>(r) * a.prefix_stride;
  const size_t row = MODE == CHOSEN ? static_cast<size_t>(r) * a.pool.n_kv_head + head : MODE == PARTS ? r - a.n_prefix : r;
  return a.page_table + row * a.table_stride;
}
// The last i of n with begin[i] <= x, or -1, by a warp: 32 places at a time.
__device__ __forceinline__ int last_begun(const int32_t* begin, uint32_t n, int x, uint32_t lane) {
  uint32_t lo = 0, len = n;  // it is lo - 1 or one of [lo, lo + len)
  while (len > 0) {
    const uint32_t step = (len + 31) / 32, at = lo + min(lane * step, len - 1);
    const uint32_t begun = __popc(__ballot_sync(FULL, lane * step < len && begin[at] <= x));
    if (begun == 0) break;
    const uint32_t from = lo + (begun - 1) * step;  // this one has begun, the next one asked for has not
    len = min(step, lo + len - from) - 1;
    lo = from + 1;
  }
  return static_cast<int>(lo) - 1;
}

// A bounded wait for a barrier's phase: false after 2^20 polls or two seconds, or when *stop (may be null) is set.
__device__ __forceinline__ bool wait_phase(uint32_t bar, uint32_t parity, const volatile uint32_t* stop = nullptr) {
  if (mbar_test(bar, parity)) return true;
  unsigned long long t0 = 0, t;
  for (uint32_t i = 0; i < 1u << 20; i++) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 15) != 15) continue;
    if (stop && *stop) return false;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    if (t0 == 0) t0 = t;
    if (t - t0 > 2000000000ull) return false;
  }
  return false;
}

// One more piece of an item has been written (by threads that have met this one at a barrier since); the count before it. What the other
// pieces' writers had written is visible to whoever meets this thread at a barrier afterwards.
__device__ __forceinline__ uint32_t arrive(uint32_t* counter) {
  uint32_t before;
  asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
  return before;
}

// Which of the two blocks whose d's and m's are the halves of d and m have a scale that is no finite number.
__device__ __forceinline__ uint32_t no_numbers(uint32_t d, uint32_t m) {
  constexpr uint32_t LO = 0x7c00u, HI = 0x7c000000u;
  return ((d & LO) == LO || (m & LO) == LO ? 1u : 0u) | ((d & HI) == HI || (m & HI) == HI ? 2u : 0u);
}
// Four dims of an output row.
__device__ __forceinline__ void store4(bool bf, uint16_t* p, float a, float b, float c, float d) {
  const uint32_t x = bf ? pack2<true>(a, b) : pack2<false>(a, b), y = bf ? pack2<true>(c, d) : pack2<false>(c, d);
  if ((reinterpret_cast<uintptr_t>(p) & 7) == 0) {
    *reinterpret_cast<uint2*>(p) = make_uint2(x, y);
  } else {
    p[0] = static_cast<uint16_t>(x);
    p[1] = static_cast<uint16_t>(x >> 16);
    p[2] = static_cast<uint16_t>(y);
    p[3] = static_cast<uint16_t>(y >> 16);
  }
}
__device__ __forceinline__ uint16_t* out_row(const AttnArgs& a, int q0, uint32_t head, uint32_t row) {
  return a.out.data + static_cast<int64_t>(q0 + row / a.group) * a.out.tok + static_cast<int64_t>(head * a.group + row % a.group) * a.out.head;
}
// The same row's record, of the prefix or the own keys.
template <int D>
__device__ __forceinline__ float* record_of(const AttnArgs& a, bool prefix, int q0, uint32_t head, uint32_t row) {
  const size_t at = static_cast<size_t>(q0 + row / a.group) * a.n_head + head * a.group + row % a.group;
  return a.part + ((prefix ? 0 : static_cast<size_t>(a.total_q) * a.n_head) + at) * RECORD<D>;
}
template <int D>
__device__ __forceinline__ void end_record(float* record, float m, float l, uint32_t c = 0, uint32_t n = 0, uint32_t r = 0) {
  *reinterpret_cast<float4*>(record + D) = make_float4(m, l, __uint_as_float(c), __uint_as_float(n << 16 | r));
}

// One row of an item's partial results, joined by a warp: a lane has V dims.
template <int D>
struct RowJoin {
  static constexpr int V = D / 32;
  float m = NEG_BIG, l = 0.f, o[V] = {};
  // The pieces of the lanes in `mask`, in their order: `at` is the row in the lane's piece. N of them are on their way together, the first before
  // anything is known of their weights.
  template <int N>
  __device__ __forceinline__ void add(uint32_t mask, const float* at, uint32_t lane) {
    const float2 ml = mask >> lane & 1 ? *reinterpret_cast<const float2*>(at + D) : make_float2(NEG_BIG, 0.f);
    float e[N][V];
    int of[N];
    auto ask = [&]() {
#pragma unroll
      for (int q = 0; q < N; q++) {
        of[q] = mask ? __ffs(mask) - 1 : -1;
        const float* v = reinterpret_cast<const float*>(__shfl_sync(FULL, reinterpret_cast<unsigned long long>(at), of[q] & 31)) + V * lane;
        if (mask == 0) {
#pragma unroll
          for (int k = 0; k < V; k++) e[q][k] = 0.f;
        } else if constexpr (V == 4) {
          const float4 f = *reinterpret_cast<const float4*>(v);
          e[q][0] = f.x, e[q][1] = f.y, e[q][2] = f.z, e[q][3] = f.w;
        } else {
          const float2 f = *reinterpret_cast<const float2*>(v);
          e[q][0] = f.x, e[q][1] = f.y;
        }
        mask &= mask - 1;
      }
    };
    ask();
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
    while (true) {
#pragma unroll
      for (int q = 0; q < N; q++) {
        const float w = __shfl_sync(FULL, weight, of[q] & 31);
        if (of[q] < 0) continue;
#pragma unroll
        for (int k = 0; k < V; k++) o[k] = fmaf(e[q][k], w, o[k]);
      }
      if (mask == 0) break;
      ask();
    }
  }
  // A partial result again, or the output's dims from `out` on.
  __device__ __forceinline__ void put(float* to, uint32_t lane) const {
    if constexpr (V == 4) *reinterpret_cast<float4*>(to + V * lane) = make_float4(o[0], o[1], o[2], o[3]);
    else *reinterpret_cast<float2*>(to + V * lane) = make_float2(o[0], o[1]);
    if (lane == 0) *reinterpret_cast<float2*>(to + D) = make_float2(m, l);
  }
  __device__ __forceinline__ void put(bool bf, uint16_t* out, uint32_t lane) const {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    out += V * lane;
    if constexpr (V == 4) {
      store4(bf, out, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
    } else {
      const uint32_t h = bf ? pack2<true>(o[0] * inv, o[1] * inv) : pack2<false>(o[0] * inv, o[1] * inv);
      out[0] = static_cast<uint16_t>(h);
      out[1] = static_cast<uint16_t>(h >> 16);
    }
  }
};

}  // namespace kv4
}  // namespace bp

cudaError_t bp_kv4_prefill_init(bp_paged_ctx* c);
// Launches over `ctas` CTAs (0: all); rows: of an item at most. In PARTS pieces go to *slots, `piece` floats each.
cudaError_t bp_launch_kv4_prefill(bp_paged_ctx* c, cudaStream_t s, uint32_t head_dim, int mode, uint64_t rows, uint32_t ctas, const bp::kv4::AttnArgs& a,
                                  const float** slots = nullptr, uint32_t* piece = nullptr);
cudaError_t bp_launch_kv4_few_rows(bp_paged_ctx* c, cudaStream_t s, uint32_t head_dim, int mode, uint64_t rows, uint32_t ctas, const bp::kv4::AttnArgs& a,
                                   const float** slots = nullptr, uint32_t* piece = nullptr);
constexpr uint32_t BP_KV4_ITEM_COST_IN_PARTS = 10;  // what an item of the kernel for many rows costs in PARTS besides its tiles of 64 keys, in such tiles (bp_kv4_prefill.cu)
constexpr uint64_t BP_KV4_FEW_ROWS = 32;  // of a request, that the kernel for few rows takes (bp_kv4_attention.cu has the reason)
// The scale and what belongs to the context and the pool.
uint32_t bp_kv4_table_pages(const bp::Pool& pool, uint32_t stride);
void bp_kv4_attention_args(const bp_paged_ctx* c, bool bf, const bp::Pool& pool, const bp_rows& q, const bp_rows& out, uint32_t n_head, float scale, bp::kv4::AttnArgs* a);
