// What the two attention kernels over 4-bit pages share (bp_kv4_attention.cu: few rows per request; bp_kv4_prefill.cu: many).
#pragma once

#include "bp_paged.cuh"

namespace bp {
namespace kv4 {

constexpr unsigned FULL = 0xffffffffu;
constexpr float NEG_BIG = -3e38f;  // the maximum of no score, below every score that 32 bits hold but the last few
constexpr float P_UP = 10.f;   // P is stored as f16 times 2^10: it keeps its bits down to 2^-24 of the maximum

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
__device__ __forceinline__ Lengths lengths_of(const AttnArgs& a, uint32_t r, bool report) {
  const int start = a.q_start[r], stop = a.q_start[r + 1], keys = a.kv_len[r], q0 = max(start, 0);
  const int given_q = max(stop, q0) - q0, given_kv = max(keys, 0);
  const Lengths n{q0, min(min(given_q, static_cast<int>(a.max_q)), max(static_cast<int>(a.total_q) - q0, 0)),
                  min(given_kv, static_cast<int>(min(a.max_kv, a.table_pages << a.pool.log_page)))};
  if (report && (given_q > n.q_len || given_kv > n.kv_len || (start < 0 && stop > start))) note_range(a.err);
  return n;
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

}  // namespace kv4
}  // namespace bp

cudaError_t bp_kv4_prefill_init(bp_paged_ctx* c);
cudaError_t bp_launch_kv4_prefill(bp_paged_ctx* c, cudaStream_t s, uint32_t head_dim, const bp::kv4::AttnArgs& a);
