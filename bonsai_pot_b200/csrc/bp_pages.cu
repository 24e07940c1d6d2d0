// Page tables on the device and the copying of pages (include/bonsai_pages.h).
//
// The tables' calls are chains of small steps whose time is latency, not bytes: each is one launch where one CTA can see the whole
// result coming (grow, the end of a fork), rows are spread over CTAs where each is for itself (release, a fork's rows, the tables behind a
// compaction). Free pages are found by looking at the reference counts, 32 per warp and load, in the order of the pages, so results do not depend on
// who comes when; integer counts do not depend on the order of their atomics.
#include "bp_kv4_attention.cuh"
#include "bp_paged_host.cuh"

namespace {

using namespace bp;
using namespace bp::paged;

using kv4::FULL;
constexpr uint32_t WORDS = 8;  // words of 32 pages that a warp looks at at a time: as many loads are on their way
constexpr uint32_t MAX_ROWS = 16384, MAX_OUT = 1u << 24;

struct Tables {
  int32_t *table, *kv_len, *refs;
  uint32_t n_rows, row_pages, stride, n_pages, page, log_page;
  uint32_t* err;
  __device__ uint32_t pages_of(uint32_t tokens) const { return (tokens + page - 1) >> log_page; }
  __device__ int32_t* row(uint32_t r) const { return table + static_cast<size_t>(r) * stride; }
};

// The sum of v over the threads before this one, and of all.
template <uint32_t THREADS, typename T>
__device__ __forceinline__ T block_scan(T v, T* sums, T& total) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  T up = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T x = __shfl_up_sync(FULL, up, o);
    if (lane >= o) up += x;
  }
  if (lane == 31) sums[warp] = up;
  __syncthreads();
  T before = 0;
  total = 0;
#pragma unroll
  for (uint32_t w = 0; w < THREADS / 32; w++) {
    if (w == warp) before = total;
    total += sums[w];
  }
  __syncthreads();
  return before + up - v;
}

// The first `want` pages that are free (or the last that are used), as use(rank, page), a thread each; how many there are, `want` at most.
// list: THREADS * WORDS places in shared memory.
template <uint32_t THREADS, bool USED_FROM_TOP, typename Use>
__device__ __forceinline__ uint32_t find_pages(const Tables& t, uint32_t want, uint32_t* list, uint32_t* sums, Use use) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t found = 0;
  for (uint32_t base = 0; base < t.n_pages && found < want; base += THREADS * WORDS) {
    uint32_t mask[WORDS], mine = 0;
    int32_t refs[WORDS];
#pragma unroll
    for (uint32_t k = 0; k < WORDS; k++) {
      const uint32_t at = base + (warp * WORDS + k) * 32 + lane;
      refs[k] = at < t.n_pages ? t.refs[USED_FROM_TOP ? t.n_pages - 1 - at : at] : USED_FROM_TOP ? 0 : 1;
    }
#pragma unroll
    for (uint32_t k = 0; k < WORDS; k++) {
      mask[k] = __ballot_sync(FULL, USED_FROM_TOP ? refs[k] > 0 : refs[k] == 0);
      mine += __popc(mask[k]);
    }
    if (lane == 0) sums[warp] = mine;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (uint32_t w = 0; w < THREADS / 32; w++) {
      if (w == warp) before = all;
      all += sums[w];
    }
#pragma unroll
    for (uint32_t k = 0; k < WORDS; k++) {
      const uint32_t at = base + (warp * WORDS + k) * 32 + lane;
      if (mask[k] >> lane & 1) list[before + __popc(mask[k] & ((1u << lane) - 1))] = USED_FROM_TOP ? t.n_pages - 1 - at : at;
      before += __popc(mask[k]);
    }
    __syncthreads();
    const uint32_t n = min(all, want - found);
    for (uint32_t i = threadIdx.x; i < n; i += THREADS) use(found + i, list[i]);
    found += n;
    __syncthreads();
  }
  return found;
}

// The last i with begin[i] <= x (begin[0] <= x, n entries, ascending).
__device__ __forceinline__ uint32_t last_begun(const uint32_t* begin, uint32_t n, uint32_t x) {
  uint32_t lo = 0, hi = n;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) >> 1;
    if (begin[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// ---- grow ------------------------------------------------------------------------------------------------------------

constexpr uint32_t GROW_THREADS = 1024;

struct GrowArgs {
  Tables t;
  const int32_t* n_new;
  int32_t *q_start, *positions;
  int64_t* slots;
  uint32_t n_out;
  uint32_t later;  // the tokens' positions and slots are written by pages_place_kernel; a row's first one gets the position alone
};

// Whether row r has room for its tokens, which begin at `start` of the output; the pages that it needs.
__device__ __forceinline__ bool row_fits(const GrowArgs& g, uint32_t r, uint64_t start, uint32_t& need) {
  const int32_t kv = g.t.kv_len[r], n = g.n_new[r];
  need = 0;
  if (kv < 0 || n < 0 || start + n > g.n_out) return false;
  const uint64_t after = static_cast<uint64_t>(kv) + n;
  if (after > 0x7fffffffu || g.t.pages_of(static_cast<uint32_t>(after)) > g.t.row_pages) return false;
  need = g.t.pages_of(static_cast<uint32_t>(after)) - g.t.pages_of(kv);
  return true;
}

// One CTA. A thread has `per` rows side by side; their starts and the ranks of their new pages lie in shared memory, where a new page and a token find their row.
__global__ void __launch_bounds__(GROW_THREADS, 1) pages_grow_kernel(const __grid_constant__ GrowArgs g) {
  extern __shared__ uint32_t smem[];
  uint32_t *list = smem, *starts = list + GROW_THREADS * WORDS, *ranks = starts + g.t.n_rows + 1, *refused = ranks + g.t.n_rows + 1;
  __shared__ uint64_t sums64[GROW_THREADS / 32];
  __shared__ uint32_t sums[GROW_THREADS / 32];
  const Tables& t = g.t;
  const uint32_t per = (t.n_rows + GROW_THREADS - 1) / GROW_THREADS, r0 = min(threadIdx.x * per, t.n_rows), r1 = min(r0 + per, t.n_rows);
  for (uint32_t i = threadIdx.x; i < (t.n_rows + 31) / 32; i += GROW_THREADS) refused[i] = 0;
  pdl_launch_dependents();
  pdl_wait();
  uint64_t n = 0, total, need_all;
  for (uint32_t r = r0; r < r1; r++) n += max(g.n_new[r], 0);
  uint64_t at = block_scan<GROW_THREADS>(n, sums64, total);
  uint64_t need = 0;
  for (uint32_t r = r0; r < r1; r++) {
    uint32_t more;
    starts[r] = static_cast<uint32_t>(min(at, static_cast<uint64_t>(0x7fffffffu)));
    if (!row_fits(g, r, at, more)) {
      atomicOr(&refused[r >> 5], 1u << (r & 31));
      note_range(t.err);
    }
    need += more;
    at += max(g.n_new[r], 0);
  }
  uint64_t rank = block_scan<GROW_THREADS>(need, sums64, need_all);
  for (uint32_t r = r0; r < r1; r++) {
    uint32_t more;
    ranks[r] = static_cast<uint32_t>(min(rank, static_cast<uint64_t>(0xffffffffu)));
    (void)row_fits(g, r, starts[r], more);
    rank += more;
    g.q_start[r] = static_cast<int32_t>(starts[r]);
  }
  if (threadIdx.x == 0) g.q_start[t.n_rows] = static_cast<int32_t>(min(total, static_cast<uint64_t>(0x7fffffffu)));
  __syncthreads();
  const uint32_t want = static_cast<uint32_t>(min(need_all, static_cast<uint64_t>(t.n_pages)));
  const uint32_t found = find_pages<GROW_THREADS, false>(t, want, list, sums, [&](uint32_t k, uint32_t page) {
    const uint32_t r = last_begun(ranks, t.n_rows, k);
    t.row(r)[t.pages_of(t.kv_len[r]) + k - ranks[r]] = static_cast<int32_t>(page);
    t.refs[page] = 1;
  });
  if (found < need_all) {  // some rows do not get all their pages: they get none
    __syncthreads();
    for (uint32_t r = r0; r < r1; r++) {
      uint32_t more;
      if (!row_fits(g, r, starts[r], more) || more == 0 || static_cast<uint64_t>(ranks[r]) + more <= found) continue;
      for (uint32_t k = ranks[r]; k < found; k++) t.refs[t.row(r)[t.pages_of(t.kv_len[r]) + k - ranks[r]]] = 0;
      atomicOr(&refused[r >> 5], 1u << (r & 31));
      note_range(t.err);
    }
  }
  __syncthreads();
  if (g.later) {
    for (uint32_t r = r0; r < r1; r++) {
      const bool fits = !(refused[r >> 5] >> (r & 31) & 1);
      if (g.n_new[r] > 0 && starts[r] < g.n_out) g.positions[starts[r]] = fits ? t.kv_len[r] : -1;
      if (fits) t.kv_len[r] += g.n_new[r];
    }
    return;
  }
  for (uint32_t i = threadIdx.x; i < g.n_out; i += GROW_THREADS) {
    int32_t pos = -1;
    int64_t slot = -1;
    if (i < total) {
      const uint32_t r = last_begun(starts, t.n_rows, i);
      if (!(refused[r >> 5] >> (r & 31) & 1)) {
        pos = t.kv_len[r] + static_cast<int32_t>(i - starts[r]);
        slot = (static_cast<int64_t>(t.row(r)[pos >> t.log_page]) << t.log_page) + (pos & (t.page - 1));
      }
    }
    g.positions[i] = pos;
    g.slots[i] = slot;
  }
  __syncthreads();
  for (uint32_t r = r0; r < r1; r++)
    if (!(refused[r >> 5] >> (r & 31) & 1)) t.kv_len[r] += g.n_new[r];
}

// A thread per token. (The row of a warp's first token and of its last one are looked for by the warp.)
constexpr uint32_t PLACE_THREADS = 256;
__global__ void __launch_bounds__(PLACE_THREADS) pages_place_kernel(const __grid_constant__ GrowArgs g) {
  const Tables& t = g.t;
  const uint32_t lane = threadIdx.x & 31, i = blockIdx.x * PLACE_THREADS + threadIdx.x, i0 = i - lane;
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t total = g.q_start[t.n_rows], last = min(i0 + 31, g.n_out - 1);
  int32_t pos = -1;
  int64_t slot = -1;
  if (i0 < total) {  // (the whole warp; q_start[0] is 0)
    uint32_t lo = kv4::last_begun(g.q_start, t.n_rows, static_cast<int>(i0), lane), hi = kv4::last_begun(g.q_start, t.n_rows, static_cast<int>(last), lane) + 1;
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) >> 1;
      if (static_cast<uint32_t>(g.q_start[mid]) <= i) lo = mid;
      else hi = mid;
    }
    const uint32_t start = g.q_start[lo];
    const int32_t base = g.positions[start];
    if (i <= last && i < total && base >= 0) {
      pos = base + static_cast<int32_t>(i - start);
      slot = (static_cast<int64_t>(t.row(lo)[pos >> t.log_page]) << t.log_page) + (pos & (t.page - 1));
    }
  }
  if (i >= g.n_out) return;
  g.positions[i] = pos;  // (a row's first one: what it is already)
  g.slots[i] = slot;
}

// ---- release ---------------------------------------------------------------------------------------------------------

// One holder of a page less.
__device__ __forceinline__ void let_go(const Tables& t, int32_t page) {
  if (static_cast<uint32_t>(page) >= t.n_pages) {
    note_range(t.err);
  } else if (atomicSub(&t.refs[page], 1) <= 0) {  // nobody held it
    atomicAdd(&t.refs[page], 1);
    note_range(t.err);
  }
}
// The entries of a row of `tokens` tokens, cut to what a row has.
__device__ __forceinline__ uint32_t entries_of(const Tables& t, uint32_t tokens) {
  const uint32_t n = t.pages_of(tokens);
  if (n > t.row_pages) note_range(t.err);
  return min(n, t.row_pages);
}

constexpr uint32_t ROW_THREADS = 512;

// A CTA per row. (A row that is there twice has been emptied by who came first.)
__global__ void __launch_bounds__(ROW_THREADS) pages_release_kernel(const __grid_constant__ Tables t, const int32_t* __restrict__ rows) {
  __shared__ int32_t tokens_s;
  pdl_launch_dependents();
  pdl_wait();
  const int32_t r = rows[blockIdx.x];
  if (r < 0) return;
  if (static_cast<uint32_t>(r) >= t.n_rows) {
    if (threadIdx.x == 0) note_range(t.err);
    return;
  }
  if (threadIdx.x == 0) tokens_s = atomicExch(&t.kv_len[r], 0);
  __syncthreads();
  const int32_t tokens = tokens_s;
  if (tokens < 0 && threadIdx.x == 0) note_range(t.err);
  const uint32_t n = entries_of(t, max(tokens, 0));
  const int32_t* row = t.row(r);
  for (uint32_t i0 = threadIdx.x; i0 < n; i0 += 4 * ROW_THREADS) {  // four of a thread on their way
    int32_t page[4], refs[4];
#pragma unroll
    for (uint32_t k = 0; k < 4; k++) page[k] = i0 + k * ROW_THREADS < n ? row[i0 + k * ROW_THREADS] : 0;
#pragma unroll
    for (uint32_t k = 0; k < 4; k++) {
      refs[k] = 1;
      if (i0 + k * ROW_THREADS >= n) continue;
      if (static_cast<uint32_t>(page[k]) < t.n_pages) refs[k] = atomicSub(&t.refs[page[k]], 1);
      else note_range(t.err);
    }
#pragma unroll
    for (uint32_t k = 0; k < 4; k++) {
      if (refs[k] > 0) continue;  // (nobody held it)
      atomicAdd(&t.refs[page[k]], 1);
      note_range(t.err);
    }
  }
}

// ---- fork ------------------------------------------------------------------------------------------------------------

// A CTA per pair copies the row's full pages; the CTA that comes last hands out the pages for those that are not full. A child is claimed by -1 - i in its
// length, so a row that is a child twice is one pair's alone.
struct ForkArgs {
  Tables t;
  const int32_t *parents, *children;
  int32_t *src, *dst;
  uint32_t n;
  uint32_t* counter;
};
__device__ __forceinline__ bool is_pair(const ForkArgs& f, uint32_t i, uint32_t& parent, uint32_t& child) {
  const int32_t p = f.parents[i], c = f.children[i];
  parent = p;
  child = c;
  return p >= 0 && c >= 0 && parent < f.t.n_rows && child < f.t.n_rows;
}
__global__ void __launch_bounds__(ROW_THREADS) pages_fork_kernel(const __grid_constant__ ForkArgs f) {
  extern __shared__ uint32_t smem[];
  uint32_t *list = smem, *ranks = smem + ROW_THREADS * WORDS;
  int32_t* lengths = reinterpret_cast<int32_t*>(ranks + f.n);  // tokens of the pairs' parents, -1 where there is no pair that holds its child
  __shared__ uint32_t sums[ROW_THREADS / 32], last_s;
  __shared__ int32_t tokens_s;
  const Tables& t = f.t;
  pdl_launch_dependents();
  pdl_wait();
  {
    const uint32_t i = blockIdx.x;
    uint32_t parent, child;
    const bool pair = is_pair(f, i, parent, child);
    if (threadIdx.x == 0) {
      int32_t tokens = -1;
      if (pair) {
        tokens = *reinterpret_cast<volatile int32_t*>(&t.kv_len[parent]);
        if (parent == child || tokens < 0 || t.pages_of(tokens) > t.row_pages || atomicCAS(&t.kv_len[child], 0, -1 - static_cast<int32_t>(i)) != 0) tokens = -1;
        if (tokens < 0) note_range(t.err);
      } else if (f.parents[i] >= 0 && f.children[i] >= 0) {
        note_range(t.err);
      }
      tokens_s = tokens;
    }
    __syncthreads();
    const int32_t tokens = tokens_s;
    if (tokens > 0) {
      const int32_t* from = t.row(parent);
      int32_t* to = t.row(child);
#pragma unroll 4
      for (uint32_t k = threadIdx.x; k < static_cast<uint32_t>(tokens) >> t.log_page; k += ROW_THREADS) {
        const int32_t page = from[k];
        to[k] = page;
        if (static_cast<uint32_t>(page) < t.n_pages) atomicAdd(&t.refs[page], 1);
        else note_range(t.err);
      }
    }
  }
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last_s = atomicAdd(f.counter, 1) == gridDim.x - 1;
  __syncthreads();
  if (!last_s) return;
  __threadfence();
  if (threadIdx.x == 0) *f.counter = 0;  // for the next launch

  // ---- the last CTA ----
  const uint32_t per = (f.n + ROW_THREADS - 1) / ROW_THREADS, i0 = min(threadIdx.x * per, f.n), i1 = min(i0 + per, f.n);
  uint32_t need = 0, want, parent, child;
  for (uint32_t i = i0; i < i1; i++) {
    int32_t tokens = -1;
    if (is_pair(f, i, parent, child) && *reinterpret_cast<volatile int32_t*>(&t.kv_len[child]) == -1 - static_cast<int32_t>(i))
      tokens = max(*reinterpret_cast<volatile int32_t*>(&t.kv_len[parent]), 0);  // (a parent that is somebody's child, too, was empty)
    lengths[i] = tokens;
    need += tokens > 0 && (tokens & (t.page - 1));
    f.src[i] = f.dst[i] = -1;
  }
  uint32_t rank = block_scan<ROW_THREADS>(need, sums, want);
  for (uint32_t i = i0; i < i1; i++) {
    ranks[i] = rank;
    rank += lengths[i] > 0 && (lengths[i] & (t.page - 1));
  }
  __syncthreads();
  const uint32_t found = find_pages<ROW_THREADS, false>(t, want, list, sums, [&](uint32_t k, uint32_t page) {
    const uint32_t i = last_begun(ranks, f.n, k), at = static_cast<uint32_t>(lengths[i]) >> t.log_page;
    const int32_t from = t.row(f.parents[i])[at];
    t.row(f.children[i])[at] = static_cast<int32_t>(page);
    t.refs[page] = 1;
    if (static_cast<uint32_t>(from) < t.n_pages) {
      f.src[i] = from;
      f.dst[i] = static_cast<int32_t>(page);
    } else {
      note_range(t.err);
    }
  });
  __syncthreads();
  for (uint32_t i = i0; i < i1; i++) {
    int32_t tokens = lengths[i];
    if (tokens < 0) continue;
    if ((tokens & (t.page - 1)) && ranks[i] >= found) {  // no page for it: it stays empty
      for (uint32_t k = 0; k < static_cast<uint32_t>(tokens) >> t.log_page; k++) let_go(t, *reinterpret_cast<volatile int32_t*>(t.row(f.children[i]) + k));
      note_range(t.err);
      tokens = 0;
    }
    t.kv_len[f.children[i]] = tokens;
  }
}

// ---- compact ---------------------------------------------------------------------------------------------------------

struct CompactArgs {
  Tables t;
  int32_t *src, *dst;
  uint32_t most;
  uint32_t* counter;
};
// One CTA: what moves where. The count of a page that moves becomes -1 - (where it goes) for the kernel behind this one.
__global__ void __launch_bounds__(GROW_THREADS, 1) pages_plan_kernel(const __grid_constant__ CompactArgs c) {
  extern __shared__ uint32_t smem[];
  __shared__ uint32_t sums[GROW_THREADS / 32];
  const Tables& t = c.t;
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t low = find_pages<GROW_THREADS, false>(t, c.most, smem, sums, [&](uint32_t i, uint32_t page) { c.dst[i] = static_cast<int32_t>(page); });
  const uint32_t high = find_pages<GROW_THREADS, true>(t, c.most, smem, sums, [&](uint32_t i, uint32_t page) { c.src[i] = static_cast<int32_t>(page); });
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < c.most; i += GROW_THREADS) {
    const int32_t from = i < high ? c.src[i] : -1, to = i < low ? c.dst[i] : -1;
    if (from >= 0 && to >= 0 && from > to) {
      t.refs[to] = t.refs[from];
      t.refs[from] = -1 - to;
    } else {
      c.src[i] = c.dst[i] = -1;
    }
  }
}
// The tables' entries follow; the CTA that comes last makes the pages that have moved free.
__global__ void __launch_bounds__(ROW_THREADS) pages_follow_kernel(const __grid_constant__ CompactArgs c) {
  __shared__ uint32_t last_s;
  const Tables& t = c.t;
  pdl_launch_dependents();
  pdl_wait();
  for (uint32_t r = blockIdx.x; r < t.n_rows; r += gridDim.x) {
    const int32_t tokens = t.kv_len[r];
    if (tokens < 0 && threadIdx.x == 0) note_range(t.err);
    const uint32_t n = entries_of(t, max(tokens, 0));
    for (uint32_t i = threadIdx.x; i < n; i += ROW_THREADS) {
      const int32_t page = t.row(r)[i];
      if (static_cast<uint32_t>(page) >= t.n_pages) {
        note_range(t.err);
        continue;
      }
      const int32_t refs = t.refs[page];
      if (refs < 0) t.row(r)[i] = -1 - refs;
    }
  }
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last_s = atomicAdd(c.counter, 1) == gridDim.x - 1;
  __syncthreads();
  if (!last_s) return;
  __threadfence();
  if (threadIdx.x == 0) *c.counter = 0;
  for (uint32_t i = threadIdx.x; i < c.most; i += ROW_THREADS)
    if (c.src[i] >= 0) t.refs[c.src[i]] = 0;
}

// ---- copy ------------------------------------------------------------------------------------------------------------

constexpr uint32_t COPY_THREADS = 256, COPY_UNROLL = 8, MAX_ARRAYS = 128;

struct CopyArgs {
  uint8_t* data[MAX_ARRAYS];
  uint32_t words[MAX_ARRAYS];  // of a page, 16 or 4 bytes each
  const int32_t *src, *dst;
  uint32_t n, n_arrays, n_pages, pieces;
  uint32_t* err;
};
// A CTA copies one piece of COPY_THREADS * COPY_UNROLL words: x = piece and pair, y = array.
template <typename Word>
__global__ void __launch_bounds__(COPY_THREADS) pages_copy_kernel(const __grid_constant__ CopyArgs a) {
  const uint32_t pair = blockIdx.x / a.pieces, piece = blockIdx.x - pair * a.pieces, words = a.words[blockIdx.y];
  pdl_launch_dependents();
  pdl_wait();
  const int32_t from = a.src[pair], to = a.dst[pair];
  if (from < 0 || to < 0) return;
  if (static_cast<uint32_t>(from) >= a.n_pages || static_cast<uint32_t>(to) >= a.n_pages) {
    if (threadIdx.x == 0) note_range(a.err);
    return;
  }
  const Word* x = reinterpret_cast<const Word*>(a.data[blockIdx.y]) + static_cast<size_t>(from) * words;
  Word* y = reinterpret_cast<Word*>(a.data[blockIdx.y]) + static_cast<size_t>(to) * words;
  const uint32_t w0 = piece * (COPY_THREADS * COPY_UNROLL) + threadIdx.x;
  Word v[COPY_UNROLL];
#pragma unroll
  for (uint32_t k = 0; k < COPY_UNROLL; k++)
    if (w0 + k * COPY_THREADS < words) v[k] = x[w0 + k * COPY_THREADS];
#pragma unroll
  for (uint32_t k = 0; k < COPY_UNROLL; k++)
    if (w0 + k * COPY_THREADS < words) y[w0 + k * COPY_THREADS] = v[k];
}

const char* check_tables(const bp_paged_ctx* c, const bp_page_tables* in, Tables* t) {
  if (in->page_tokens != 16 && in->page_tokens != 32 && in->page_tokens != 64) return "page_tokens must be 16, 32 or 64";
  if (in->n_rows == 0 || in->n_rows > MAX_ROWS) return "page tables have 1 .. 16384 rows";
  if (in->row_pages == 0 || in->row_pages > 0x7fffffffu / in->page_tokens) return "a row of a page table has 1 .. 2^31 / page_tokens pages";
  if (in->n_rows > 1 && in->table_stride < in->row_pages) return "the rows of a page table must not overlap";
  if (in->n_pages == 0 || in->n_pages > 0x7fffffffu) return "n_pages must be 1 .. 2^31 - 1";
  if (!aligned_to(in->table, 4) || !aligned_to(in->kv_len, 4) || !aligned_to(in->refs, 4)) return "page tables must be 4-byte aligned";
  *t = Tables{static_cast<int32_t*>(in->table), static_cast<int32_t*>(in->kv_len), static_cast<int32_t*>(in->refs), in->n_rows, in->row_pages, in->table_stride,
              in->n_pages, in->page_tokens, in->page_tokens == 16 ? 4u : in->page_tokens == 32 ? 5u : 6u, c->err_dev};
  return nullptr;
}

}  // namespace

cudaError_t bp_pages_init(bp_paged_ctx* c) {
  cudaError_t e = cudaFuncSetAttribute(pages_grow_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (GROW_THREADS * WORDS + 2 * (MAX_ROWS + 1) + MAX_ROWS / 32) * 4);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(pages_fork_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (ROW_THREADS * WORDS + 2 * MAX_ROWS) * 4);
  if (e == cudaSuccess) e = cudaMalloc(&c->page_counter, sizeof(uint32_t));
  if (e == cudaSuccess) e = cudaMemset(c->page_counter, 0, sizeof(uint32_t));
  return e;
}

extern "C" {

int bp_pages_grow(bp_paged_ctx* c, void* stream, const bp_page_tables* tables, const void* n_new, void* q_start, void* positions, void* slots, uint32_t n_out) {
  if (int s = enter(c)) return s;
  if (!tables) return fail(c, BP_ERR_NULL, "null pointer argument");
  GrowArgs g = {};
  BP_CHECK(c, check_tables(c, tables, &g.t));
  if (n_out > MAX_OUT) return fail_config(c, "at most 2^24 tokens");
  if (!aligned_to(n_new, 4) || !aligned_to(q_start, 4) || !aligned_to(positions, 4) || !aligned_to(slots, 8))
    return fail_config(c, "n_new, q_start and positions must be 4-byte, slots 8-byte aligned");
  if (!g.t.table || !g.t.kv_len || !g.t.refs || !n_new || !q_start || (n_out != 0 && (!positions || !slots))) return fail(c, BP_ERR_NULL, "null pointer argument");
  g.n_new = static_cast<const int32_t*>(n_new);
  g.q_start = static_cast<int32_t*>(q_start);
  g.positions = static_cast<int32_t*>(positions);
  g.slots = static_cast<int64_t*>(slots);
  g.n_out = n_out;
  OnDevice on(c->device);
  BP_TRY(c, on.err);
  const size_t smem = (GROW_THREADS * WORDS + 2 * (g.t.n_rows + 1) + (g.t.n_rows + 31) / 32) * 4;
  // A second launch costs some 2 us, a thousand tokens in one CTA 0.6.
  g.later = n_out > 4096;
  BP_TRY(c, bp_launch(true, pages_grow_kernel, dim3(1), dim3(GROW_THREADS), smem, static_cast<cudaStream_t>(stream), g));
  if (g.later) BP_TRY(c, bp_launch(true, pages_place_kernel, dim3((n_out + PLACE_THREADS - 1) / PLACE_THREADS), dim3(PLACE_THREADS), 0, static_cast<cudaStream_t>(stream), g));
  return BP_OK;
}

int bp_pages_release(bp_paged_ctx* c, void* stream, const bp_page_tables* tables, const void* rows, uint32_t n) {
  if (int s = enter(c)) return s;
  if (!tables) return fail(c, BP_ERR_NULL, "null pointer argument");
  Tables t;
  BP_CHECK(c, check_tables(c, tables, &t));
  if (!aligned_to(rows, 4)) return fail_config(c, "rows must be 4-byte aligned");
  if (n > 0x7fffffffu) return fail_config(c, "at most 2^31 - 1 rows");
  if (n == 0) return BP_OK;
  if (!t.table || !t.kv_len || !t.refs || !rows) return fail(c, BP_ERR_NULL, "null pointer argument");
  OnDevice on(c->device);
  BP_TRY(c, on.err);
  BP_TRY(c, bp_launch(true, pages_release_kernel, dim3(n), dim3(ROW_THREADS), 0, static_cast<cudaStream_t>(stream), t, static_cast<const int32_t*>(rows)));
  return BP_OK;
}

int bp_pages_fork(bp_paged_ctx* c, void* stream, const bp_page_tables* tables, const void* parents, const void* children, uint32_t n, void* src, void* dst) {
  if (int s = enter(c)) return s;
  if (!tables) return fail(c, BP_ERR_NULL, "null pointer argument");
  ForkArgs f = {};
  BP_CHECK(c, check_tables(c, tables, &f.t));
  if (n > MAX_ROWS) return fail_config(c, "at most 16384 pairs");
  if (!aligned_to(parents, 4) || !aligned_to(children, 4) || !aligned_to(src, 4) || !aligned_to(dst, 4)) return fail_config(c, "parents, children, src and dst must be 4-byte aligned");
  if (n == 0) return BP_OK;
  if (!f.t.table || !f.t.kv_len || !f.t.refs || !parents || !children || !src || !dst) return fail(c, BP_ERR_NULL, "null pointer argument");
  f.parents = static_cast<const int32_t*>(parents);
  f.children = static_cast<const int32_t*>(children);
  f.src = static_cast<int32_t*>(src);
  f.dst = static_cast<int32_t*>(dst);
  f.n = n;
  f.counter = c->page_counter;
  OnDevice on(c->device);
  BP_TRY(c, on.err);
  BP_TRY(c, bp_launch(true, pages_fork_kernel, dim3(n), dim3(ROW_THREADS), (ROW_THREADS * WORDS + 2 * n) * 4, static_cast<cudaStream_t>(stream), f));
  return BP_OK;
}

int bp_pages_compact(bp_paged_ctx* c, void* stream, const bp_page_tables* tables, void* src, void* dst, uint32_t most) {
  if (int s = enter(c)) return s;
  if (!tables) return fail(c, BP_ERR_NULL, "null pointer argument");
  CompactArgs a = {};
  BP_CHECK(c, check_tables(c, tables, &a.t));
  if (!aligned_to(src, 4) || !aligned_to(dst, 4)) return fail_config(c, "src and dst must be 4-byte aligned");
  if (most > 0x7fffffffu) return fail_config(c, "at most 2^31 - 1 pages");
  if (most == 0) return BP_OK;
  if (!a.t.table || !a.t.kv_len || !a.t.refs || !src || !dst) return fail(c, BP_ERR_NULL, "null pointer argument");
  a.src = static_cast<int32_t*>(src);
  a.dst = static_cast<int32_t*>(dst);
  a.most = most;
  a.counter = c->page_counter;
  OnDevice on(c->device);
  BP_TRY(c, on.err);
  BP_TRY(c, bp_launch(true, pages_plan_kernel, dim3(1), dim3(GROW_THREADS), GROW_THREADS * WORDS * 4, static_cast<cudaStream_t>(stream), a));
  const uint32_t ctas = a.t.n_rows < 4u * c->sm_count ? a.t.n_rows : 4u * c->sm_count;
  BP_TRY(c, bp_launch(true, pages_follow_kernel, dim3(ctas), dim3(ROW_THREADS), 0, static_cast<cudaStream_t>(stream), a));
  return BP_OK;
}

int bp_pages_copy(bp_paged_ctx* c, void* stream, const bp_page_array* arrays, uint32_t n_arrays, uint32_t n_pages, const void* src, const void* dst, uint32_t n) {
  if (int s = enter(c)) return s;
  if (n_arrays != 0 && !arrays) return fail(c, BP_ERR_NULL, "null pointer argument");
  if (n_pages == 0 || n_pages > 0x7fffffffu) return fail_config(c, "n_pages must be 1 .. 2^31 - 1");
  if (!aligned_to(src, 4) || !aligned_to(dst, 4)) return fail_config(c, "src and dst must be 4-byte aligned");
  for (uint32_t i = 0; i < n_arrays; i++) {
    if (arrays[i].page_bytes == 0 || arrays[i].page_bytes % 4 || arrays[i].page_bytes > 1u << 30) return fail_config(c, "a page has 4 .. 2^30 bytes, a multiple of 4");
    if (!aligned_to(arrays[i].data, 4)) return fail_config(c, "arrays of pages must be 4-byte aligned");
    if ((arrays[i].page_bytes / (4 * COPY_THREADS * COPY_UNROLL) + 1) * n > 0x7fffffffu) return fail_config(c, "too many bytes to copy in one call");
  }
  if (n == 0 || n_arrays == 0) return BP_OK;
  if (!src || !dst) return fail(c, BP_ERR_NULL, "null pointer argument");
  for (uint32_t i = 0; i < n_arrays; i++)
    if (!arrays[i].data) return fail(c, BP_ERR_NULL, "null pointer argument");
  OnDevice on(c->device);
  BP_TRY(c, on.err);
  CopyArgs a;
  a.src = static_cast<const int32_t*>(src);
  a.dst = static_cast<const int32_t*>(dst);
  a.n_pages = n_pages;
  a.n = n;
  a.err = c->err_dev;
  // those whose pages are 16-byte aligned together, then the others
  for (uint32_t wide = 0; wide < 2; wide++) {
    const uint32_t bytes = wide ? 4 : 16;
    for (uint32_t i = 0; i < n_arrays;) {
      uint32_t most = 0;
      for (a.n_arrays = 0; i < n_arrays && a.n_arrays < MAX_ARRAYS; i++) {
        const bool is_wide = arrays[i].page_bytes % 16 == 0 && aligned_to(arrays[i].data, 16);
        if (is_wide != (bytes == 16)) continue;
        a.data[a.n_arrays] = static_cast<uint8_t*>(arrays[i].data);
        a.words[a.n_arrays] = static_cast<uint32_t>(arrays[i].page_bytes / bytes);
        most = a.words[a.n_arrays] > most ? a.words[a.n_arrays] : most;
        a.n_arrays++;
      }
      if (a.n_arrays == 0) continue;
      a.pieces = (most + COPY_THREADS * COPY_UNROLL - 1) / (COPY_THREADS * COPY_UNROLL);
      const dim3 grid(a.pieces * n, a.n_arrays);
      BP_TRY(c, bytes == 16 ? bp_launch(true, pages_copy_kernel<uint4>, grid, dim3(COPY_THREADS), 0, static_cast<cudaStream_t>(stream), a)
                            : bp_launch(true, pages_copy_kernel<uint32_t>, grid, dim3(COPY_THREADS), 0, static_cast<cudaStream_t>(stream), a));
    }
  }
  return BP_OK;
}

}  // extern "C"
