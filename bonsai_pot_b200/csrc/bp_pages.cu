// Page tables on the device and the copying of pages (include/bonsai_pages.h).
//
// The tables' calls are chains of small steps whose time is latency, not bytes: each is one launch where one CTA can see the whole
// result coming (grow, the end of a fork), rows are spread over CTAs where each is for itself (release, a fork's rows, the tables behind a
// compaction). Free pages are found by looking at the reference counts, 32 per warp and load, in the order of the pages, so results do not depend on
// who comes when; integer counts do not depend on the order of their atomics.
// Where the result is then spread out over many tokens or rows, the CTA has seven others beside it in a cluster, which wait for it at the cluster's barrier: one
// launch (2.8 us on the host) less.
// us on the device: 3 rows end and 64 grow 9 (a call's issue from Python takes 4 to 6), 16 rows of up to 30000 tokens end and get up to 2047 again in a pool of 17000 pages, all but 30 of which
// they need, 13; 4 forks 7, compaction of 300 pages 7. Copied pages go at the rate of memory: 94 MB 18.4 (what is written stays in L2 at first), 708 MB 212, 6.7 TB/s read and written.
#include "bp_paged_host.cuh"

namespace {

using namespace bp;
using namespace bp::paged;

constexpr unsigned FULL = 0xffffffffu;
constexpr uint32_t WORDS = 8;  // words of 32 pages that a warp looks at at a time: as many loads are on their way
constexpr uint32_t MAX_ROWS = 16384, MAX_OUT = 1u << 24;

struct Tables {
  int32_t *table, *kv_len, *refs;
  uint32_t n_rows, row_pages, stride, n_pages, page, log_page;
  uint32_t* err;
  __device__ uint32_t pages_of(uint32_t tokens) const { return (tokens + page - 1) >> log_page; }
  __device__ int32_t* row(uint32_t r) const { return table + static_cast<size_t>(r) * stride; }
};

// Sums are limited to 2^30, more than any call takes: nothing wraps.
constexpr uint32_t MANY = 1u << 30;
__device__ __forceinline__ uint32_t plus(uint32_t a, uint32_t b) { return min(a + b, MANY); }  // (of two up to MANY)

// The sums of v.x and v.y over the threads before this one, and of all.
template <uint32_t THREADS>
__device__ __forceinline__ uint2 block_scan(uint2 v, uint2* sums, uint2& total) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint2 up = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t x = __shfl_up_sync(FULL, up.x, o), y = __shfl_up_sync(FULL, up.y, o);
    if (lane >= o) up = make_uint2(plus(up.x, x), plus(up.y, y));
  }
  if (lane == 31) sums[warp] = up;
  uint2 before = make_uint2(__shfl_up_sync(FULL, up.x, 1), __shfl_up_sync(FULL, up.y, 1));
  if (lane == 0) before = make_uint2(0, 0);
  __syncthreads();
  total = make_uint2(0, 0);
  uint2 warps = make_uint2(0, 0);
#pragma unroll
  for (uint32_t w = 0; w < THREADS / 32; w++) {
    if (w == warp) warps = total;
    const uint2 s = sums[w];
    total = make_uint2(plus(total.x, s.x), plus(total.y, s.y));
  }
  __syncthreads();
  return make_uint2(plus(warps.x, before.x), plus(warps.y, before.y));
}

// The counts of the pages that a lane looks at next, from `base` on (or from the last page down).
template <bool USED_FROM_TOP>
struct Look {
  int32_t refs[WORDS];
  __device__ __forceinline__ void ask(const Tables& t, uint32_t base) {
#pragma unroll
    for (uint32_t k = 0; k < WORDS; k++) {
      const uint32_t at = base + ((threadIdx.x >> 5) * WORDS + k) * 32 + (threadIdx.x & 31);
      refs[k] = at < t.n_pages ? t.refs[USED_FROM_TOP ? t.n_pages - 1 - at : at] : USED_FROM_TOP ? 0 : 1;
    }
  }
};
// The first `want` pages that are free (or the last that are used), as use(rank, page), a thread each; how many there are, `want` at most.
// look: has asked for the first ones. list: THREADS * WORDS places in shared memory.
template <uint32_t THREADS, bool USED_FROM_TOP, typename Use>
__device__ __forceinline__ uint32_t find_pages(const Tables& t, Look<USED_FROM_TOP>& look, uint32_t want, uint32_t* list, uint32_t* sums, Use use) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t found = 0;
  for (uint32_t base = 0; base < t.n_pages && found < want; base += THREADS * WORDS) {
    uint32_t mask[WORDS], mine = 0;
#pragma unroll
    for (uint32_t k = 0; k < WORDS; k++) {
      mask[k] = __ballot_sync(FULL, USED_FROM_TOP ? look.refs[k] > 0 : look.refs[k] == 0);
      mine += __popc(mask[k]);
    }
    if (base + THREADS * WORDS < t.n_pages) look.ask(t, base + THREADS * WORDS);
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
// Places of new tokens that one CTA fills in; more are spread over a cluster of eight. us on the device, one CTA / eight:
//   places    512       2048      4096      8192      16384      32768        256 rows: 2048      4096      16384
//   16 rows   6.4/7.0   7.0/8.0   7.9/8.1   9.9/8.2   14.1/9.2   22.7/10.4              7.6/8.3   8.9/8.7   18.3/10.3
constexpr uint32_t GROW_ALONE = 4 * GROW_THREADS;

struct GrowArgs {
  Tables t;
  const int32_t* n_new;
  int32_t *q_start, *positions;
  int64_t* slots;
  uint32_t n_out;
};

// Whether row r has room for its tokens; the pages that it needs.
__device__ __forceinline__ bool row_fits(const GrowArgs& g, uint32_t r, uint32_t& need) {
  const int32_t kv = g.t.kv_len[r], n = g.n_new[r];
  need = 0;
  if (kv < 0 || n < 0) return false;
  const uint64_t after = static_cast<uint64_t>(kv) + n;
  if (after > 0x7fffffffu || g.t.pages_of(static_cast<uint32_t>(after)) > g.t.row_pages) return false;
  need = g.t.pages_of(static_cast<uint32_t>(after)) - g.t.pages_of(kv);
  return true;
}
// Its tokens, which begin at `start` of the output, have places there.
__device__ __forceinline__ bool has_places(const GrowArgs& g, uint32_t r, uint32_t start) { return static_cast<uint64_t>(start) + max(g.n_new[r], 0) <= g.n_out; }

__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// What the rows get, by one CTA. A thread has `per` rows side by side; where a row's tokens start and the rank of its first new page lie in shared memory, where a new page
// finds its row. In the end ranks[r] is the row's length before, -1 if it is refused; to the other CTAs its first token's position says so.
__device__ __forceinline__ void grow_rows(const GrowArgs& g, uint32_t* list, uint32_t* starts, uint32_t* ranks, uint2* sums2, uint32_t* sums) {
  const Tables& t = g.t;
  const uint32_t per = (t.n_rows + GROW_THREADS - 1) / GROW_THREADS, r0 = min(threadIdx.x * per, t.n_rows), r1 = min(r0 + per, t.n_rows);
  Look<false> look;
  look.ask(t, 0);
  uint2 sum = make_uint2(0, 0), total;
  uint32_t need;
  for (uint32_t r = r0; r < r1; r++) {
    (void)row_fits(g, r, need);
    sum = make_uint2(plus(sum.x, min(static_cast<uint32_t>(max(g.n_new[r], 0)), MANY)), plus(sum.y, need));
  }
  uint2 at = block_scan<GROW_THREADS>(sum, sums2, total);
  const uint32_t tokens = total.x;
  if (tokens > g.n_out) {  // some rows' tokens have no places: these rows need no pages
    uint32_t start = at.x;
    sum.y = 0;
    for (uint32_t r = r0; r < r1; r++) {
      (void)row_fits(g, r, need);
      if (has_places(g, r, start)) sum.y = plus(sum.y, need);
      start = plus(start, min(static_cast<uint32_t>(max(g.n_new[r], 0)), MANY));
    }
    at.y = block_scan<GROW_THREADS>(sum, sums2, total).y;
  }
  for (uint32_t r = r0; r < r1; r++) {
    starts[r] = at.x;
    ranks[r] = at.y;
    g.q_start[r] = static_cast<int32_t>(at.x);
    (void)row_fits(g, r, need);
    at = make_uint2(plus(at.x, min(static_cast<uint32_t>(max(g.n_new[r], 0)), MANY)), has_places(g, r, starts[r]) ? plus(at.y, need) : at.y);
  }
  if (threadIdx.x == 0) {
    starts[t.n_rows] = tokens;
    g.q_start[t.n_rows] = static_cast<int32_t>(tokens);
  }
  __syncthreads();
  const uint32_t found = find_pages<GROW_THREADS, false>(t, look, total.y, list, sums, [&](uint32_t k, uint32_t page) {
    const uint32_t r = last_begun(ranks, t.n_rows, k);
    t.row(r)[t.pages_of(t.kv_len[r]) + k - ranks[r]] = static_cast<int32_t>(page);
    t.refs[page] = 1;
  });
  __syncthreads();
  for (uint32_t r = r0; r < r1; r++) {
    const int32_t kv = t.kv_len[r];
    bool fits = row_fits(g, r, need) && has_places(g, r, starts[r]);
    if (fits && need > 0 && ranks[r] + need > found) {  // it does not get all its pages: it gets none
      for (uint32_t k = ranks[r]; k < found; k++) t.refs[t.row(r)[t.pages_of(kv) + k - ranks[r]]] = 0;
      fits = false;
    }
    if (!fits) note_range(t.err);
    ranks[r] = fits ? static_cast<uint32_t>(kv) : 0xffffffffu;
    if (gridDim.x > 1 && g.n_new[r] > 0 && starts[r] < g.n_out) g.positions[starts[r]] = fits ? kv : -1;
    if (fits) t.kv_len[r] = kv + g.n_new[r];
  }
}
__global__ void __launch_bounds__(GROW_THREADS, 1) pages_grow_kernel(const __grid_constant__ GrowArgs g) {
  extern __shared__ uint32_t smem[];
  uint32_t *list = smem, *starts = list + GROW_THREADS * WORDS, *bases = starts + g.t.n_rows + 1;
  __shared__ uint2 sums2[GROW_THREADS / 32];
  __shared__ uint32_t sums[GROW_THREADS / 32];
  const Tables& t = g.t;
  pdl_launch_dependents();
  pdl_wait();
  if (blockIdx.x == 0) grow_rows(g, list, starts, bases, sums2, sums);
  if (gridDim.x > 1) cluster_sync();
  if (blockIdx.x != 0) {
    for (uint32_t r = threadIdx.x; r <= t.n_rows; r += GROW_THREADS) {
      const uint32_t start = g.q_start[r];
      starts[r] = start;
      if (r < t.n_rows) bases[r] = start < g.n_out ? g.positions[start] : -1;
    }
  }
  __syncthreads();
  const uint32_t total = starts[t.n_rows];
#pragma unroll 2
  for (uint32_t i = blockIdx.x * GROW_THREADS + threadIdx.x; i < g.n_out; i += gridDim.x * GROW_THREADS) {
    int32_t pos = -1;
    int64_t slot = -1;
    if (i < total) {
      const uint32_t r = last_begun(starts, t.n_rows, i);
      if (bases[r] != 0xffffffffu) {
        pos = static_cast<int32_t>(bases[r] + (i - starts[r]));
        slot = (static_cast<int64_t>(t.row(r)[pos >> t.log_page]) << t.log_page) + (pos & (t.page - 1));
      }
    }
    g.positions[i] = pos;  // (a row's first one: what it is already)
    g.slots[i] = slot;
  }
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

// A CTA per row. A row whose length can be none is left; one that is there twice has been emptied by who came first.
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
  if (threadIdx.x == 0) {
    const int32_t tokens = *reinterpret_cast<volatile int32_t*>(&t.kv_len[r]);
    const bool good = tokens >= 0 && t.pages_of(tokens) <= t.row_pages;
    if (!good) note_range(t.err);
    tokens_s = good && atomicCAS(&t.kv_len[r], tokens, 0) == tokens ? tokens : 0;
  }
  __syncthreads();
  const uint32_t n = t.pages_of(tokens_s);
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
// length, so a row that is a child twice is one pair's alone; whose it is src says until then (a length may have been negative before).
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
  __shared__ uint2 sums2[ROW_THREADS / 32];
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
      tokens_s = f.src[i] = tokens;
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
  Look<false> look;
  look.ask(t, 0);
  uint32_t need = 0;
  uint2 total;
  for (uint32_t i = i0; i < i1; i++) {
    const int32_t tokens = *reinterpret_cast<volatile int32_t*>(&f.src[i]);
    lengths[i] = tokens;
    need += tokens > 0 && (tokens & (t.page - 1));
    f.src[i] = f.dst[i] = -1;
  }
  uint32_t rank = block_scan<ROW_THREADS>(make_uint2(need, 0), sums2, total).x;
  for (uint32_t i = i0; i < i1; i++) {
    ranks[i] = rank;
    rank += lengths[i] > 0 && (lengths[i] & (t.page - 1));
  }
  __syncthreads();
  const uint32_t found = find_pages<ROW_THREADS, false>(t, look, total.x, list, sums, [&](uint32_t k, uint32_t page) {
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
// What moves where, by one CTA. The count of a page that moves becomes -1 - (which move it is) for the tables' entries; src tells it from a count that was negative before.
__device__ __forceinline__ void plan_moves(const CompactArgs& c, uint32_t* smem, uint32_t* sums) {
  const Tables& t = c.t;
  Look<false> first;
  Look<true> last;
  first.ask(t, 0);
  last.ask(t, 0);
  const uint32_t low = find_pages<GROW_THREADS, false>(t, first, c.most, smem, sums, [&](uint32_t i, uint32_t page) { c.dst[i] = static_cast<int32_t>(page); });
  const uint32_t high = find_pages<GROW_THREADS, true>(t, last, c.most, smem, sums, [&](uint32_t i, uint32_t page) { c.src[i] = static_cast<int32_t>(page); });
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < c.most; i += GROW_THREADS) {
    const int32_t from = i < high ? c.src[i] : -1, to = i < low ? c.dst[i] : -1;
    if (from >= 0 && to >= 0 && from > to) {
      t.refs[to] = t.refs[from];
      t.refs[from] = -1 - static_cast<int32_t>(i);
    } else {
      c.src[i] = c.dst[i] = -1;
    }
  }
}
// A row's entries follow, four of a lane on their way.
__device__ __forceinline__ void follow_moves(const CompactArgs& c, uint32_t r, uint32_t lane) {
  const Tables& t = c.t;
  const int32_t tokens = t.kv_len[r];
  if (tokens < 0 && lane == 0) note_range(t.err);
  const uint32_t n = entries_of(t, max(tokens, 0));
  int32_t* row = t.row(r);
  for (uint32_t i0 = lane; i0 < n; i0 += 128) {
    int32_t page[4], refs[4];
#pragma unroll
    for (uint32_t k = 0; k < 4; k++) page[k] = i0 + 32 * k < n ? row[i0 + 32 * k] : 0;
#pragma unroll
    for (uint32_t k = 0; k < 4; k++) refs[k] = static_cast<uint32_t>(page[k]) < t.n_pages ? t.refs[page[k]] : 0;
    int32_t from[4], to[4];
#pragma unroll
    for (uint32_t k = 0; k < 4; k++) {
      const uint32_t move = static_cast<uint32_t>(-1 - refs[k]);  // (of a count that is none: beyond `most`)
      from[k] = move < c.most ? c.src[move] : -1;
      to[k] = move < c.most ? c.dst[move] : -1;
    }
#pragma unroll
    for (uint32_t k = 0; k < 4; k++) {
      if (i0 + 32 * k >= n) continue;
      if (static_cast<uint32_t>(page[k]) >= t.n_pages || (refs[k] < 0 && from[k] != page[k])) note_range(t.err);
      else if (refs[k] < 0) row[i0 + 32 * k] = to[k];
    }
  }
}
__device__ __forceinline__ void free_moved(const CompactArgs& c) {
  for (uint32_t i = threadIdx.x; i < c.most; i += blockDim.x)
    if (c.src[i] >= 0) c.t.refs[c.src[i]] = 0;
}
// All of it by a cluster, a warp per row: tables of up to COMPACT_ENTRIES entries. us on the device for 64 pages, one launch / two (whose issue takes 3 more of the host):
//   rows x pages of a row   16 x 64   64 x 256   64 x 1024   256 x 512   64 x 4096   512 x 512   1024 x 512   4096 x 1024
//                           6.6/7.1   9.1/9.9    14.6/15.1   12.5/12.0   46.2/33.1   18.2/12.3   29.0/12.1    167/20.3
constexpr uint32_t COMPACT_ENTRIES = 1u << 17;
__global__ void __launch_bounds__(GROW_THREADS, 1) pages_compact_kernel(const __grid_constant__ CompactArgs c) {
  extern __shared__ uint32_t smem[];
  __shared__ uint32_t sums[GROW_THREADS / 32];
  pdl_launch_dependents();
  pdl_wait();
  if (blockIdx.x == 0) plan_moves(c, smem, sums);
  cluster_sync();
  for (uint32_t r = blockIdx.x * (GROW_THREADS / 32) + (threadIdx.x >> 5); r < c.t.n_rows; r += gridDim.x * (GROW_THREADS / 32)) follow_moves(c, r, threadIdx.x & 31);
  cluster_sync();
  if (blockIdx.x == 0) free_moved(c);
}
// Larger ones: the plan, then the rows by all SMs; the CTA that comes last makes the pages that have moved free.
__global__ void __launch_bounds__(GROW_THREADS, 1) pages_plan_kernel(const __grid_constant__ CompactArgs c) {
  extern __shared__ uint32_t smem[];
  __shared__ uint32_t sums[GROW_THREADS / 32];
  pdl_launch_dependents();
  pdl_wait();
  plan_moves(c, smem, sums);
}
__global__ void __launch_bounds__(ROW_THREADS) pages_follow_kernel(const __grid_constant__ CompactArgs c) {
  __shared__ uint32_t last_s;
  pdl_launch_dependents();
  pdl_wait();
  for (uint32_t r = blockIdx.x * (ROW_THREADS / 32) + (threadIdx.x >> 5); r < c.t.n_rows; r += gridDim.x * (ROW_THREADS / 32)) follow_moves(c, r, threadIdx.x & 31);
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last_s = atomicAdd(c.counter, 1) == gridDim.x - 1;
  __syncthreads();
  if (!last_s) return;
  __threadfence();
  if (threadIdx.x == 0) *c.counter = 0;
  free_moved(c);
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

// One cluster of `ctas` CTAs of GROW_THREADS threads.
template <typename Args>
cudaError_t launch_cluster(void (*kernel)(Args), uint32_t ctas, uint32_t smem, cudaStream_t s, const Args& args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(GROW_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ctas > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args);
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
  cudaError_t e = cudaFuncSetAttribute(pages_grow_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (GROW_THREADS * WORDS + 2 * (MAX_ROWS + 1)) * 4);
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
  const uint32_t smem = (GROW_THREADS * WORDS + 2 * (g.t.n_rows + 1)) * 4;
  BP_TRY(c, launch_cluster(pages_grow_kernel, n_out > GROW_ALONE ? 8 : 1, smem, static_cast<cudaStream_t>(stream), g));
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
  const uint32_t smem = GROW_THREADS * WORDS * 4;
  if (static_cast<uint64_t>(a.t.n_rows) * a.t.row_pages <= COMPACT_ENTRIES) {
    BP_TRY(c, launch_cluster(pages_compact_kernel, 8, smem, static_cast<cudaStream_t>(stream), a));
    return BP_OK;
  }
  BP_TRY(c, bp_launch(true, pages_plan_kernel, dim3(1), dim3(GROW_THREADS), smem, static_cast<cudaStream_t>(stream), a));
  const uint32_t rows = (a.t.n_rows + ROW_THREADS / 32 - 1) / (ROW_THREADS / 32), ctas = rows < 4u * c->sm_count ? rows : 4u * c->sm_count;
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
