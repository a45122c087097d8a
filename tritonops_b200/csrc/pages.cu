// Pages of a paged KV cache on the device: hand-out for the tokens to come, forking / reordering /
// freeing of sequences, compaction.  No counterpart in the reference, whose caches are padded and
// belong to one sequence each (flash_attn_triton/flash_attn_decoding.py:62-69).
//
// State: the page table [slots, width] and a count per page of the rows that hold it.  Which pages
// move where is an ordered enumeration (the i-th free page for the i-th place that needs one), so
// the results are a pure function of the inputs; the steps of one call depend on one another, so
// its bookkeeping is one cluster of CTAs with cluster barriers between the steps (a few hundred
// nanoseconds each, against microseconds for a launch), and the pages themselves are then copied by
// a second kernel that fills the chip and takes the list from memory: the host fetches nothing.
#include <limits.h>

#include <algorithm>

#include "common.cuh"
#include "sm100.cuh"

namespace b200attn {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr int kPlanCtas = 8;             // the largest portable cluster
constexpr long long kOneCta = 8192;      // entries and pages that one CTA goes through alone
constexpr int kMaxSlots = 32768;         // slots of a fork: their keepers stay in shared memory
constexpr int kHeader = 64;              // ints at the front of every workspace
constexpr int kCopies = 0, kCountA = 8, kCountB = 24, kCountC = 40;   // in the header: copies, counts per CTA

__device__ __forceinline__ int cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return (int)r;
}
__device__ __forceinline__ int cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return (int)r;
}
// Barrier of all threads of the cluster; what they wrote before it is visible behind it (read with
// __ldcg where it was written by another CTA of this launch).
__device__ __forceinline__ void cluster_barrier() {
  if (cluster_size() == 1) __syncthreads();
  else asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// Of a value that a warp's lanes share, the sum over the warps before this one; `total` is the CTA's.
// Ends with a barrier.
__device__ __forceinline__ int warps_before(int v, int& total) {
  __shared__ int sums[kPlanWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (lane == 0) sums[warp] = v;
  __syncthreads();
  int s = sums[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += t;
  }
  const int base = __shfl_sync(0xffffffffu, s, (warp + 31) & 31);
  total = __shfl_sync(0xffffffffu, s, 31);
  __syncthreads();
  return warp ? base : 0;
}
__device__ __forceinline__ int block_sum(int v) {
  int total;
  warps_before(__reduce_add_sync(0xffffffffu, v), total);
  return total;
}

// f(i, value(i)) for the i in [lo, hi), kAhead loads of a thread in flight together: a CTA has one
// thousand threads for lists of up to hundreds of thousands, so a load at a time would cost its latency
// hundreds of times over (1024 rows of 537 entries and 327,000 pages: 62 us a hand-out).
constexpr int kAhead = 8;
template <typename Value, typename F>
__device__ __forceinline__ void each(int lo, int hi, int step, Value value, F f) {
  for (long long i0 = lo; i0 < hi; i0 += (long long)kAhead * step) {
    int v[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (i0 + j * step < hi) v[j] = value((int)(i0 + j * step));
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (i0 + j * step < hi) f((int)(i0 + j * step), v[j]);
  }
}

// emit(i, rank) for the i in [lo, hi) with pred(value(i)), ascending, ranks from `rank0`, those below
// `limit`.  A warp takes 256 neighbours at a time.
template <typename Value, typename Pred, typename Emit>
__device__ __forceinline__ void enumerate(int lo, int hi, int rank0, int limit, Value value, Pred pred, Emit emit) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (long long start = lo; start < hi && rank0 < limit; start += kAhead * kPlanThreads) {
    const long long i0 = start + warp * (32 * kAhead) + lane;
    int v[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (i0 + 32 * j < hi) v[j] = value((int)(i0 + 32 * j));
    unsigned has[kAhead];
    int count = 0, total;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      has[j] = __ballot_sync(0xffffffffu, i0 + 32 * j < hi && pred(v[j]));
      count += __popc(has[j]);
    }
    int rank = rank0 + warps_before(count, total);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int mine = rank + __popc(has[j] & ((1u << lane) - 1u));
      if (((has[j] >> lane) & 1u) && mine < limit) emit((int)(i0 + 32 * j), mine);
      rank += __popc(has[j]);
    }
    rank0 += total;
  }
}

// this CTA's part of [0, n)
__device__ __forceinline__ void segment(int n, int& lo, int& hi) {
  const int size = cluster_size(), rank = cluster_rank();
  const int each = (n + size - 1) / size;
  lo = min(n, each * rank);
  hi = min(n, lo + each);
}
// counts that the CTAs left in the header: what the CTAs before this one have, and all of them
__device__ __forceinline__ void counts_of(const int* counts, int& before, int& all) {
  before = all = 0;
  for (int c = 0; c < cluster_size(); ++c) {
    const int v = __ldcg(counts + c);
    if (c < cluster_rank()) before += v;
    all += v;
  }
}

// ---------------------------------------------------------------------------- hand-out
struct GrowParams {
  const int32_t* table;
  const int32_t* lens;
  const int32_t* refs;
  const int32_t* fresh;
  int32_t* table_out;
  int32_t* refs_out;
  int32_t* missing;
  int slots, width, pages, page_size;
  int* header;
  int* need;       // [slots] pages a row lacks
  int* first;      // [slots] the first entry that does
  int* rank0;      // [slots] pages that the rows before lack
  int* free_list;  // [pages]
};

__device__ __forceinline__ long long pages_wanted(const GrowParams& p, int b) {
  const long long tokens = (long long)max(p.lens[b], 0) + max(p.fresh[b], 0);
  return (tokens + p.page_size - 1) / p.page_size;
}

__global__ void __launch_bounds__(kPlanThreads, 1) grow_kernel(const GrowParams p) {
  sm100::launch_dependents();
  sm100::grid_dependency_wait();
  const int tid = cluster_rank() * kPlanThreads + threadIdx.x, threads = cluster_size() * kPlanThreads;
  const int lane = threadIdx.x & 31, warp = tid >> 5, warps = threads >> 5;
  int lo, hi;
  segment(p.pages, lo, hi);
  int free_here = 0;
  each(lo + threadIdx.x, hi, kPlanThreads, [&](int i) { return p.refs[i]; },
       [&](int i, int r) { p.refs_out[i] = r; free_here += r <= 0; });
  for (int b = warp; b < p.slots; b += warps) {
    const long long row = (long long)b * p.width;
    const int want = (int)min((long long)p.width, pages_wanted(p, b));
    int lacks = 0, first = INT_MAX;      // entries without a page, the first of them
    each(lane, p.width, 32, [&](int i) { return p.table[row + i]; }, [&](int i, int e) {
      const bool held = e >= 0 && e < p.pages;
      p.table_out[row + i] = held ? e : -1;
      if (i < want && !held) { ++lacks; first = min(first, i); }
    });
    lacks = __reduce_add_sync(0xffffffffu, lacks);
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) { p.need[b] = lacks; p.first[b] = first; }
  }
  free_here = block_sum(free_here);
  if (threadIdx.x == 0) p.header[kCountA + cluster_rank()] = free_here;
  cluster_barrier();

  int free_before, free_all, asked = 0;
  counts_of(p.header + kCountA, free_before, free_all);
  each(threadIdx.x, p.slots, kPlanThreads, [&](int b) { return __ldcg(p.need + b); }, [&](int, int n) { asked += n; });
  asked = block_sum(asked);
  enumerate(lo, hi, free_before, asked, [&](int i) { return p.refs[i]; }, [](int r) { return r <= 0; },
            [&](int i, int rank) { p.free_list[rank] = i; });
  if (cluster_rank() == cluster_size() - 1) {          // what the rows before each lack
    long long over = 0;
    for (int b = threadIdx.x; b < p.slots; b += kPlanThreads) over += max(pages_wanted(p, b) - p.width, 0LL);
    __shared__ unsigned long long over_all;
    if (threadIdx.x == 0) over_all = 0;
    __syncthreads();
    if (over) atomicAdd(&over_all, (unsigned long long)over);
    for (int start = 0, run = 0; start < p.slots; start += kPlanThreads) {
      const int b = start + threadIdx.x;
      int n = b < p.slots ? __ldcg(p.need + b) : 0, total;
      const int own = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, n, o);
        if (lane >= o) n += t;
      }
      const int before = run + warps_before(__shfl_sync(0xffffffffu, n, 31), total) + n - own;
      if (b < p.slots) p.rank0[b] = before;
      run += total;
    }
    if (threadIdx.x == 0)
      *p.missing = (int)min((long long)INT_MAX, (long long)over_all + max(asked - free_all, 0));
  }
  cluster_barrier();

  // (a lane looks up one of the warp's rows each; most rows lack their last entries, which then need not
  // be read again)
  for (int b0 = warp; b0 < p.slots; b0 += 32 * warps) {
    const long long looked = min((long long)b0 + (long long)lane * warps, (long long)p.slots - 1);
    const int all_need = __ldcg(p.need + looked), all_first = __ldcg(p.first + looked), all_rank = __ldcg(p.rank0 + looked);
    const int all_want = (int)min((long long)p.width, pages_wanted(p, (int)looked));
    for (int k = 0; k < 32 && b0 + (long long)k * warps < p.slots; ++k) {
      const int need = __shfl_sync(0xffffffffu, all_need, k), first = __shfl_sync(0xffffffffu, all_first, k),
                want = __shfl_sync(0xffffffffu, all_want, k);
      int rank = __shfl_sync(0xffffffffu, all_rank, k);
      int32_t* row = p.table_out + (b0 + (long long)k * warps) * p.width;
      for (int i0 = need ? first : want; i0 < want; i0 += 32) {
        const int i = i0 + lane;
        const bool lacks = i < want && (need == want - first || __ldcg(row + i) < 0);
        const unsigned all = __ballot_sync(0xffffffffu, lacks);
        const int mine = rank + __popc(all & ((1u << lane) - 1u));
        if (lacks && mine < free_all) {
          const int page = __ldcg(p.free_list + mine);
          row[i] = page;
          p.refs_out[page] = 1;
        }
        rank += __popc(all);
      }
    }
  }
}

// ---------------------------------------------------------------------------- forking
struct ForkParams {
  const int32_t* table;
  const int32_t* lens;
  const int32_t* refs;
  const int32_t* parents;
  int32_t* table_out;
  int32_t* lens_out;
  int32_t* refs_out;
  int32_t* missing;
  int slots, width, pages, page_size;
  int* header;
  int* want;       // [slots] the page a slot needs a copy of, or -1
  int* free_list;  // [slots]
  int* src;        // [slots] the copies
  int* dst;
};

__global__ void __launch_bounds__(kPlanThreads, 1) fork_kernel(const ForkParams p) {
  extern __shared__ int keeper[];        // [slots] the slot that has the row of this one whole
  sm100::launch_dependents();
  sm100::grid_dependency_wait();
  const int tid = cluster_rank() * kPlanThreads + threadIdx.x, threads = cluster_size() * kPlanThreads;
  const int lane = threadIdx.x & 31, warp = tid >> 5, warps = threads >> 5;
  for (int b = threadIdx.x; b < p.slots; b += kPlanThreads) keeper[b] = INT_MAX;
  __syncthreads();
  for (int b = threadIdx.x; b < p.slots; b += kPlanThreads) {
    const int parent = p.parents[b];
    if (parent >= 0 && parent < p.slots) atomicMin(&keeper[parent], parent == b ? -1 : b);
  }
  each(tid, p.pages, threads, [&](int i) { return p.refs[i]; }, [&](int i, int r) { p.refs_out[i] = r; });
  cluster_barrier();

  for (int b = warp; b < p.slots; b += warps) {
    const int parent = p.parents[b];
    const bool alive = parent >= 0 && parent < p.slots, stays = alive && parent == b;
    const bool keeps = stays || (alive && keeper[parent] == b);
    const int len = alive ? (int)min((long long)max(p.lens[parent], 0), (long long)p.width * p.page_size) : 0;
    const int full = len / p.page_size;
    const bool part = len % p.page_size != 0;
    int copy = -1;
    const int32_t* theirs = p.table + (long long)parent * p.width;
    const long long row = (long long)b * p.width;
    each(lane, p.width, 32, [&](int i) { return alive ? theirs[i] : -1; }, [&](int i, int e) {
      if (e >= p.pages) e = -1;
      const int taken = e >= 0 && (keeps || i < full) ? e : -1;
      if (!stays && taken >= 0) atomicAdd(p.refs_out + taken, 1);
      p.table_out[row + i] = taken;
      if (part && i == full && !keeps) copy = e;
    });
    if (!stays)
      each(lane, p.width, 32, [&](int i) { return p.table[row + i]; },
           [&](int, int old) { if (old >= 0 && old < p.pages) atomicSub(p.refs_out + old, 1); });
    copy = __reduce_max_sync(0xffffffffu, copy);
    if (lane == 0) {
      p.want[b] = copy;
      p.lens_out[b] = len;
    }
  }
  cluster_barrier();

  int lo, hi, asked = 0, free_here = 0;
  segment(p.pages, lo, hi);
  each(threadIdx.x, p.slots, kPlanThreads, [&](int b) { return __ldcg(p.want + b); }, [&](int, int e) { asked += e >= 0; });
  asked = block_sum(asked);
  if (asked > 0)      // (the same in every CTA)
    each(lo + threadIdx.x, hi, kPlanThreads, [&](int i) { return __ldcg(p.refs_out + i); },
         [&](int, int r) { free_here += r <= 0; });
  free_here = block_sum(free_here);
  if (threadIdx.x == 0) p.header[kCountA + cluster_rank()] = free_here;
  cluster_barrier();
  int free_before, free_all;
  counts_of(p.header + kCountA, free_before, free_all);
  enumerate(lo, hi, free_before, asked, [&](int i) { return __ldcg(p.refs_out + i); }, [](int r) { return r <= 0; },
            [&](int i, int rank) { p.free_list[rank] = i; });
  cluster_barrier();

  if (cluster_rank() != 0) return;
  enumerate(0, p.slots, 0, asked, [&](int b) { return __ldcg(p.want + b); }, [](int e) { return e >= 0; }, [&](int b, int rank) {
    const int len = __ldcg(p.lens_out + b), full = len / p.page_size;
    if (rank < free_all) {
      const int page = __ldcg(p.free_list + rank);
      p.table_out[(long long)b * p.width + full] = page;
      p.refs_out[page] = 1;
      p.src[rank] = __ldcg(p.want + b);
      p.dst[rank] = page;
    } else {
      p.lens_out[b] = full * p.page_size;
    }
  });
  if (threadIdx.x == 0) {
    p.header[kCopies] = min(asked, free_all);
    *p.missing = max(asked - free_all, 0);
  }
}

// ---------------------------------------------------------------------------- compaction
struct CompactParams {
  const int32_t* table;
  const int32_t* refs;
  int32_t* table_out;
  int32_t* refs_out;
  int32_t* live;
  int slots, width, pages;
  int* header;
  int* rank_of;    // [pages] the number of a page among the free places below n, or among those that move
  int* src;        // [pages]
  int* dst;
};

__global__ void __launch_bounds__(kPlanThreads, 1) compact_kernel(const CompactParams p) {
  sm100::launch_dependents();
  sm100::grid_dependency_wait();
  const int tid = cluster_rank() * kPlanThreads + threadIdx.x, threads = cluster_size() * kPlanThreads;
  int lo, hi, count = 0, unused, n;
  segment(p.pages, lo, hi);
  each(lo + threadIdx.x, hi, kPlanThreads, [&](int i) { return p.refs[i]; }, [&](int, int r) { count += r > 0; });
  count = block_sum(count);
  if (threadIdx.x == 0) p.header[kCountA + cluster_rank()] = count;
  cluster_barrier();
  counts_of(p.header + kCountA, unused, n);

  int holes = 0, movers = 0;
  each(lo + threadIdx.x, hi, kPlanThreads, [&](int i) { return p.refs[i]; }, [&](int i, int r) {
    holes += i < n && r <= 0;
    movers += i >= n && r > 0;
  });
  holes = block_sum(holes);
  movers = block_sum(movers);
  if (threadIdx.x == 0) {
    p.header[kCountB + cluster_rank()] = holes;
    p.header[kCountC + cluster_rank()] = movers;
  }
  cluster_barrier();
  int holes_before, movers_before, moves;
  counts_of(p.header + kCountB, holes_before, unused);
  counts_of(p.header + kCountC, movers_before, moves);
  const auto refs = [&](int i) { return p.refs[i]; };
  enumerate(lo, min(hi, n), holes_before, INT_MAX, refs, [](int r) { return r <= 0; },
            [&](int i, int rank) { p.dst[rank] = i; p.rank_of[i] = rank; });
  enumerate(max(lo, n), hi, movers_before, INT_MAX, refs, [](int r) { return r > 0; },
            [&](int i, int rank) { p.src[rank] = i; p.rank_of[i] = rank; });
  cluster_barrier();

  each(tid, p.pages, threads, refs, [&](int i, int r) {
    if (i >= n) r = 0;
    else if (r <= 0) r = p.refs[__ldcg(p.src + __ldcg(p.rank_of + i))];
    p.refs_out[i] = r;
  });
  each(tid, p.slots * p.width, threads, [&](int i) {
    const int e = p.table[i];
    return e >= 0 && e < p.pages && p.refs[e] > 0 ? e : -1;
  }, [&](int i, int e) { p.table_out[i] = e < n ? e : __ldcg(p.dst + __ldcg(p.rank_of + e)); });
  if (tid == 0) {
    p.header[kCopies] = moves;
    *p.live = n;
  }
}

// ---------------------------------------------------------------------------- copies
constexpr int kCopyPools = 128;          // pools one launch takes (its parameters stay below 4 KB)
constexpr int kCopyThreads = 256;
constexpr int kCopyUnit = 16384;         // bytes of a page that a CTA moves at a time

struct CopyParams {
  const int* count;
  const int* src;
  const int* dst;
  int n_pools;
  int unit0[kCopyPools + 1];             // units of a page in the pools before this one
  b200attn_page_pool pools[kCopyPools];
};

template <typename V>
__device__ __forceinline__ void copy_unit(const char* src, char* dst, int bytes) {
  constexpr int kPer = 4;
  const V* s = reinterpret_cast<const V*>(src);
  V* d = reinterpret_cast<V*>(dst);
  const int n = bytes / (int)sizeof(V);
  for (int i0 = threadIdx.x; i0 < n; i0 += kPer * kCopyThreads) {
    V v[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (i0 + j * kCopyThreads < n) v[j] = s[i0 + j * kCopyThreads];
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (i0 + j * kCopyThreads < n) d[i0 + j * kCopyThreads] = v[j];
  }
}

// pool[dst[i]] = pool[src[i]] for every pool; no page is both a source and a destination.
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const __grid_constant__ CopyParams p) {
  sm100::launch_dependents();
  sm100::grid_dependency_wait();
  const int each = p.unit0[p.n_pools];
  const long long units = (long long)*p.count * each;
  for (long long u = blockIdx.x; u < units; u += gridDim.x) {
    const int copy = (int)(u / each), unit = (int)(u % each);
    int a = 0, b = p.n_pools;            // the pool with unit0[a] <= unit < unit0[a + 1]
    while (b - a > 1) {
      const int m = (a + b) >> 1;
      if (p.unit0[m] <= unit) a = m; else b = m;
    }
    const b200attn_page_pool& pool = p.pools[a];
    const long long off = (long long)(unit - p.unit0[a]) * kCopyUnit;
    const int bytes = (int)min((long long)kCopyUnit, (long long)pool.page_bytes - off);
    const char* src = (const char*)pool.base + p.src[copy] * (long long)pool.stride_bytes + off;
    char* dst = (char*)pool.base + p.dst[copy] * (long long)pool.stride_bytes + off;
    if ((((uintptr_t)pool.base | pool.stride_bytes | pool.page_bytes) & 15) == 0) copy_unit<uint4>(src, dst, bytes);
    else copy_unit<unsigned>(src, dst, bytes);
  }
}

// ---------------------------------------------------------------------------- host side
bool overlap(const void* a, size_t a_bytes, const void* b, size_t b_bytes) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return x < y + b_bytes && y < x + a_bytes;
}

int check_book(const int32_t* table, const int32_t* refs, const int32_t* table_out, const int32_t* refs_out, int slots,
               int width, int pages) {
  if (!table || !refs || !table_out || !refs_out) return B200ATTN_ERR_NULL;
  if (slots <= 0 || width <= 0 || pages <= 0) return B200ATTN_ERR_SHAPE;
  if ((long long)slots * width > INT_MAX) return B200ATTN_ERR_TOO_LARGE;
  if (((uintptr_t)table | (uintptr_t)refs | (uintptr_t)table_out | (uintptr_t)refs_out) & 3) return B200ATTN_ERR_ALIGN;
  const size_t t = (size_t)slots * width * 4, r = (size_t)pages * 4;
  if (overlap(table, t, table_out, t) || overlap(refs, r, refs_out, r) || overlap(table, t, refs_out, r) ||
      overlap(refs, r, table_out, t) || overlap(table_out, t, refs_out, r))
    return B200ATTN_ERR_SHAPE;
  return B200ATTN_OK;
}

int check_workspace(const void* ws, size_t bytes, size_t need) {
  if (!ws || bytes < need) return B200ATTN_ERR_WORKSPACE;
  return ((uintptr_t)ws & 15) ? B200ATTN_ERR_ALIGN : B200ATTN_OK;
}

int check_pools(const b200attn_page_pool* pools, int n) {
  if (n < 0) return B200ATTN_ERR_SHAPE;
  if (n > 0 && !pools) return B200ATTN_ERR_NULL;
  for (int i = 0; i < n; ++i) {
    if (!pools[i].base) return B200ATTN_ERR_NULL;
    if (pools[i].page_bytes <= 0 || pools[i].stride_bytes < pools[i].page_bytes) return B200ATTN_ERR_SHAPE;
    if (pools[i].page_bytes > (1LL << 30)) return B200ATTN_ERR_TOO_LARGE;
    if (((uintptr_t)pools[i].base | pools[i].page_bytes | pools[i].stride_bytes) & 3) return B200ATTN_ERR_ALIGN;
  }
  return B200ATTN_OK;
}

template <typename P>
int launch_plan(void (*kernel)(P), const P& p, long long entries, size_t smem, cudaStream_t stream) {
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return B200ATTN_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  const int ctas = entries <= kOneCta ? 1 : kPlanCtas;
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kPlanThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, p) == cudaSuccess ? B200ATTN_OK : B200ATTN_ERR_CUDA;
}

// The copies of the list in the workspace, kCopyPools pools a launch; `launches` counts them.
int launch_copies(const b200attn_page_pool* pools, int n_pools, const int* count, const int* src, const int* dst,
                  int sm_count, cudaStream_t stream, int& launches) {
  for (int at = 0; at < n_pools; at += kCopyPools) {
    CopyParams p;
    p.count = count; p.src = src; p.dst = dst;
    p.n_pools = std::min(kCopyPools, n_pools - at);
    p.unit0[0] = 0;
    for (int i = 0; i < p.n_pools; ++i) {
      p.pools[i] = pools[at + i];
      const long long units = p.unit0[i] + (pools[at + i].page_bytes + kCopyUnit - 1) / kCopyUnit;
      if (units > INT_MAX) return B200ATTN_ERR_TOO_LARGE;
      p.unit0[i + 1] = (int)units;
    }
    if (launch_after(copy_pages_kernel, dim3(sm_count * 8), dim3(kCopyThreads), 0, stream, p) != cudaSuccess)
      return B200ATTN_ERR_CUDA;
    ++launches;
  }
  return B200ATTN_OK;
}

}  // namespace

size_t pages_grow_workspace_bytes(const b200attn_pages_grow_args* a) {
  if (!a || a->slots <= 0 || a->num_pages <= 0) return 0;
  return 4 * ((size_t)kHeader + 3 * (size_t)a->slots + a->num_pages);
}

int pages_grow(const b200attn_pages_grow_args* a, cudaStream_t stream) {
  if (!a || !a->seqlens || !a->new_tokens || !a->missing_out) return B200ATTN_ERR_NULL;
  int st = check_book(a->page_table, a->page_refs, a->page_table_out, a->page_refs_out, a->slots, a->max_pages_per_seq,
                      a->num_pages);
  if (st != B200ATTN_OK) return st;
  if (a->page_size <= 0) return B200ATTN_ERR_SHAPE;
  st = check_workspace(a->workspace, a->workspace_bytes, pages_grow_workspace_bytes(a));
  if (st != B200ATTN_OK) return st;
  if ((st = device_info(nullptr)) != B200ATTN_OK) return st;
  GrowParams p;
  p.table = a->page_table; p.lens = a->seqlens; p.refs = a->page_refs; p.fresh = a->new_tokens;
  p.table_out = a->page_table_out; p.refs_out = a->page_refs_out; p.missing = a->missing_out;
  p.slots = a->slots; p.width = a->max_pages_per_seq; p.pages = a->num_pages; p.page_size = a->page_size;
  p.header = (int*)a->workspace;
  p.need = p.header + kHeader;
  p.first = p.need + a->slots;
  p.rank0 = p.first + a->slots;
  p.free_list = p.rank0 + a->slots;
  st = launch_plan(grow_kernel, p, (long long)p.slots * p.width + p.pages, 0, stream);
  if (st != B200ATTN_OK) return st;
  set_launch_count(1);
  return cudaGetLastError() == cudaSuccess ? B200ATTN_OK : B200ATTN_ERR_CUDA;
}

size_t pages_fork_workspace_bytes(const b200attn_pages_fork_args* a) {
  if (!a || a->slots <= 0) return 0;
  return 4 * ((size_t)kHeader + 4 * (size_t)a->slots);
}

int pages_fork(const b200attn_pages_fork_args* a, cudaStream_t stream) {
  if (!a || !a->seqlens || !a->parents || !a->seqlens_out || !a->missing_out) return B200ATTN_ERR_NULL;
  int st = check_book(a->page_table, a->page_refs, a->page_table_out, a->page_refs_out, a->slots, a->max_pages_per_seq,
                      a->num_pages);
  if (st != B200ATTN_OK) return st;
  if (a->page_size <= 0) return B200ATTN_ERR_SHAPE;
  if (a->slots > kMaxSlots || (long long)a->max_pages_per_seq * a->page_size > INT_MAX) return B200ATTN_ERR_TOO_LARGE;
  const size_t n = (size_t)a->slots * 4;
  if (overlap(a->seqlens, n, a->seqlens_out, n) || overlap(a->parents, n, a->seqlens_out, n)) return B200ATTN_ERR_SHAPE;
  st = check_pools(a->pools, a->n_pools);
  if (st != B200ATTN_OK) return st;
  st = check_workspace(a->workspace, a->workspace_bytes, pages_fork_workspace_bytes(a));
  if (st != B200ATTN_OK) return st;
  const DeviceInfo* di = nullptr;
  if ((st = device_info(&di)) != B200ATTN_OK) return st;
  ForkParams p;
  p.table = a->page_table; p.lens = a->seqlens; p.refs = a->page_refs; p.parents = a->parents;
  p.table_out = a->page_table_out; p.lens_out = a->seqlens_out; p.refs_out = a->page_refs_out;
  p.missing = a->missing_out;
  p.slots = a->slots; p.width = a->max_pages_per_seq; p.pages = a->num_pages; p.page_size = a->page_size;
  p.header = (int*)a->workspace;
  p.want = p.header + kHeader;
  p.free_list = p.want + a->slots;
  p.src = p.free_list + a->slots;
  p.dst = p.src + a->slots;
  st = launch_plan(fork_kernel, p, (long long)p.slots * p.width + p.pages, n, stream);
  if (st != B200ATTN_OK) return st;
  int launches = 1;
  st = launch_copies(a->pools, a->n_pools, p.header + kCopies, p.src, p.dst, di->sm_count, stream, launches);
  if (st != B200ATTN_OK) return st;
  set_launch_count(launches);
  return cudaGetLastError() == cudaSuccess ? B200ATTN_OK : B200ATTN_ERR_CUDA;
}

size_t pages_compact_workspace_bytes(const b200attn_pages_compact_args* a) {
  if (!a || a->num_pages <= 0) return 0;
  return 4 * ((size_t)kHeader + 3 * (size_t)a->num_pages);
}

int pages_compact(const b200attn_pages_compact_args* a, cudaStream_t stream) {
  if (!a || !a->live_out) return B200ATTN_ERR_NULL;
  int st = check_book(a->page_table, a->page_refs, a->page_table_out, a->page_refs_out, a->slots, a->max_pages_per_seq,
                      a->num_pages);
  if (st != B200ATTN_OK) return st;
  st = check_pools(a->pools, a->n_pools);
  if (st != B200ATTN_OK) return st;
  st = check_workspace(a->workspace, a->workspace_bytes, pages_compact_workspace_bytes(a));
  if (st != B200ATTN_OK) return st;
  const DeviceInfo* di = nullptr;
  if ((st = device_info(&di)) != B200ATTN_OK) return st;
  CompactParams p;
  p.table = a->page_table; p.refs = a->page_refs;
  p.table_out = a->page_table_out; p.refs_out = a->page_refs_out; p.live = a->live_out;
  p.slots = a->slots; p.width = a->max_pages_per_seq; p.pages = a->num_pages;
  p.header = (int*)a->workspace;
  p.rank_of = p.header + kHeader;
  p.src = p.rank_of + a->num_pages;
  p.dst = p.src + a->num_pages;
  st = launch_plan(compact_kernel, p, (long long)p.slots * p.width + p.pages, 0, stream);
  if (st != B200ATTN_OK) return st;
  int launches = 1;
  st = launch_copies(a->pools, a->n_pools, p.header + kCopies, p.src, p.dst, di->sm_count, stream, launches);
  if (st != B200ATTN_OK) return st;
  set_launch_count(launches);
  return cudaGetLastError() == cudaSuccess ? B200ATTN_OK : B200ATTN_ERR_CUDA;
}

}  // namespace b200attn
