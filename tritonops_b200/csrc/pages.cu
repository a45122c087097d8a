// Pages of a paged KV cache on the device: hand-out for the tokens to come, forking / reordering /
// freeing of sequences, compaction.  No counterpart in the reference, whose caches are padded and
// belong to one sequence each (flash_attn_triton/flash_attn_decoding.py:62-69).
//
// State: the page table [slots, width] and a count per page of the rows that hold it.  Which pages
// move where is an ordered enumeration (the i-th free page for the i-th place that needs one), so
// the results are a pure function of the inputs.  The host fetches nothing, and the steps of one call
// depend on one another, so there are two forms:
//   * Where a CTA can keep the bookkeeping in shared memory (a fork: pages + 8 slots up to 28,672; a
//     compaction: 14,335 pages; a hand-out: pages + 3 slots up to 12,288, and 16,384 of pages and table
//     entries together, where one CTA does it all), every CTA of the copying grid works it out for itself
//     from the same inputs, writes its share of the new tables and copies its share of the pages: one
//     launch, nothing exchanged.  Each CTA of a fork reads the whole table for that, which rows much wider
//     than what they hold make dear.
//   * Beyond, a fork's or compaction's books are kept by one cluster of CTAs (cluster barriers between the
//     steps: a few hundred nanoseconds, against microseconds for a launch) and a second kernel copies from
//     its list; a hand-out, which copies nothing, spreads the tables over the chip in two launches.
// Measured on B200, replayed from a graph:
//   hand-out    8 rows of 63 entries 4.1 us (one CTA); 1024 rows of 537 entries and 327,000 pages 11.0 us,
//               33.9 us by one cluster: 2 MB of table through eight SMs
//   fork        one sequence into four 7.3 us; 64 into 256, 40 MB copied, 22.4 us: 8 us of launch and books (a
//               chain of look-ups and barriers) and the copies, whose floor is 12.3 us.  256 slots that hold 24 pages
//               each, books alone: rows of 24 entries 12.1 us, 512 68.6, 2048 247, 8192 957.  By a cluster: 1024 slots,
//               rows of 537, 332,538 pages 67.5 us
//   compaction  47 small pages 4.7 us; 0.79 GB moved 275 us, 5.8 TB/s = 0.89 of a copy (both tables included).  By a
//               cluster, the books just named, alone: 93 us
#include <limits.h>

#include <algorithm>
#include <initializer_list>

#include "common.cuh"
#include "sm100.cuh"

namespace b200attn {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanCtas = 8;             // the largest portable cluster
constexpr int kMaxSlots = 32768;         // slots of a fork: their keepers stay in shared memory
constexpr int kHeader = 64;              // ints at the front of a fork's or compaction's workspace
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
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// Of a value that a warp's lanes share, the sum over the warps before this one; `total` is the CTA's.
// Ends with a barrier.
__device__ __forceinline__ int warps_before(int v, int& total) {
  __shared__ int sums[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (lane == 0) sums[warp] = v;
  __syncthreads();
  int s = lane < blockDim.x >> 5 ? sums[lane] : 0;
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

// f(b, i, value(b, i)) for every entry i < width of the rows b < slots, by `warps` warps of which this is
// number `warp`: eight rows at a time, so that no entry's row has to be divided for.
template <typename Value, typename F>
__device__ __forceinline__ void each_entry(int slots, int width, int warp, int warps, Value value, F f) {
  const int lane = threadIdx.x & 31;
  for (long long b0 = (long long)warp * kAhead; b0 < slots; b0 += (long long)warps * kAhead)
    for (int i = lane; i < width; i += 32) {
      int v[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (b0 + j < slots) v[j] = value((int)b0 + j, i);
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (b0 + j < slots) f((int)b0 + j, i, v[j]);
    }
}

// emit(i, rank) for the i in [lo, hi) with pred(value(i)), ascending, ranks from `rank0`, those below
// `limit`; the number of ranks counted, at least `limit` if there are as many.  A warp takes 256 neighbours
// at a time.
template <typename Value, typename Pred, typename Emit>
__device__ __forceinline__ int enumerate(int lo, int hi, int rank0, int limit, Value value, Pred pred, Emit emit) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (long long start = lo; start < hi && rank0 < limit; start += kAhead * blockDim.x) {
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
  return rank0;
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
  int* need;       // [slots] pages a row lacks
  int* first;      // [slots] the first entry that does
  int* free_list;  // [pages]
};

__device__ __forceinline__ long long pages_wanted(const GrowParams& p, int b) {
  const long long tokens = (long long)max(p.lens[b], 0) + max(p.fresh[b], 0);
  return (tokens + p.page_size - 1) / p.page_size;
}

// A warp copies row b, its entries without a page as -1, and finds how many of those the coming tokens
// need, and the first of them.
__device__ __forceinline__ void look_at_row(const GrowParams& p, int b, int& lacks, int& first) {
  const long long row = (long long)b * p.width;
  const int want = (int)min((long long)p.width, pages_wanted(p, b));
  lacks = 0; first = INT_MAX;
  each(threadIdx.x & 31, p.width, 32, [&](int i) { return p.table[row + i]; }, [&](int i, int e) {
    const bool held = e >= 0 && e < p.pages;
    p.table_out[row + i] = held ? e : -1;
    if (i < want && !held) { ++lacks; first = min(first, i); }
  });
  lacks = __reduce_add_sync(0xffffffffu, lacks);
  first = __reduce_min_sync(0xffffffffu, first);
}
// A warp gives row b the pages free_list[rank ..] for its `need` entries that lack one (`rank` below
// `free_all` only).  Most rows lack their last entries, which then need not be read again.
template <typename FreeList>
__device__ __forceinline__ void give(const GrowParams& p, long long b, int need, int first, int want, int rank, int free_all,
                                     FreeList free_list) {
  const int lane = threadIdx.x & 31;
  int32_t* row = p.table_out + b * p.width;
  for (int i0 = need ? first : want; i0 < want; i0 += 32) {
    const int i = i0 + lane;
    const bool lacks = i < want && (need == want - first || __ldcg(row + i) < 0);
    const unsigned all = __ballot_sync(0xffffffffu, lacks);
    const int mine = rank + __popc(all & ((1u << lane) - 1u));
    if (lacks && mine < free_all) {
      const int page = free_list(mine);
      row[i] = page;
      p.refs_out[page] = 1;
    }
    rank += __popc(all);
  }
}
// rank0[b]: what the rows before b lack, by one CTA; `missing` is told.  need(b) may be read by everyone.
template <typename Need>
__device__ __forceinline__ void rank_rows(const GrowParams& p, int* rank0, int asked, int free_all, Need need) {
  const int lane = threadIdx.x & 31;
  __shared__ unsigned long long over;
  if (threadIdx.x == 0) over = 0;
  __syncthreads();
  for (int start = 0, run = 0; start < p.slots; start += blockDim.x) {
    const int b = start + threadIdx.x;
    const int own = b < p.slots ? need(b) : 0;
    if (b < p.slots) {
      const long long past = pages_wanted(p, b) - p.width;
      if (past > 0) atomicAdd(&over, (unsigned long long)past);
    }
    int n = own, total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, n, o);
      if (lane >= o) n += t;
    }
    const int before = run + warps_before(__shfl_sync(0xffffffffu, n, 31), total) + n - own;
    if (b < p.slots) rank0[b] = before;
    run += total;
  }
  __syncthreads();
  if (threadIdx.x == 0) *p.missing = (int)min((long long)INT_MAX, (long long)over + max(asked - free_all, 0));
}

// Large books: two launches of the whole grid.  A CTA looks at its share of the rows and lists the free ones
// of its share of the pages; what the CTAs before it lack and have makes the ranks in the second kernel.
struct GrowShare {
  int free, lacks;           // pages of the CTA's share that are free; pages its rows lack
  unsigned long long past;   // pages that its rows want past the table's width
};
struct GrowGridParams {
  GrowParams book;           // (free_list: share after share, each from its first page's place on)
  GrowShare* shares;         // [kGrowCtas]
  int rows_each, pages_each; // shares
};
// (Two for each SM of the chip; any number is right.  A constant, as the workspace is asked for without a device.)
constexpr int kGrowCtas = 2 * 148, kGrowThreads = 256;

__global__ void __launch_bounds__(kGrowThreads) grow_look_kernel(const GrowGridParams q) {
  const GrowParams& p = q.book;
  __shared__ unsigned long long past;
  sm100::launch_dependents();
  if (threadIdx.x == 0) past = 0;
  sm100::grid_dependency_wait();
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long row0 = (long long)blockIdx.x * q.rows_each, row1 = min((long long)p.slots, row0 + q.rows_each);
  int lacks = 0;
  for (long long b = row0 + warp; b < row1; b += kGrowThreads / 32) {
    int own, first;
    look_at_row(p, (int)b, own, first);
    if (lane == 0) {
      p.need[b] = own; p.first[b] = first;
      const long long over = pages_wanted(p, (int)b) - p.width;
      if (over > 0) atomicAdd(&past, (unsigned long long)over);
    }
    lacks += own;
  }
  const long long lo = min((long long)p.pages, (long long)blockIdx.x * q.pages_each);
  const long long hi = min((long long)p.pages, lo + q.pages_each);
  const int free = enumerate((int)lo, (int)hi, 0, INT_MAX,
      [&](int i) { const int r = p.refs[i]; p.refs_out[i] = r; return r; }, [](int r) { return r <= 0; },
      [&](int i, int rank) { p.free_list[lo + rank] = i; });
  int all;
  warps_before(lacks, all);
  if (threadIdx.x == 0) q.shares[blockIdx.x] = {free, all, past};
}

__global__ void __launch_bounds__(kGrowThreads) grow_give_kernel(const GrowGridParams q) {
  const GrowParams& p = q.book;
  __shared__ int free_before[kGrowCtas + 1], lacks_before[kGrowCtas + 1];
  sm100::launch_dependents();
  sm100::grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long row0 = (long long)blockIdx.x * q.rows_each, row1 = min((long long)p.slots, row0 + q.rows_each);
  if (warp < 2) {            // sums over the shares before each
    int* const to = warp == 0 ? free_before : lacks_before;
    int run = 0;
    for (int c0 = 0; c0 < kGrowCtas; c0 += 32) {
      int n = c0 + lane < kGrowCtas ? (warp == 0 ? q.shares[c0 + lane].free : q.shares[c0 + lane].lacks) : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, n, o);
        if (lane >= o) n += t;
      }
      if (c0 + lane < kGrowCtas) to[c0 + lane + 1] = run + n;
      run += __shfl_sync(0xffffffffu, n, 31);
    }
    if (lane == 0) to[0] = 0;
  }
  __syncthreads();
  const int free_all = free_before[kGrowCtas];
  if (blockIdx.x == 0 && warp == 2) {
    unsigned long long past = 0;
    for (int c = lane; c < kGrowCtas; c += 32) past += q.shares[c].past;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) past += __shfl_xor_sync(0xffffffffu, past, o);
    if (lane == 0)
      *p.missing = (int)min((unsigned long long)INT_MAX, past + max(lacks_before[kGrowCtas] - free_all, 0));
  }
  auto page_at = [&](int rank) {
    int lo = 0, hi = kGrowCtas;                // the share with free_before[lo] <= rank < free_before[hi = lo + 1]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (free_before[mid] <= rank) lo = mid;
      else hi = mid;
    }
    return p.free_list[(long long)lo * q.pages_each + rank - free_before[lo]];
  };
  int rank0 = lacks_before[blockIdx.x];
  for (long long b0 = row0; b0 < row1; b0 += 32) {               // a lane looks up one row each
    const long long b = min(b0 + lane, row1 - 1);
    const int own = b0 + lane < row1 ? p.need[b] : 0, first = p.first[b];
    const int want = (int)min((long long)p.width, pages_wanted(p, (int)b));
    int upto = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += t;
    }
    for (int k = warp; k < 32 && b0 + k < row1; k += kGrowThreads / 32)
      give(p, b0 + k, __shfl_sync(0xffffffffu, own, k), __shfl_sync(0xffffffffu, first, k), __shfl_sync(0xffffffffu, want, k),
           rank0 + __shfl_sync(0xffffffffu, upto - own, k), free_all, page_at);
    rank0 += __shfl_sync(0xffffffffu, upto, 31);
  }
}

// The same by one CTA, with its lists in shared memory: for a small cache what counts is the number of
// trips to memory one after another.
constexpr int kGrowOneThreads = 512;
constexpr long long kGrowOneEntries = 16384, kGrowOneInts = 12288;
__global__ void __launch_bounds__(kGrowOneThreads, 1) grow_one_kernel(const GrowParams p) {
  extern __shared__ int smem[];
  int* const need = smem;
  int* const first = need + p.slots;
  int* const rank0 = first + p.slots;
  int* const free_list = rank0 + p.slots;    // [pages]
  sm100::launch_dependents();
  sm100::grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = kGrowOneThreads / 32;
  int free_all = 0, asked = 0;
  // (the first counts are on their way while the rows are looked at)
  int refs0[kAhead];
#pragma unroll
  for (int j = 0; j < kAhead; ++j)
    if (threadIdx.x + j * kGrowOneThreads < p.pages) refs0[j] = p.refs[threadIdx.x + j * kGrowOneThreads];
  for (int b = warp; b < p.slots; b += warps) {
    int lacks, at;
    look_at_row(p, b, lacks, at);
    if (lane == 0) { need[b] = lacks; first[b] = at; asked += lacks; }
  }
  auto count = [&](int i, int r) { p.refs_out[i] = r; free_all += r <= 0; };
#pragma unroll
  for (int j = 0; j < kAhead; ++j)
    if (threadIdx.x + j * kGrowOneThreads < p.pages) count(threadIdx.x + j * kGrowOneThreads, refs0[j]);
  each(threadIdx.x + kAhead * kGrowOneThreads, p.pages, kGrowOneThreads, [&](int i) { return p.refs[i]; }, count);
  free_all = block_sum(free_all);
  asked = block_sum(asked);
  rank_rows(p, rank0, asked, free_all, [&](int b) { return need[b]; });
  enumerate(0, p.pages, 0, asked, [&](int i) { return p.refs[i]; }, [](int r) { return r <= 0; },
            [&](int i, int rank) { free_list[rank] = i; });
  __syncthreads();
  for (int b = warp; b < p.slots; b += warps)
    give(p, b, need[b], first[b], (int)min((long long)p.width, pages_wanted(p, b)), rank0[b], free_all,
         [&](int i) { return free_list[i]; });
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
constexpr int kCopyThreads = 512;
constexpr int kTeam = 256;               // threads that move a unit, 128 bytes each at a time
constexpr int kCopyUnit = 32768;         // bytes

struct CopyPools {
  int n_pools;
  int unit0[kCopyPools + 1];             // units of a page in the pools before this one
  b200attn_page_pool pools[kCopyPools];
};
struct CopyParams {
  const int* count;
  const int* src;
  const int* dst;
  CopyPools to;
};

template <typename V>
__device__ __forceinline__ void copy_unit(const char* src, char* dst, int bytes) {
  constexpr int kPer = 8;
  const V* s = reinterpret_cast<const V*>(src);
  V* d = reinterpret_cast<V*>(dst);
  const int n = bytes / (int)sizeof(V), tid = threadIdx.x % kTeam;
  for (int i0 = tid; i0 < n; i0 += kPer * kTeam) {
    V v[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (i0 + j * kTeam < n) v[j] = __ldcs(s + i0 + j * kTeam);
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (i0 + j * kTeam < n) __stcs(d + i0 + j * kTeam, v[j]);
  }
}
// This CTA's share of: pool[dst[i]] = pool[src[i]] for i < count and every pool.  No page is both a source
// and a destination.
__device__ __forceinline__ void copy_share(const CopyPools& to, int count, const int* src, const int* dst) {
  const int each = to.unit0[to.n_pools];
  const long long units = (long long)count * each;
  constexpr int kTeams = kCopyThreads / kTeam;
  for (long long u = blockIdx.x * kTeams + threadIdx.x / kTeam; u < units; u += gridDim.x * kTeams) {
    const int copy = (int)(u / each), unit = (int)(u % each);
    int a = 0, b = to.n_pools;           // the pool with unit0[a] <= unit < unit0[a + 1]
    while (b - a > 1) {
      const int m = (a + b) >> 1;
      if (to.unit0[m] <= unit) a = m; else b = m;
    }
    const b200attn_page_pool& pool = to.pools[a];
    const long long off = (long long)(unit - to.unit0[a]) * kCopyUnit;
    const int bytes = (int)min((long long)kCopyUnit, (long long)pool.page_bytes - off);
    const char* from = (const char*)pool.base + src[copy] * (long long)pool.stride_bytes + off;
    char* at = (char*)pool.base + dst[copy] * (long long)pool.stride_bytes + off;
    if ((((uintptr_t)pool.base | pool.stride_bytes | pool.page_bytes) & 15) == 0) copy_unit<uint4>(from, at, bytes);
    else copy_unit<unsigned>(from, at, bytes);
  }
}

__global__ void __launch_bounds__(kCopyThreads, 2) copy_pages_kernel(const __grid_constant__ CopyParams p) {
  sm100::launch_dependents();
  sm100::grid_dependency_wait();
  copy_share(p.to, *p.count, p.src, p.dst);
}

// ---------------------------------------------------------------------------- both in one launch
struct ForkCopyParams {
  ForkParams book;
  int books;                             // this launch writes the tables (the others copy further pools)
  CopyPools to;
};

__global__ void __launch_bounds__(kCopyThreads, 2) fork_copy_kernel(const __grid_constant__ ForkCopyParams q) {
  extern __shared__ int smem[];
  const ForkParams& p = q.book;
  int* const count = smem;               // [pages] rows that hold a page
  int* const keeper = count + p.pages;   // [slots] the slot that has the row of this one whole; then number of the slot's copy
  int* const lens = keeper + p.slots;    // [slots]
  int* const from = lens + p.slots;      // [slots] its parent, kFreed or kStays
  int* const upto = from + p.slots;      // [slots] entries it shares (all: INT_MAX)
  int* const last = upto + p.slots;      // [slots] the entry it needs a copy of, or -1
  int* const want = last + p.slots;      // [slots] the page there, or -1
  int* const src = want + p.slots;       // [slots]
  int* const dst = src + p.slots;
  constexpr int kFreed = -1, kStays = -2;
  sm100::launch_dependents();
  const int tid = threadIdx.x;
  for (int b = tid; b < p.slots; b += kCopyThreads) { keeper[b] = INT_MAX; want[b] = -1; }
  __syncthreads();
  sm100::grid_dependency_wait();
  // (one trip to memory for the first of all three lists)
  int refs0[kAhead];
#pragma unroll
  for (int j = 0; j < kAhead; ++j)
    if (tid + j * kCopyThreads < p.pages) refs0[j] = p.refs[tid + j * kCopyThreads];
  for (int b = tid; b < p.slots; b += kCopyThreads) {
    const int n = p.lens[b], parent = p.parents[b];
    lens[b] = (int)min((long long)max(n, 0), (long long)p.width * p.page_size);
    const bool alive = parent >= 0 && parent < p.slots;
    from[b] = !alive ? kFreed : parent == b ? kStays : parent;
    if (alive) atomicMin(&keeper[parent], parent == b ? -1 : b);
  }
#pragma unroll
  for (int j = 0; j < kAhead; ++j)
    if (tid + j * kCopyThreads < p.pages) count[tid + j * kCopyThreads] = refs0[j];
  each(tid + kAhead * kCopyThreads, p.pages, kCopyThreads, [&](int i) { return p.refs[i]; }, [&](int i, int r) { count[i] = r; });
  __syncthreads();
  auto length = [&](int b) -> int {      // of the sequence that slot b becomes
    const int parent = from[b] == kStays ? b : from[b];
    return parent < 0 ? 0 : lens[parent];
  };
  for (int b = tid; b < p.slots; b += kCopyThreads) {
    const int len = length(b), full = len / p.page_size;
    const bool keeps = from[b] == kStays || (from[b] >= 0 && keeper[from[b]] == b);
    upto[b] = keeps ? INT_MAX : full;
    last[b] = !keeps && len % p.page_size ? full : -1;
  }
  __syncthreads();
  // rows let go and taken, the entries of both asked for together
  const int warp = tid >> 5, warps = kCopyThreads / 32, lane = tid & 31;
  auto inherited = [&](int b, int i) -> int {   // an entry of the row that slot b becomes
    const int parent = from[b];
    return parent == kFreed ? -1 : p.table[(long long)(parent == kStays ? b : parent) * p.width + i];
  };
  constexpr int kRows = kAhead;
  for (int b0 = warp * kRows; b0 < p.slots; b0 += warps * kRows)
    for (int i = lane; i < p.width; i += 32) {
      int gone[kRows], taken[kRows];
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        const bool moves = b0 + j < p.slots && from[b0 + j] != kStays;
        gone[j] = moves ? p.table[(long long)(b0 + j) * p.width + i] : -1;
        taken[j] = moves ? inherited(b0 + j, i) : -1;
      }
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        if (gone[j] >= 0 && gone[j] < p.pages) atomicSub(&count[gone[j]], 1);
        if (taken[j] < 0 || taken[j] >= p.pages) continue;
        if (i < upto[b0 + j]) atomicAdd(&count[taken[j]], 1);
        else if (i == last[b0 + j]) want[b0 + j] = taken[j];
      }
    }
  __syncthreads();
  int* const place = keeper;
  const int asked = enumerate(0, p.slots, 0, INT_MAX, [&](int b) { return want[b]; }, [](int e) { return e >= 0; },
            [&](int b, int rank) { src[rank] = want[b]; place[b] = rank; });
  // (the count of a page handed out is set behind the enumeration, which reads the counts)
  const int given = min(asked, enumerate(0, p.pages, 0, asked, [&](int i) { return count[i]; },
                                         [](int r) { return r <= 0; }, [&](int i, int rank) { dst[rank] = i; }));
  __syncthreads();
  for (int i = tid; i < given; i += kCopyThreads) count[dst[i]] = 1;
  __syncthreads();
  if (q.books) {                         // this CTA's share of the new tables
    const int at0 = blockIdx.x * kCopyThreads + tid, step = gridDim.x * kCopyThreads;
    each_entry(p.slots, p.width, blockIdx.x * warps + warp, gridDim.x * warps, inherited, [&](int b, int i, int e) {
      int taken = e >= 0 && e < p.pages && i < upto[b] ? e : -1;
      if (i == last[b] && want[b] >= 0 && place[b] < given) taken = dst[place[b]];
      p.table_out[(long long)b * p.width + i] = taken;
    });
    for (int b = at0; b < p.slots; b += step) {
      const int len = length(b);
      p.lens_out[b] = want[b] >= 0 && place[b] >= given ? len / p.page_size * p.page_size : len;
    }
    for (int i = at0; i < p.pages; i += step) p.refs_out[i] = count[i];
    if (blockIdx.x == 0 && tid == 0) *p.missing = asked - given;
  }
  copy_share(q.to, given, src, dst);
}

struct CompactCopyParams {
  CompactParams book;
  int books;
  CopyPools to;
};

__global__ void __launch_bounds__(kCopyThreads, 2) compact_copy_kernel(const __grid_constant__ CompactCopyParams q) {
  extern __shared__ int smem[];
  const CompactParams& p = q.book;
  constexpr int kStays = -1, kFree = -2;
  int* const what = smem;                // [pages] kStays, kFree, or the page a moving one goes to, or that a free place gets
  int* const src = what + p.pages;       // [pages / 2 + 1]
  int* const dst = src + p.pages / 2 + 1;
  sm100::launch_dependents();
  sm100::grid_dependency_wait();
  const int tid = threadIdx.x;
  int n = 0;
  each(tid, p.pages, kCopyThreads, [&](int i) { return p.refs[i]; }, [&](int i, int r) {
    what[i] = r > 0 ? kStays : kFree;
    n += r > 0;
  });
  n = block_sum(n);                      // (also the barrier in front of the reads)
  auto state = [&](int i) { return what[i]; };
  const int moves = enumerate(0, n, 0, INT_MAX, state, [](int w) { return w == kFree; }, [&](int i, int rank) { dst[rank] = i; });
  enumerate(n, p.pages, 0, INT_MAX, state, [](int w) { return w == kStays; }, [&](int i, int rank) { src[rank] = i; });
  __syncthreads();
  for (int i = tid; i < moves; i += kCopyThreads) {
    what[src[i]] = dst[i];
    what[dst[i]] = src[i];
  }
  __syncthreads();
  if (q.books) {                         // this CTA's share of the new tables
    const int at = blockIdx.x * kCopyThreads + tid, step = gridDim.x * kCopyThreads;
    for (int i = at; i < p.pages; i += step) p.refs_out[i] = i < n ? p.refs[what[i] == kStays ? i : what[i]] : 0;
    each(at, p.slots * p.width, step, [&](int i) { return p.table[i]; }, [&](int i, int e) {
      int to = -1;
      if (e >= 0 && e < p.pages) {
        if (e < n) to = what[e] == kStays ? e : -1;
        else to = what[e] >= 0 ? what[e] : -1;
      }
      p.table_out[i] = to;
    });
    if (blockIdx.x == 0 && tid == 0) *p.live = n;
  }
  copy_share(q.to, moves, src, dst);
}

// ---------------------------------------------------------------------------- host side
int check_book(const int32_t* table, const int32_t* refs, const int32_t* table_out, const int32_t* refs_out, int slots,
               int width, int pages) {
  if (!table || !refs || !table_out || !refs_out) return B200ATTN_ERR_NULL;
  if (slots <= 0 || width <= 0 || pages <= 0) return B200ATTN_ERR_SHAPE;
  if ((long long)slots * width > INT_MAX) return B200ATTN_ERR_TOO_LARGE;
  return aligned4({table, refs, table_out, refs_out}) ? B200ATTN_OK : B200ATTN_ERR_ALIGN;
}

// A list of a call's.  The kernels read their inputs again after they have written results, so what is written lies
// apart from everything else.
struct Span {
  const void* at;
  size_t bytes;
  bool written;
};
int check_apart(std::initializer_list<Span> spans) {
  for (const Span* a = spans.begin(); a != spans.end(); ++a)
    for (const Span* b = spans.begin(); b != a; ++b) {
      const uintptr_t x = (uintptr_t)a->at, y = (uintptr_t)b->at;
      if ((a->written || b->written) && a->bytes && b->bytes && x < y + b->bytes && y < x + a->bytes) return B200ATTN_ERR_SHAPE;
    }
  return B200ATTN_OK;
}

int check_workspace(const void* ws, size_t bytes, size_t need) {
  if (need == 0) return B200ATTN_OK;
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

// Raises the kernel's limit where `smem` needs it.  48 KB are granted without asking, of which the kernel's own
// __shared__ variables (144 bytes at most in this file) take their part.  The limit is the process's, so it is always
// set to the same number, the most that any call of the kernel asks for: another thread may be about to launch.
template <typename P>
bool allow(void (*kernel)(P), size_t smem, size_t most) {
  return smem <= 47 * 1024 ||
         cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most) == cudaSuccess;
}

template <typename P>
int launch_plan(void (*kernel)(P), const P& p, size_t smem, cudaStream_t stream) {
  if (!allow(kernel, smem, 4 * kMaxSlots)) return B200ATTN_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kPlanCtas);
  cfg.blockDim = dim3(kPlanThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = kPlanCtas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, p) == cudaSuccess ? B200ATTN_OK : B200ATTN_ERR_CUDA;
}

// Pools [at, at + kCopyPools) of the caller's.
int pools_of(const b200attn_page_pool* pools, int n_pools, int at, CopyPools& to) {
  to.n_pools = std::min(kCopyPools, n_pools - at);
  to.unit0[0] = 0;
  for (int i = 0; i < to.n_pools; ++i) {
    to.pools[i] = pools[at + i];
    const long long units = to.unit0[i] + (pools[at + i].page_bytes + kCopyUnit - 1) / kCopyUnit;
    if (units > INT_MAX) return B200ATTN_ERR_TOO_LARGE;
    to.unit0[i + 1] = (int)units;
  }
  return B200ATTN_OK;
}

// The copies of the list in the workspace, kCopyPools pools a launch; `launches` counts them.
int launch_copies(const b200attn_page_pool* pools, int n_pools, const int* count, const int* src, const int* dst,
                  int sm_count, cudaStream_t stream, int& launches) {
  for (int at = 0; at < n_pools; at += kCopyPools) {
    CopyParams p;
    p.count = count; p.src = src; p.dst = dst;
    if (int st = pools_of(pools, n_pools, at, p.to)) return st;
    if (launch_after(copy_pages_kernel, dim3(sm_count * 2), dim3(kCopyThreads), 0, stream, p) != cudaSuccess)
      return B200ATTN_ERR_CUDA;
    ++launches;
  }
  return B200ATTN_OK;
}

// Shared memory with which two CTAs fit an SM.
constexpr size_t kBothSmem = 112 * 1024;

// Books and copies in one kernel, again for every kCopyPools pools (once without any).
template <typename P, typename B>
int launch_both(void (*kernel)(P), const B& book, size_t smem, const b200attn_page_pool* pools, int n_pools, int sm_count,
                cudaStream_t stream, int& launches) {
  if (!allow(kernel, smem, kBothSmem)) return B200ATTN_ERR_CUDA;
  for (int at = 0; at == 0 || at < n_pools; at += kCopyPools) {
    P p;
    p.book = book;
    p.books = at == 0;
    if (int st = pools_of(pools, n_pools, at, p.to)) return st;
    if (launch_after(kernel, dim3(sm_count * 2), dim3(kCopyThreads), smem, stream, p) != cudaSuccess) return B200ATTN_ERR_CUDA;
    ++launches;
  }
  return B200ATTN_OK;
}
size_t fork_smem(long long pages, long long slots) { return 4 * (size_t)(pages + 8 * slots); }
size_t compact_smem(long long pages) { return 4 * (size_t)(pages + 2 * (pages / 2 + 1)); }

// one CTA with its lists in shared memory
bool grow_by_one(const b200attn_pages_grow_args* a) {
  return (long long)a->slots * a->max_pages_per_seq + a->num_pages <= kGrowOneEntries &&
         3LL * a->slots + a->num_pages <= kGrowOneInts;
}

}  // namespace

size_t pages_grow_workspace_bytes(const b200attn_pages_grow_args* a) {
  if (!a || a->slots <= 0 || a->num_pages <= 0 || a->max_pages_per_seq <= 0 || grow_by_one(a)) return 0;
  return kGrowCtas * sizeof(GrowShare) + 4 * (2 * (size_t)a->slots + a->num_pages);
}

int pages_grow(const b200attn_pages_grow_args* a, cudaStream_t stream) {
  if (!a || !a->seqlens || !a->new_tokens || !a->missing_out) return B200ATTN_ERR_NULL;
  int st = check_book(a->page_table, a->page_refs, a->page_table_out, a->page_refs_out, a->slots, a->max_pages_per_seq,
                      a->num_pages);
  if (st != B200ATTN_OK) return st;
  if (a->page_size <= 0) return B200ATTN_ERR_SHAPE;
  if (!aligned4({a->seqlens, a->new_tokens, a->missing_out})) return B200ATTN_ERR_ALIGN;
  const size_t scratch = pages_grow_workspace_bytes(a), n = (size_t)a->slots * 4;
  const size_t table = n * a->max_pages_per_seq, counts = (size_t)a->num_pages * 4;
  st = check_workspace(a->workspace, a->workspace_bytes, scratch);
  if (st != B200ATTN_OK) return st;
  st = check_apart({{a->page_table, table, false}, {a->seqlens, n, false}, {a->page_refs, counts, false},
                    {a->new_tokens, n, false}, {a->page_table_out, table, true}, {a->page_refs_out, counts, true},
                    {a->missing_out, 4, true}, {a->workspace, scratch, true}});
  if (st != B200ATTN_OK) return st;
  if ((st = device_info(nullptr)) != B200ATTN_OK) return st;
  GrowParams p;
  p.table = a->page_table; p.lens = a->seqlens; p.refs = a->page_refs; p.fresh = a->new_tokens;
  p.table_out = a->page_table_out; p.refs_out = a->page_refs_out; p.missing = a->missing_out;
  p.slots = a->slots; p.width = a->max_pages_per_seq; p.pages = a->num_pages; p.page_size = a->page_size;
  if (grow_by_one(a)) {
    const size_t smem = 4 * (3 * (size_t)a->slots + a->num_pages);
    if (!allow(grow_one_kernel, smem, 4 * kGrowOneInts)) return B200ATTN_ERR_CUDA;
    if (launch_after(grow_one_kernel, dim3(1), dim3(kGrowOneThreads), smem, stream, p) != cudaSuccess) return B200ATTN_ERR_CUDA;
    set_launch_count(1);
    return cudaGetLastError() == cudaSuccess ? B200ATTN_OK : B200ATTN_ERR_CUDA;
  }
  GrowGridParams q;
  q.shares = (GrowShare*)a->workspace;
  p.need = (int*)(q.shares + kGrowCtas);
  p.first = p.need + a->slots;
  p.free_list = p.first + a->slots;
  q.book = p;
  q.rows_each = (int)(((long long)a->slots + kGrowCtas - 1) / kGrowCtas);
  q.pages_each = (int)(((long long)a->num_pages + kGrowCtas - 1) / kGrowCtas);
  for (auto kernel : {grow_look_kernel, grow_give_kernel})
    if (launch_after(kernel, dim3(kGrowCtas), dim3(kGrowThreads), 0, stream, q) != cudaSuccess) return B200ATTN_ERR_CUDA;
  set_launch_count(2);
  return cudaGetLastError() == cudaSuccess ? B200ATTN_OK : B200ATTN_ERR_CUDA;
}

size_t pages_fork_workspace_bytes(const b200attn_pages_fork_args* a) {
  if (!a || a->slots <= 0 || a->num_pages <= 0 || fork_smem(a->num_pages, a->slots) <= kBothSmem) return 0;
  return 4 * ((size_t)kHeader + 4 * (size_t)a->slots);
}

int pages_fork(const b200attn_pages_fork_args* a, cudaStream_t stream) {
  if (!a || !a->seqlens || !a->parents || !a->seqlens_out || !a->missing_out) return B200ATTN_ERR_NULL;
  int st = check_book(a->page_table, a->page_refs, a->page_table_out, a->page_refs_out, a->slots, a->max_pages_per_seq,
                      a->num_pages);
  if (st != B200ATTN_OK) return st;
  if (a->page_size <= 0) return B200ATTN_ERR_SHAPE;
  if (a->slots > kMaxSlots || (long long)a->max_pages_per_seq * a->page_size > INT_MAX) return B200ATTN_ERR_TOO_LARGE;
  if (!aligned4({a->seqlens, a->parents, a->seqlens_out, a->missing_out})) return B200ATTN_ERR_ALIGN;
  st = check_pools(a->pools, a->n_pools);
  if (st != B200ATTN_OK) return st;
  const size_t scratch = pages_fork_workspace_bytes(a), n = (size_t)a->slots * 4;
  const size_t table = n * a->max_pages_per_seq, counts = (size_t)a->num_pages * 4;
  st = check_workspace(a->workspace, a->workspace_bytes, scratch);
  if (st != B200ATTN_OK) return st;
  st = check_apart({{a->page_table, table, false}, {a->seqlens, n, false}, {a->page_refs, counts, false},
                    {a->parents, n, false}, {a->page_table_out, table, true}, {a->seqlens_out, n, true},
                    {a->page_refs_out, counts, true}, {a->missing_out, 4, true}, {a->workspace, scratch, true}});
  if (st != B200ATTN_OK) return st;
  const DeviceInfo* di = nullptr;
  if ((st = device_info(&di)) != B200ATTN_OK) return st;
  ForkParams p;
  p.table = a->page_table; p.lens = a->seqlens; p.refs = a->page_refs; p.parents = a->parents;
  p.table_out = a->page_table_out; p.lens_out = a->seqlens_out; p.refs_out = a->page_refs_out;
  p.missing = a->missing_out;
  p.slots = a->slots; p.width = a->max_pages_per_seq; p.pages = a->num_pages; p.page_size = a->page_size;
  int launches = 0;
  const size_t smem = fork_smem(a->num_pages, a->slots);
  if (smem <= kBothSmem) {
    st = launch_both(fork_copy_kernel, p, smem, a->pools, a->n_pools, di->sm_count, stream, launches);
    if (st != B200ATTN_OK) return st;
    set_launch_count(launches);
    return cudaGetLastError() == cudaSuccess ? B200ATTN_OK : B200ATTN_ERR_CUDA;
  }
  p.header = (int*)a->workspace;
  p.want = p.header + kHeader;
  p.free_list = p.want + a->slots;
  p.src = p.free_list + a->slots;
  p.dst = p.src + a->slots;
  st = launch_plan(fork_kernel, p, n, stream);
  if (st != B200ATTN_OK) return st;
  launches = 1;
  st = launch_copies(a->pools, a->n_pools, p.header + kCopies, p.src, p.dst, di->sm_count, stream, launches);
  if (st != B200ATTN_OK) return st;
  set_launch_count(launches);
  return cudaGetLastError() == cudaSuccess ? B200ATTN_OK : B200ATTN_ERR_CUDA;
}

size_t pages_compact_workspace_bytes(const b200attn_pages_compact_args* a) {
  if (!a || a->num_pages <= 0 || compact_smem(a->num_pages) <= kBothSmem) return 0;
  return 4 * ((size_t)kHeader + 3 * (size_t)a->num_pages);
}

int pages_compact(const b200attn_pages_compact_args* a, cudaStream_t stream) {
  if (!a || !a->live_out) return B200ATTN_ERR_NULL;
  int st = check_book(a->page_table, a->page_refs, a->page_table_out, a->page_refs_out, a->slots, a->max_pages_per_seq,
                      a->num_pages);
  if (st != B200ATTN_OK) return st;
  if (!aligned4({a->live_out})) return B200ATTN_ERR_ALIGN;
  st = check_pools(a->pools, a->n_pools);
  if (st != B200ATTN_OK) return st;
  const size_t scratch = pages_compact_workspace_bytes(a), counts = (size_t)a->num_pages * 4;
  const size_t table = (size_t)a->slots * a->max_pages_per_seq * 4;
  st = check_workspace(a->workspace, a->workspace_bytes, scratch);
  if (st != B200ATTN_OK) return st;
  st = check_apart({{a->page_table, table, false}, {a->page_refs, counts, false}, {a->page_table_out, table, true},
                    {a->page_refs_out, counts, true}, {a->live_out, 4, true}, {a->workspace, scratch, true}});
  if (st != B200ATTN_OK) return st;
  const DeviceInfo* di = nullptr;
  if ((st = device_info(&di)) != B200ATTN_OK) return st;
  CompactParams p;
  p.table = a->page_table; p.refs = a->page_refs;
  p.table_out = a->page_table_out; p.refs_out = a->page_refs_out; p.live = a->live_out;
  p.slots = a->slots; p.width = a->max_pages_per_seq; p.pages = a->num_pages;
  int launches = 0;
  const size_t smem = compact_smem(a->num_pages);
  if (smem <= kBothSmem) {
    st = launch_both(compact_copy_kernel, p, smem, a->pools, a->n_pools, di->sm_count, stream, launches);
    if (st != B200ATTN_OK) return st;
    set_launch_count(launches);
    return cudaGetLastError() == cudaSuccess ? B200ATTN_OK : B200ATTN_ERR_CUDA;
  }
  p.header = (int*)a->workspace;
  p.rank_of = p.header + kHeader;
  p.src = p.rank_of + a->num_pages;
  p.dst = p.src + a->num_pages;
  st = launch_plan(compact_kernel, p, 0, stream);
  if (st != B200ATTN_OK) return st;
  launches = 1;
  st = launch_copies(a->pools, a->n_pools, p.header + kCopies, p.src, p.dst, di->sm_count, stream, launches);
  if (st != B200ATTN_OK) return st;
  set_launch_count(launches);
  return cudaGetLastError() == cudaSuccess ? B200ATTN_OK : B200ATTN_ERR_CUDA;
}

}  // namespace b200attn
