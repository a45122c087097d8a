// New K / V rows quantised into a paged cache of 8-bit numbers with a scale for each block of tokens
// and head, for sm_100a.  The reference's caches are 16-bit and filled by Python copy loops
// (flash_attn_triton/flash_attn_decoding.py:404-425).
//
//   need = the smallest power of two with max|x| <= need * M     (M = 448 for e4m3, 127 for int8)
//   s'   = max(s, need) where the block holds earlier tokens of scale s, else need
//   x   -> round(x / s'),  and the numbers q of the earlier tokens -> round(q * s / s') where s' > s
//
// Powers of two: x / s' and s / s' are exact, so a number is rounded once however it got into the
// cache, e4m3 rows that are taken over to a larger scale keep their bits but for the subnormals,
// and the scale of a block that fills token by token moves at most once per octave (max / M would
// move with every new maximum and round the block's int8 rows again each time).
//
// A task is one (block, head, K or V): the block's 16-row units go to a warp each, 16 bytes per lane
// and row, stay in registers between the maximum and the rounding, and leave as 8-byte pieces.
//
// Bound: two bytes read and one written for each number; behind them the instructions, about five for a
// number (56 % of the issue slots while it runs).  Measured on B200, 8 heads of 128:
//   packed rows   6 prompts of 37 to 5000 rows, fp16 to int8 (98 MB)       23.4 us  4.2 TB/s
//                 16 prompts of 3000 to 5000 rows, bf16 to e4m3 (411 MB)   78.7 us  5.2 TB/s, 0.81 of a copy
//                 128 sequences of 3 to 6 rows                             12.6 us
//     (a CTA for a run of rows, with the blocks that begin there: 27.4, 89.5 and 27.1 us: a partial second
//     wave, and the look-ups once for every block)
//   one row each  256 sequences 3.1 us, 64 sequences 2.4 us, replayed from a graph; where all 256 rows raise
//                 their block's scale, blocks about half full, e4m3: 5.9 us with blocks of 16, 14.3 of 64, 25.8 of 128
//                 (the block's earlier rows are read and written again, by the lanes that hold the new one)
#include <limits.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "sm100.cuh"

namespace b200attn {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kAppendWarps = kAppendThreads / 32;
constexpr int kCtasPerSm = 2;
constexpr int kListed = 128;                   // blocks a CTA looks up at a time
constexpr int kUnitRows = 16;

struct AppendParams {
  const void* rows[2];             // K, V: new rows [tokens, heads, head_dim]
  void* pages[2];
  float* scales[2];
  long long row_st[2], row_sh[2];
  long long page_sp[2], page_st[2], page_sh[2];
  long long scale_sp[2], scale_sb[2], scale_sh[2];
  const int32_t* table;
  const int32_t* lens;
  const int32_t* cu;               // nullptr: token t is sequence t's only new one
  int tokens, batch, heads, head_dim;
  int page_size, block, num_pages, width;
  int warps_per_task;              // one for each 16-row unit of a block
};

// one block that gets new rows
struct AppendBlock {
  int row0;                        // the first of them
  int off, fresh;                  // tokens the block holds already, new ones (none: its page is nowhere)
  int page, index;                 // page of the pool, block of the page
};

// the rows sequence i gets, as far as the table has room, and the blocks they fall into
struct AppendRun {
  int first, count, len, blocks;
  __device__ __forceinline__ AppendRun(const AppendParams& p, int i) : first(0), count(0), len(0), blocks(0) {
    if (i < 0 || i >= p.batch) return;
    first = p.cu[i];
    const int end = min(p.cu[i + 1], p.tokens);
    len = p.lens[i];
    if (first < 0 || first >= end || len < 0) return;
    count = (int)max(0ll, min((long long)(end - first), (long long)p.width * p.page_size - len));
    if (count > 0) blocks = (int)(((long long)(len & (p.block - 1)) + count + p.block - 1) / p.block);
  }
};

// sum of n over the CTA's threads before this one, and over all of them
__device__ __forceinline__ long long sum_before(long long n, long long* sums, long long& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long upto = n;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long other = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += other;
  }
  __syncthreads();
  if (lane == 31) sums[warp] = upto;
  __syncthreads();
  long long before = upto - n;
  all = 0;
#pragma unroll
  for (int i = 0; i < kAppendWarps; ++i) {
    if (i < warp) before += sums[i];
    all += sums[i];
  }
  return before;
}

// max(m, |x|) of two numbers; NaN stays
template <typename T>
__device__ __forceinline__ unsigned max_abs2(unsigned m, unsigned x);
template <>
__device__ __forceinline__ unsigned max_abs2<__half>(unsigned m, unsigned x) {
  asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(m) : "r"(x & 0x7fff7fffu));
  return m;
}
template <>
__device__ __forceinline__ unsigned max_abs2<__nv_bfloat16>(unsigned m, unsigned x) {
  asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(x & 0x7fff7fffu));
  return m;
}

template <typename T>
__device__ __forceinline__ float2 unpack2(unsigned x);
template <>
__device__ __forceinline__ float2 unpack2<__half>(unsigned x) {
  return __half22float2(*reinterpret_cast<const __half2*>(&x));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(unsigned x) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x));
}

// The scale `top` = max|x| (its 15 bits in the rows' type) asks for.
template <typename T, bool kE4M3>
__device__ __forceinline__ float scale_for(unsigned top) {
  const float x = unpack2<T>(top).x;
  const unsigned bits = __float_as_uint(x);
  if (bits == 0) return 0.f;
  const int e = (int)(bits >> 23);
  if (e == 255) return __uint_as_float(0x7fc00000u);
  const bool fits = (bits & 0x7fffffu) <= (kE4M3 ? 0x600000u : 0x7e0000u);   // mantissa of 1.75 (448), 127 / 64
  const int s = e - (kE4M3 ? 8 : 6) + (fits ? 0 : 1);
  return __uint_as_float((unsigned)max(s, 1) << 23);    // (not below 2^-126)
}

// round(x * inv), four numbers of at most the type's largest.  int8: added to 1.5 * 2^23 a number is rounded
// to an integer, ties to even, whose low byte it then ends with.
template <bool kE4M3>
__device__ __forceinline__ unsigned quantise4(float a, float b, float c, float d, float inv) {
  if (kE4M3) {
    unsigned short lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b * inv), "f"(a * inv));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d * inv), "f"(c * inv));
    return (unsigned)lo | ((unsigned)hi << 16);
  }
  auto one = [&](float x) { return __float_as_uint(fmaf(x, inv, 12582912.f)); };
  return __byte_perm(__byte_perm(one(a), one(b), 0x0040), __byte_perm(one(c), one(d), 0x0040), 0x5410);
}
template <bool kE4M3>
__device__ __forceinline__ float4 unquantise4(unsigned q) {
  if (kE4M3) {
    unsigned lo, hi;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"((unsigned short)(q & 0xffffu)));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"((unsigned short)(q >> 16)));
    const float2 a = unpack2<__half>(lo), b = unpack2<__half>(hi);
    return make_float4(a.x, a.y, b.x, b.y);
  }
  return make_float4((float)(signed char)q, (float)(signed char)(q >> 8), (float)(signed char)(q >> 16),
                     (float)(signed char)(q >> 24));
}

// What a block's numbers are divided by and turned into, given the maximum over its new rows and the
// scale `before` of its earlier ones (0: none).
template <typename T, bool kE4M3>
struct Scaling {
  float before, after, inv;
  bool pow2;
  __device__ __forceinline__ Scaling(unsigned top, float before_) : before(before_) {
    const float need = scale_for<T, kE4M3>(top);
    after = (need != need || before != before) ? __uint_as_float(0x7fc00000u) : fmaxf(need, before);
    // the reciprocal of a power of two is exact; scales that came from elsewhere are divided by
    const unsigned bits = __float_as_uint(after);
    pow2 = (bits & 0x7fffffu) == 0 && bits >= 0x00800000u && bits < 0x7f000000u;
    inv = pow2 ? __uint_as_float(0x7f000000u - bits) : 0.f;
  }
  // eight numbers of a new row; kPow2: as `pow2` says
  template <bool kPow2>
  __device__ __forceinline__ uint2 eight(const uint4& x) const {
    const unsigned w[4] = {x.x, x.y, x.z, x.w};
    unsigned q[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float2 a = unpack2<T>(w[2 * i]), b = unpack2<T>(w[2 * i + 1]);
      if (!kPow2) {
        auto over = [&](float v) { return after > 0.f ? __fdiv_rn(v, after) : 0.f; };   // (numbers of a NaN block are 0)
        a = make_float2(over(a.x), over(a.y));
        b = make_float2(over(b.x), over(b.y));
      }
      q[i] = quantise4<kE4M3>(a.x, a.y, b.x, b.y, kPow2 ? inv : 1.f);
    }
    return make_uint2(q[0], q[1]);
  }
  // eight numbers of an earlier row to the new scale
  __device__ __forceinline__ uint2 again(const uint2& old) const {
    const float ratio = __fdiv_rn(before, after);
    const float4 a = unquantise4<kE4M3>(old.x), c = unquantise4<kE4M3>(old.y);
    auto times = [&](float v) { return __fmul_rn(v, ratio); };      // (rounded before the number is)
    return make_uint2(quantise4<kE4M3>(times(a.x), times(a.y), times(a.z), times(a.w), 1.f),
                      quantise4<kE4M3>(times(c.x), times(c.y), times(c.z), times(c.w), 1.f));
  }
};
template <typename T>
__device__ __forceinline__ unsigned max_abs8(unsigned m, const uint4& x) {
  return max_abs2<T>(max_abs2<T>(max_abs2<T>(max_abs2<T>(m, x.x), x.y), x.z), x.w);
}
// the larger of the two as 15 bits (which order as the numbers do, NaN above all)
__device__ __forceinline__ unsigned larger(unsigned m) { return max(m & 0x7fffu, (m >> 16) & 0x7fffu); }

// One new row for each sequence: a few kilobytes, so the time is the chain of look-ups (length, page,
// scale).  A group of head_dim / 8 lanes takes the row of one (sequence, head, K or V), which it asks
// for before it knows where it goes, and nothing is shared between groups.
template <typename T, bool kE4M3>
__global__ void __launch_bounds__(kAppendThreads) append_8bit_one_kernel(const AppendParams p) {
  sm100::launch_dependents();
  const int lane = threadIdx.x & 31, lanes = p.head_dim >> 3, at_once = 32 / lanes;
  const int mine = lane / lanes, col = (lane - mine * lanes) * 8;
  const int job = (blockIdx.x * kAppendWarps + (threadIdx.x >> 5)) * at_once + mine;
  const bool some = mine < at_once && job < 2 * p.tokens * p.heads;
  const int which = job & 1, t = (job >> 1) / p.heads, h = (job >> 1) % p.heads;
  sm100::grid_dependency_wait();
  if (!some) return;
  const uint4 x = *reinterpret_cast<const uint4*>((const T*)p.rows[which] + (long long)t * p.row_st[which] +
                                                  h * p.row_sh[which] + col);
  const int len = p.lens[t];
  if (len < 0 || len / p.page_size >= p.width) return;
  const int page = p.table[(long long)t * p.width + len / p.page_size];
  if (page < 0 || page >= p.num_pages) return;
  const int in_page = len % p.page_size, index = in_page / p.block, off = in_page % p.block;
  float* scale = p.scales[which] + page * p.scale_sp[which] + index * p.scale_sb[which] + h * p.scale_sh[which];
  unsigned char* base = (unsigned char*)p.pages[which] + page * p.page_sp[which] +
                        (long long)index * p.block * p.page_st[which] + h * p.page_sh[which] + col;
  const unsigned group = (lanes == 32 ? 0xffffffffu : (1u << lanes) - 1u) << (mine * lanes);
  const float before = off ? *scale : 0.f;
  const unsigned top = __reduce_max_sync(group, larger(max_abs8<T>(0u, x)));
  const Scaling<T, kE4M3> sc(top, before);
  *reinterpret_cast<uint2*>(base + off * p.page_st[which]) = sc.pow2 ? sc.template eight<true>(x) : sc.template eight<false>(x);
  if (off && sc.after > before) {              // (eight rows' loads together: the others wait for this)
    for (int r0 = 0; r0 < off; r0 += 8) {
      uint2 old[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (r0 + i < off) old[i] = *reinterpret_cast<const uint2*>(base + (r0 + i) * p.page_st[which]);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (r0 + i < off) *reinterpret_cast<uint2*>(base + (r0 + i) * p.page_st[which]) = sc.again(old[i]);
    }
  }
  __syncwarp(group);                           // (the others have read the scale)
  if (col == 0) *scale = sc.after;
}

// Packed new rows.  The tasks of all sequences form one list, of which each CTA takes an equal share.  The
// loads of the next task are under way while a warp works on one.
template <typename T, bool kE4M3>
__global__ void __launch_bounds__(kAppendThreads, kCtasPerSm) append_8bit_kernel(const AppendParams p) {
  __shared__ AppendBlock blocks[kListed];
  __shared__ int owner[kListed];               // sequence of a listed block
  __shared__ int nth[kListed];                 // which of the sequence's blocks it is
  __shared__ long long sums[kAppendWarps], share[2];
  __shared__ unsigned tops[2][kAppendWarps];
  sm100::launch_dependents();
  sm100::grid_dependency_wait();
  const int n_jobs = 2 * p.heads;
  long long list0;                             // the first block of the list (of all sequences' blocks)
  {
    long long total = 0, all;
    for (int i0 = 0; i0 < p.batch; i0 += kAppendThreads) {
      sum_before(AppendRun(p, i0 + threadIdx.x).blocks, sums, all);
      total += all;
    }
    if (total > p.tokens / p.block + 2ll * p.batch) return;     // (not ascending: rows of more sequences than one)
    total *= n_jobs;
    list0 = total * blockIdx.x / gridDim.x / n_jobs;
    if (threadIdx.x == 0) {
      share[0] = total * blockIdx.x / gridDim.x;
      share[1] = total * (blockIdx.x + 1) / gridDim.x;
    }
    __syncthreads();
  }
  for (int turn = 0; list0 * n_jobs < share[1]; list0 += kListed) {
  // ---- look the blocks up
  const int n_listed = (int)min((long long)kListed, (share[1] + n_jobs - 1) / n_jobs - list0);
  long long at = -list0;
  for (int i0 = 0; i0 < p.batch && at < n_listed; i0 += kAppendThreads) {
    const AppendRun run(p, i0 + threadIdx.x);
    long long all;
    const long long mine = at + sum_before(run.blocks, sums, all);
    const int end = (int)max(0ll, min((long long)n_listed, mine + run.blocks));
    for (int j = (int)max(0ll, min((long long)n_listed, mine)); j < end; ++j) {
      owner[j] = i0 + threadIdx.x;
      nth[j] = (int)(j - mine);
    }
    at += all;
  }
  __syncthreads();
  if ((int)threadIdx.x < n_listed) {
    const int i = owner[threadIdx.x];
    const AppendRun run(p, i);
    AppendBlock g = {0, 0, 0, 0, 0};
    const int at_block = nth[threadIdx.x];
    if (at_block >= 0 && at_block < run.blocks) {                 // (always, unless someone writes the lengths meanwhile)
      const int skip = run.len & (p.block - 1);                   // tokens of the first block that are there already
      const int r = at_block == 0 ? 0 : at_block * p.block - skip;     // the block's first new row
      const long long pos = (long long)run.len + r;
      const int page = p.table[(long long)i * p.width + pos / p.page_size];
      g.row0 = run.first + r;
      g.off = at_block == 0 ? skip : 0;
      if (page >= 0 && page < p.num_pages) g.fresh = min(run.count - r, p.block - g.off);
      g.page = page;
      g.index = (int)(pos % p.page_size) / p.block;
    }
    blocks[threadIdx.x] = g;
  }
  __syncthreads();
  // ---- the tasks
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int wpt = p.warps_per_task, groups = kAppendWarps / wpt, group = warp / wpt, w = warp - group * wpt;
  const int task_from = (int)max(0ll, share[0] - list0 * n_jobs);
  const int n_tasks = (int)min((long long)n_listed * n_jobs, share[1] - list0 * n_jobs);
  const int lanes = p.head_dim >> 3, rows_at_once = 32 / lanes;      // a lane holds 8 numbers of a row
  const int my_row = lane / lanes, my_col = (lane - my_row * lanes) * 8;
  const bool active = my_row < rows_at_once;
  struct Task {                                // (what else a task needs is looked up again: the registers are rows)
    uint4 x[kUnitRows / 2];                    // the warp's rows of the block
    float before;
  };
  auto load = [&](int task, Task& k) {
    if (task >= n_tasks) return;
    const AppendBlock g = blocks[task / n_jobs];
    const int job = task % n_jobs, which = job & 1, h = job >> 1;
    k.before = 0.f;
    if (g.off && g.fresh)
      k.before = p.scales[which][g.page * p.scale_sp[which] + g.index * p.scale_sb[which] + h * p.scale_sh[which]];
    const T* rows = (const T*)p.rows[which] + h * p.row_sh[which] + my_col;
#pragma unroll
    for (int i = 0; i < kUnitRows / 2; ++i) {
      const int r = w * kUnitRows + i * rows_at_once + my_row - g.off;           // of the block's new rows
      k.x[i] = make_uint4(0, 0, 0, 0);
      if (active && i * rows_at_once < kUnitRows && r >= 0 && r < g.fresh)
        k.x[i] = *reinterpret_cast<const uint4*>(rows + (long long)(g.row0 + r) * p.row_st[which]);
    }
  };
  Task now, next;
  load(task_from + group, now);
  for (int task = task_from + group; task < n_tasks; task += groups, turn ^= 1) {
    load(task + groups, next);
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < kUnitRows / 2; ++i) top = max_abs8<T>(top, now.x[i]);
    top = __reduce_max_sync(0xffffffffu, larger(top));
    if (wpt > 1) {                             // the warps of a task meet (two sets of places, one barrier)
      if (lane == 0) tops[turn][warp] = top;
      asm volatile("bar.sync %0, %1;" :: "r"(1 + group), "r"(wpt * 32) : "memory");
      for (int i = 0; i < wpt; ++i) top = max(top, tops[turn][group * wpt + i]);
    }
    const AppendBlock g = blocks[task / n_jobs];
    if (g.fresh > 0) {
      const int job = task % n_jobs, which = job & 1, h = job >> 1;
      const Scaling<T, kE4M3> sc(top, now.before);
      const long long st = p.page_st[which];
      unsigned char* const base = (unsigned char*)p.pages[which] + g.page * p.page_sp[which] + h * p.page_sh[which] + my_col +
                                  (g.index * p.block + w * kUnitRows + my_row) * st;
      const int r0 = w * kUnitRows + my_row - g.off;                             // the lane's first row among the new ones
      auto store = [&](auto pow2) {
#pragma unroll
        for (int i = 0; i < kUnitRows / 2; ++i) {
          const int r = r0 + i * rows_at_once;
          if (active && i * rows_at_once < kUnitRows && r >= 0 && r < g.fresh)
            *reinterpret_cast<uint2*>(base + i * rows_at_once * st) = sc.template eight<decltype(pow2)::value>(now.x[i]);
        }
      };
      if (sc.pow2) store(std::true_type());
      else store(std::false_type());
      if (g.off && sc.after > now.before)                                        // earlier rows to the new scale
        for (int i = 0; i * rows_at_once < kUnitRows; ++i)
          if (active && r0 + i * rows_at_once < 0) {
            uint2* at = reinterpret_cast<uint2*>(base + i * rows_at_once * st);
            *at = sc.again(*at);
          }
      if (w == 0 && lane == 0)
        p.scales[which][g.page * p.scale_sp[which] + g.index * p.scale_sb[which] + h * p.scale_sh[which]] = sc.after;
    }
    now = next;
  }
  __syncthreads();                             // (the list is read)
  }
}

template <typename T, bool kE4M3>
cudaError_t launch_append(const AppendParams& p, int ctas, cudaStream_t stream) {
  if (!p.cu) {
    const int jobs = 2 * p.tokens * p.heads, each = kAppendWarps * (32 / (p.head_dim / 8));
    return launch_after(append_8bit_one_kernel<T, kE4M3>, dim3((jobs + each - 1) / each), dim3(kAppendThreads), 0, stream, p);
  }
  return launch_after(append_8bit_kernel<T, kE4M3>, dim3(ctas), dim3(kAppendThreads), 0, stream, p);
}

}  // namespace

int kv_append_8bit(const b200attn_kv_append_8bit_args* a, cudaStream_t stream) {
  if (!a || !a->k_pages || !a->v_pages || !a->k_scales || !a->v_scales || !a->page_table || !a->seqlens)
    return B200ATTN_ERR_NULL;
  if (a->tokens > 0 && (!a->new_k || !a->new_v)) return B200ATTN_ERR_NULL;
  if ((a->dtype != B200ATTN_F16 && a->dtype != B200ATTN_BF16) ||
      (a->cache_dtype != B200ATTN_E4M3 && a->cache_dtype != B200ATTN_I8))
    return B200ATTN_ERR_DTYPE;
  if (a->head_dim != 32 && a->head_dim != 64 && a->head_dim != 96 && a->head_dim != 128) return B200ATTN_ERR_HEAD_DIM;
  if (a->batch <= 0 || a->heads <= 0 || a->tokens < 0 || a->num_pages <= 0 || a->max_pages_per_seq <= 0)
    return B200ATTN_ERR_SHAPE;
  if (!a->cu_new && a->tokens != a->batch) return B200ATTN_ERR_SHAPE;
  if (a->block_tokens != 16 && a->block_tokens != 32 && a->block_tokens != 64 && a->block_tokens != 128)
    return B200ATTN_ERR_MODE;
  if (a->page_size <= 0 || a->page_size % a->block_tokens != 0) return B200ATTN_ERR_MODE;
  if (a->tokens > INT_MAX - kListed || a->heads > 16384) return B200ATTN_ERR_TOO_LARGE;
  if (!a->cu_new && 2 * a->tokens * a->heads > INT_MAX - 65536) return B200ATTN_ERR_TOO_LARGE;
  const void* ptrs[4] = {a->new_k, a->new_v, a->k_pages, a->v_pages};
  for (const void* q : ptrs)
    if ((uintptr_t)q & 15) return B200ATTN_ERR_ALIGN;
  if (!aligned4({a->k_scales, a->v_scales, a->page_table, a->seqlens, a->cu_new})) return B200ATTN_ERR_ALIGN;
  const long long rows[4] = {a->nk_stride_t, a->nk_stride_h, a->nv_stride_t, a->nv_stride_h};
  for (long long s : rows)
    if (s % 8 != 0) return B200ATTN_ERR_STRIDE;
  const long long pools[6] = {a->k_stride_page, a->k_stride_t, a->k_stride_h,
                              a->v_stride_page, a->v_stride_t, a->v_stride_h};
  for (long long s : pools)
    if (s % 16 != 0) return B200ATTN_ERR_STRIDE;
  // what is written lies apart (an axis of one may have any stride)
  auto meets = [](long long extent, long long stride) { return extent > 1 && stride == 0; };
  const int blocks = a->page_size / a->block_tokens;
  if (meets(a->num_pages, a->k_stride_page) || meets(a->num_pages, a->v_stride_page) || meets(a->page_size, a->k_stride_t) ||
      meets(a->page_size, a->v_stride_t) || meets(a->heads, a->k_stride_h) || meets(a->heads, a->v_stride_h) ||
      meets(a->num_pages, a->ks_stride_page) || meets(a->num_pages, a->vs_stride_page) || meets(blocks, a->ks_stride_blk) ||
      meets(blocks, a->vs_stride_blk) || meets(a->heads, a->ks_stride_h) || meets(a->heads, a->vs_stride_h))
    return B200ATTN_ERR_STRIDE;
  const DeviceInfo* di = nullptr;
  if (int st = device_info(&di)) return st;
  set_launch_count(0);
  if (a->tokens == 0) return B200ATTN_OK;
  AppendParams p;
  p.rows[0] = a->new_k; p.rows[1] = a->new_v;
  p.pages[0] = a->k_pages; p.pages[1] = a->v_pages;
  p.scales[0] = a->k_scales; p.scales[1] = a->v_scales;
  p.row_st[0] = a->nk_stride_t; p.row_sh[0] = a->nk_stride_h;
  p.row_st[1] = a->nv_stride_t; p.row_sh[1] = a->nv_stride_h;
  p.page_sp[0] = a->k_stride_page; p.page_st[0] = a->k_stride_t; p.page_sh[0] = a->k_stride_h;
  p.page_sp[1] = a->v_stride_page; p.page_st[1] = a->v_stride_t; p.page_sh[1] = a->v_stride_h;
  p.scale_sp[0] = a->ks_stride_page; p.scale_sb[0] = a->ks_stride_blk; p.scale_sh[0] = a->ks_stride_h;
  p.scale_sp[1] = a->vs_stride_page; p.scale_sb[1] = a->vs_stride_blk; p.scale_sh[1] = a->vs_stride_h;
  p.table = a->page_table; p.lens = a->seqlens; p.cu = a->cu_new;
  p.tokens = (int)a->tokens; p.batch = a->batch; p.heads = a->heads; p.head_dim = a->head_dim;
  p.page_size = a->page_size; p.block = a->block_tokens; p.num_pages = a->num_pages; p.width = a->max_pages_per_seq;
  p.warps_per_task = a->block_tokens / kUnitRows;
  // Packed rows: as many CTAs as are resident at once, or one for each of its tasks at a time where those are fewer.
  const long long groups = kAppendWarps / p.warps_per_task;
  const long long tasks = 2ll * a->heads * (a->tokens / a->block_tokens + 2ll * std::min<long long>(a->batch, a->tokens));
  const int ctas = (int)std::min<long long>((long long)kCtasPerSm * di->sm_count, (tasks + groups - 1) / groups);
  const bool e4m3 = a->cache_dtype == B200ATTN_E4M3;
  const cudaError_t e = a->dtype == B200ATTN_F16 ? (e4m3 ? launch_append<__half, true>(p, ctas, stream) : launch_append<__half, false>(p, ctas, stream))
                                                 : (e4m3 ? launch_append<__nv_bfloat16, true>(p, ctas, stream)
                                                         : launch_append<__nv_bfloat16, false>(p, ctas, stream));
  if (e != cudaSuccess) return B200ATTN_ERR_CUDA;
  set_launch_count(1);
  return cudaGetLastError() == cudaSuccess ? B200ATTN_OK : B200ATTN_ERR_CUDA;
}

}  // namespace b200attn
