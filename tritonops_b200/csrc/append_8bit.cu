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
// and row, stay in registers between the maximum and the rounding, and leave as 8-byte pieces.  The
// CTA that holds a block's first new token does the whole block, so no two CTAs share a scale.
#include <limits.h>

#include <algorithm>

#include "common.cuh"
#include "sm100.cuh"

namespace b200attn {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kAppendWarps = kAppendThreads / 32;
constexpr int kMaxBlockTokens = 128;
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
  int tile;                        // tokens whose blocks a CTA looks after
  int warps_per_task;              // one for each 16-row unit of a block that can hold new rows
  int jobs_per_cta;                // (head, K or V) pairs of a CTA
};

// one block that begins to be written in the CTA's tile
struct AppendBlock {
  int row0;                        // its first new row
  int off, fresh;                  // tokens the block holds already, new ones
  int page, index;                 // page of the pool, block of the page
};

__device__ __forceinline__ unsigned max_abs16(unsigned m, unsigned x) { return __vmaxu2(m, x & 0x7fff7fffu); }

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

// round(x / s), four numbers
template <bool kE4M3>
__device__ __forceinline__ unsigned quantise4(float a, float b, float c, float d) {
  if (kE4M3) {
    unsigned short lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return (unsigned)lo | ((unsigned)hi << 16);
  }
  auto one = [](float x) { return (unsigned)min(max(__float2int_rn(x), -127), 127) & 255u; };
  return one(a) | (one(b) << 8) | (one(c) << 16) | (one(d) << 24);
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

template <typename T, bool kE4M3>
__global__ void __launch_bounds__(kAppendThreads) append_8bit_kernel(const AppendParams p) {
  __shared__ AppendBlock blocks[kMaxBlockTokens];
  __shared__ int n_blocks;
  __shared__ unsigned tops[kAppendWarps];
  sm100::launch_dependents();
  if (threadIdx.x == 0) n_blocks = 0;
  sm100::grid_dependency_wait();
  // ---- which blocks begin to be written in this tile
  const int t0 = blockIdx.x * p.tile;
  int b = t0;
  if (p.cu) {
    b = 0;                                     // sequences that end at or before t0
    for (int i0 = 0; i0 < p.batch; i0 += kAppendThreads) {
      const int i = i0 + threadIdx.x;
      b += __syncthreads_count(i < p.batch && p.cu[i + 1] <= t0);
    }
  }
  __syncthreads();
  const int t = t0 + threadIdx.x;
  if ((int)threadIdx.x < p.tile && t < p.tokens) {
    int first = t, end = t + 1;
    if (p.cu) {
      while (b < p.batch && p.cu[b + 1] <= t) ++b;
      if (b < p.batch) { first = p.cu[b]; end = min(p.cu[b + 1], p.tokens); }
    } else {
      b = t;
    }
    if (b < p.batch && first >= 0 && first <= t) {
      const int len = p.lens[b];
      const long long pos = (long long)len + (t - first);
      const int off = (int)(pos % p.block);
      if (len >= 0 && (t == first || off == 0) && pos / p.page_size < p.width) {
        const int page = p.table[(long long)b * p.width + pos / p.page_size];
        if (page >= 0 && page < p.num_pages) {
          AppendBlock& g = blocks[atomicAdd(&n_blocks, 1)];
          g.row0 = t; g.off = off; g.fresh = min(end - t, p.block - off);
          g.page = page; g.index = (int)(pos % p.page_size) / p.block;
        }
      }
    }
  }
  __syncthreads();
  // ---- the tasks
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int groups = kAppendWarps / p.warps_per_task, group = warp / p.warps_per_task;
  const int w = warp - group * p.warps_per_task;
  const int job0 = blockIdx.y * p.jobs_per_cta, n_jobs = min(p.jobs_per_cta, 2 * p.heads - job0);
  const int n_tasks = n_blocks * n_jobs;
  const int lanes = p.head_dim >> 3, rows_at_once = 32 / lanes;      // a lane holds 8 numbers of a row
  const int my_row = lane / lanes, my_col = (lane - my_row * lanes) * 8;
  const bool active = my_row < rows_at_once;
  for (int task0 = 0; task0 < n_tasks; task0 += groups) {
    const int task = task0 + group;
    const bool some = task < n_tasks;
    AppendBlock g = {};
    int which = 0, h = 0;
    uint4 x[kUnitRows / 2];
    unsigned top = 0;
    float before = 0.f;
    float* scale = nullptr;
    unsigned char* base = nullptr;
    int unit = 0;                              // the warp's unit with new rows
    if (some) {
      g = blocks[task / n_jobs];
      const int job = job0 + task % n_jobs;
      which = job & 1; h = job >> 1;
      scale = p.scales[which] + g.page * p.scale_sp[which] + g.index * p.scale_sb[which] + h * p.scale_sh[which];
      base = (unsigned char*)p.pages[which] + g.page * p.page_sp[which] +
             (long long)g.index * p.block * p.page_st[which] + h * p.page_sh[which];
      if (g.off) before = *scale;
      unit = p.warps_per_task == 1 ? g.off / kUnitRows : w;
      const T* rows = (const T*)p.rows[which] + h * p.row_sh[which] + my_col;
#pragma unroll
      for (int i = 0; i < kUnitRows / 2; ++i) {
        const int r = unit * kUnitRows + i * rows_at_once + my_row - g.off;      // of the block's new rows
        x[i] = make_uint4(0, 0, 0, 0);
        if (active && i * rows_at_once < kUnitRows && r >= 0 && r < g.fresh)
          x[i] = *reinterpret_cast<const uint4*>(rows + (long long)(g.row0 + r) * p.row_st[which]);
      }
#pragma unroll
      for (int i = 0; i < kUnitRows / 2; ++i)
        top = max_abs16(max_abs16(max_abs16(max_abs16(top, x[i].x), x[i].y), x[i].z), x[i].w);
      top = max(top & 0xffffu, top >> 16);
      top = __reduce_max_sync(0xffffffffu, top);
    }
    if (p.warps_per_task > 1) {
      __syncthreads();                         // (the task before has read them)
      if (lane == 0) tops[warp] = top;
      __syncthreads();
      for (int i = 0; i < p.warps_per_task; ++i) top = max(top, tops[group * p.warps_per_task + i]);
    }
    if (!some) continue;
    const float need = scale_for<T, kE4M3>(top);
    const float after = (need != need || before != before) ? __uint_as_float(0x7fc00000u) : fmaxf(need, before);
    // the reciprocal of a power of two is exact; scales that came from elsewhere are divided by
    const unsigned bits = __float_as_uint(after);
    const bool pow2 = (bits & 0x7fffffu) == 0 && bits >= 0x00800000u && bits < 0x7f000000u;
    const float inv = pow2 ? __uint_as_float(0x7f000000u - bits) : 0.f;
    const bool stored = after > 0.f;           // (false for NaN: numbers of such a block are 0)
    auto over = [&](float v) { return !stored ? 0.f : pow2 ? v * inv : __fdiv_rn(v, after); };
#pragma unroll
    for (int i = 0; i < kUnitRows / 2; ++i) {
      const int r = unit * kUnitRows + i * rows_at_once + my_row;                // of the block
      if (active && i * rows_at_once < kUnitRows && r >= g.off && r - g.off < g.fresh) {
        const float2 a = unpack2<T>(x[i].x), c = unpack2<T>(x[i].y), d = unpack2<T>(x[i].z), e = unpack2<T>(x[i].w);
        const uint2 q = make_uint2(quantise4<kE4M3>(over(a.x), over(a.y), over(c.x), over(c.y)),
                                   quantise4<kE4M3>(over(d.x), over(d.y), over(e.x), over(e.y)));
        *reinterpret_cast<uint2*>(base + r * p.page_st[which] + my_col) = q;
      }
    }
    if (g.off && after > before) {             // earlier rows of the block to the new scale
      const float ratio = __fdiv_rn(before, after);
      for (int u = w; u * kUnitRows < g.off; u += p.warps_per_task)
        for (int i = 0; i * rows_at_once < kUnitRows; ++i) {
          const int r = u * kUnitRows + i * rows_at_once + my_row;
          if (active && r < g.off) {
            uint2* at = reinterpret_cast<uint2*>(base + r * p.page_st[which] + my_col);
            const uint2 old = *at;
            const float4 a = unquantise4<kE4M3>(old.x), c = unquantise4<kE4M3>(old.y);
            *at = make_uint2(quantise4<kE4M3>(a.x * ratio, a.y * ratio, a.z * ratio, a.w * ratio),
                             quantise4<kE4M3>(c.x * ratio, c.y * ratio, c.z * ratio, c.w * ratio));
          }
        }
    }
    if (w == 0 && lane == 0) *scale = after;
  }
}

template <typename T>
cudaError_t launch_append(const b200attn_kv_append_8bit_args* a, const AppendParams& p, dim3 grid, cudaStream_t stream) {
  return a->cache_dtype == B200ATTN_E4M3
             ? launch_after(append_8bit_kernel<T, true>, grid, dim3(kAppendThreads), 0, stream, p)
             : launch_after(append_8bit_kernel<T, false>, grid, dim3(kAppendThreads), 0, stream, p);
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
  if (a->tokens > INT_MAX - kMaxBlockTokens || a->heads > 16384) return B200ATTN_ERR_TOO_LARGE;
  const void* ptrs[4] = {a->new_k, a->new_v, a->k_pages, a->v_pages};
  for (const void* q : ptrs)
    if ((uintptr_t)q & 15) return B200ATTN_ERR_ALIGN;
  if (((uintptr_t)a->k_scales | (uintptr_t)a->v_scales) & 3) return B200ATTN_ERR_ALIGN;
  const long long rows[4] = {a->nk_stride_t, a->nk_stride_h, a->nv_stride_t, a->nv_stride_h};
  for (long long s : rows)
    if (s % 8 != 0) return B200ATTN_ERR_STRIDE;
  const long long pools[6] = {a->k_stride_page, a->k_stride_t, a->k_stride_h,
                              a->v_stride_page, a->v_stride_t, a->v_stride_h};
  for (long long s : pools)
    if (s % 16 != 0) return B200ATTN_ERR_STRIDE;
  if (int st = device_info(nullptr)) return st;
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
  // One new token each: a CTA per token and eight (head, K or V) pairs, a warp each.  Packed rows: a
  // CTA looks after a block's worth of them, with a warp for each of a block's units.
  p.tile = a->cu_new ? a->block_tokens : 1;
  p.warps_per_task = a->cu_new ? a->block_tokens / kUnitRows : 1;
  p.jobs_per_cta = std::min(kAppendWarps / p.warps_per_task, 2 * a->heads);
  const dim3 grid((unsigned)((a->tokens + p.tile - 1) / p.tile),
                  (unsigned)((2 * a->heads + p.jobs_per_cta - 1) / p.jobs_per_cta));
  const cudaError_t e = a->dtype == B200ATTN_F16 ? launch_append<__half>(a, p, grid, stream)
                                                 : launch_append<__nv_bfloat16>(a, p, grid, stream);
  if (e != cudaSuccess) return B200ATTN_ERR_CUDA;
  set_launch_count(1);
  return cudaGetLastError() == cudaSuccess ? B200ATTN_OK : B200ATTN_ERR_CUDA;
}

}  // namespace b200attn
