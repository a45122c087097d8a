// Attention of the newest tokens of each sequence over a paged cache of 8-bit numbers with a scale
// for each block of tokens and head, for sm_100a.  The reference decodes over 16-bit padded caches
// (flash_attn_triton/flash_attn_decoding.py:9-210).
//
//   k_t = ks[page, block, h] * kq_t,   v_t = vs[page, block, h] * vq_t
//   o_i = sum_t softmax_t(scale * q_i . k_t) v_t      over t < len - n + 1 + i for query i of n
#include <limits.h>

#include <algorithm>

#include "common.cuh"
#include "sm100.cuh"

namespace b200attn {
namespace {

struct Decode8Params {
  const void* q;
  const void* k;
  const void* v;
  const float* ks;
  const float* vs;
  void* o;
  const int32_t* table;
  const int32_t* lens;
  long long q_sb, q_st, q_sh, o_sb, o_st, o_sh;
  long long k_sp, k_st, k_sh, v_sp, v_st, v_sh;
  long long ks_sp, ks_sb, ks_sh, vs_sp, vs_sb, vs_sh;
  int batch, queries, heads_q, heads_kv, group, head_dim;
  int page_size, block, num_pages, width, max_len;
  float scale_log2;
};

template <bool kE4M3>
__device__ __forceinline__ float number(unsigned char x) {
  if (!kE4M3) return (float)(signed char)x;
  unsigned r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((unsigned short)x));
  return __half2float(__ushort_as_half((unsigned short)(r & 0xffffu)));
}

// One warp per query row, a key at a time: the form everything else is checked against.
template <typename T, bool kE4M3>
__global__ void __launch_bounds__(128) decode_8bit_rows_kernel(const Decode8Params p) {
  sm100::launch_dependents();
  sm100::grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= (long long)p.batch * p.queries * p.heads_q) return;
  const int hq = (int)(row % p.heads_q), i = (int)(row / p.heads_q % p.queries);
  const int b = (int)(row / p.heads_q / p.queries), h = hq / p.group;
  const int len = min(max(p.lens[b], 0), p.max_len), n = len - p.queries + 1 + i;
  const T* q = (const T*)p.q + b * p.q_sb + i * p.q_st + hq * p.q_sh;
  float qv[4], acc[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) qv[j] = lane + 32 * j < p.head_dim ? (float)q[lane + 32 * j] * p.scale_log2 : 0.f;
  for (int t = 0; t < n; ++t) {
    const int page = p.table[(long long)b * p.width + t / p.page_size], r = t % p.page_size, blk = r / p.block;
    if (page < 0 || page >= p.num_pages) continue;
    const unsigned char* k = (const unsigned char*)p.k + page * p.k_sp + r * p.k_st + h * p.k_sh;
    const unsigned char* v = (const unsigned char*)p.v + page * p.v_sp + r * p.v_st + h * p.v_sh;
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (lane + 32 * j < p.head_dim) s += qv[j] * number<kE4M3>(k[lane + 32 * j]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    s *= p.ks[page * p.ks_sp + blk * p.ks_sb + h * p.ks_sh];
    const float top = fmaxf(m, s), use = top == -INFINITY ? 0.f : top;
    const float old = exp2f(m - use), w = exp2f(s - use);
    m = top;
    l = l * old + w;
    const float wv = w * p.vs[page * p.vs_sp + blk * p.vs_sb + h * p.vs_sh];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (lane + 32 * j < p.head_dim) acc[j] = acc[j] * old + wv * number<kE4M3>(v[lane + 32 * j]);
  }
  T* o = (T*)p.o + b * p.o_sb + i * p.o_st + hq * p.o_sh;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (lane + 32 * j < p.head_dim) o[lane + 32 * j] = from_float<T>(l == 0.f ? 0.f : acc[j] / l);
}

int validate(const b200attn_paged_decode_8bit_args* a) {
  if (!a || !a->q || !a->k_pages || !a->v_pages || !a->k_scales || !a->v_scales || !a->o || !a->page_table ||
      !a->seqlens)
    return B200ATTN_ERR_NULL;
  if ((a->dtype != B200ATTN_F16 && a->dtype != B200ATTN_BF16) ||
      (a->cache_dtype != B200ATTN_E4M3 && a->cache_dtype != B200ATTN_I8))
    return B200ATTN_ERR_DTYPE;
  if (a->head_dim != 32 && a->head_dim != 64 && a->head_dim != 96 && a->head_dim != 128) return B200ATTN_ERR_HEAD_DIM;
  if (a->batch <= 0 || a->queries <= 0 || a->heads_q <= 0 || a->heads_kv <= 0 || a->max_seqlen < 0 ||
      a->num_pages <= 0 || a->max_pages_per_seq <= 0)
    return B200ATTN_ERR_SHAPE;
  if (a->batch > 65535) return B200ATTN_ERR_TOO_LARGE;
  if (a->heads_q % a->heads_kv != 0) return B200ATTN_ERR_GQA;
  if (a->block_tokens != 16 && a->block_tokens != 32 && a->block_tokens != 64 && a->block_tokens != 128)
    return B200ATTN_ERR_MODE;
  if (a->page_size <= 0 || a->page_size % a->block_tokens != 0) return B200ATTN_ERR_MODE;
  const void* ptrs[3] = {a->q, a->k_pages, a->v_pages};
  for (const void* ptr : ptrs)
    if ((uintptr_t)ptr & 15) return B200ATTN_ERR_ALIGN;
  if (((uintptr_t)a->o & 1) || (((uintptr_t)a->k_scales | (uintptr_t)a->v_scales) & 3)) return B200ATTN_ERR_ALIGN;
  const long long rows[3] = {a->q_stride_b, a->q_stride_t, a->q_stride_h};
  for (long long s : rows)
    if (s % 8 != 0) return B200ATTN_ERR_STRIDE;
  const long long pools[6] = {a->k_stride_page, a->k_stride_t, a->k_stride_h,
                              a->v_stride_page, a->v_stride_t, a->v_stride_h};
  for (long long s : pools)
    if (s % 16 != 0) return B200ATTN_ERR_STRIDE;
  if (a->chunk_tokens < 0 || a->chunk_tokens % 128 != 0) return B200ATTN_ERR_SHAPE;
  return B200ATTN_OK;
}

}  // namespace

size_t paged_decode_8bit_workspace_bytes(const b200attn_paged_decode_8bit_args* a) {
  return a ? 16 : 0;
}

int paged_decode_8bit_fwd(const b200attn_paged_decode_8bit_args* a, cudaStream_t stream) {
  int st = validate(a);
  if (st != B200ATTN_OK) return st;
  if (!a->workspace || a->workspace_bytes < paged_decode_8bit_workspace_bytes(a)) return B200ATTN_ERR_WORKSPACE;
  if ((st = device_info(nullptr)) != B200ATTN_OK) return st;
  Decode8Params p;
  p.q = a->q; p.k = a->k_pages; p.v = a->v_pages; p.ks = a->k_scales; p.vs = a->v_scales; p.o = a->o;
  p.table = a->page_table; p.lens = a->seqlens;
  p.q_sb = a->q_stride_b; p.q_st = a->q_stride_t; p.q_sh = a->q_stride_h;
  p.o_sb = a->o_stride_b; p.o_st = a->o_stride_t; p.o_sh = a->o_stride_h;
  p.k_sp = a->k_stride_page; p.k_st = a->k_stride_t; p.k_sh = a->k_stride_h;
  p.v_sp = a->v_stride_page; p.v_st = a->v_stride_t; p.v_sh = a->v_stride_h;
  p.ks_sp = a->ks_stride_page; p.ks_sb = a->ks_stride_blk; p.ks_sh = a->ks_stride_h;
  p.vs_sp = a->vs_stride_page; p.vs_sb = a->vs_stride_blk; p.vs_sh = a->vs_stride_h;
  p.batch = a->batch; p.queries = a->queries; p.heads_q = a->heads_q; p.heads_kv = a->heads_kv;
  p.group = a->heads_q / a->heads_kv; p.head_dim = a->head_dim;
  p.page_size = a->page_size; p.block = a->block_tokens; p.num_pages = a->num_pages; p.width = a->max_pages_per_seq;
  p.max_len = (int)std::min<long long>(a->max_seqlen, (long long)a->max_pages_per_seq * a->page_size);
  p.scale_log2 = a->softmax_scale * 1.4426950408889634f;
  const long long rows = (long long)a->batch * a->queries * a->heads_q;
  if (rows > INT_MAX) return B200ATTN_ERR_TOO_LARGE;
  const dim3 grid((unsigned)((rows + 3) / 4));
  auto go = [&](auto kernel) { return launch_after(kernel, grid, dim3(128), 0, stream, p); };
  const bool e4m3 = a->cache_dtype == B200ATTN_E4M3;
  const cudaError_t e = a->dtype == B200ATTN_F16
                            ? (e4m3 ? go(decode_8bit_rows_kernel<__half, true>) : go(decode_8bit_rows_kernel<__half, false>))
                            : (e4m3 ? go(decode_8bit_rows_kernel<__nv_bfloat16, true>)
                                    : go(decode_8bit_rows_kernel<__nv_bfloat16, false>));
  if (e != cudaSuccess) return B200ATTN_ERR_CUDA;
  set_launch_count(1);
  return cudaGetLastError() == cudaSuccess ? B200ATTN_OK : B200ATTN_ERR_CUDA;
}

}  // namespace b200attn
