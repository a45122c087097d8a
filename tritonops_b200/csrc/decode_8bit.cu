// Attention of the newest tokens of each sequence over a paged cache of 8-bit numbers with a scale
// for each block of tokens and head, for sm_100a.  The reference decodes over 16-bit padded caches
// (flash_attn_triton/flash_attn_decoding.py:9-210).
//
//   k_t = ks[page, block, h] * kq_t,   v_t = vs[page, block, h] * vq_t
//   o_i = sum_t softmax_t(scale * q_i . k_t) v_t      over t < len - n + 1 + i for query i of n
//
// Every cached byte is used once, so the kernel is a stream: a producer warp brings 128-key stages of
// K and V through a shared-memory ring with the copy engine, four consumer warps take 32 keys each.
// With 8-bit numbers the tensor cores want twice the keys per second that 16-bit rows ask for, so
// what a byte costs on the way decides (counted per 16 keys of a 128-wide head, for which the memory
// leaves an SM ~180 cycles):
//   * K goes to registers as 16-byte pieces in the order they lie in, already the B operand of
//       S[r, t] = sum_d Q[r, d] K[t, d]       (A = Q, 16 rows; the sum's order of d is free, and Q is
//     read in the same order), V as ldmatrix.trans of byte pairs, already the A operand of
//       O^T[d, r] = sum_t V[t, d] P[r, t]     (even and odd d of a pair are rows g and g + 8; the C
//     fragment of S is the B fragment of P as it stands).  Nothing is shuffled or written back.
//   * The numbers become fp16, which holds e4m3 and int8 exactly: one conversion for two e4m3
//     numbers, a byte permute and a subtraction for two int8 ones.
//   * ks multiplies the fp32 scores.  vs multiplies the fp32 product of the keys that share it (one
//     FMA per number of O and 16 or 32 keys): in P or in V it would have to be rounded, or could
//     leave fp16's range.
// bf16 queries are scaled by a power of two per row so that fp16 holds them; P is 2^10 times the
// weight, which keeps weights down to 2^-24 of the largest one out of fp16's subnormals.
#include <limits.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "sm100.cuh"

namespace b200attn {
namespace {

constexpr int kStageKeys = 128;    // keys per ring stage
constexpr int kWarpKeys = 32;      // of which a consumer warp takes
constexpr int kUnitKeys = 16;      // keys that are sure to share a page and a scale
constexpr int kUnits = kStageKeys / kUnitKeys;
constexpr int kRowsTile = 16;      // query rows (query x head of the group) of a work item
constexpr float kPUp = 10.f;       // P is 2^kPUp times the weight

struct Decode8Params {
  const void* q;
  const float* ks;
  const float* vs;
  void* o;
  float* part_o;     // [batch, heads_kv * rows, max_chunks, D] fp32, normalised inside the chunk
  float* part_lse;   // [batch, heads_kv * rows, max_chunks] base-2
  const int32_t* table;
  const int32_t* lens;
  int* status_word;
  long long q_sb, q_st, q_sh, o_sb, o_st, o_sh;
  long long ks_sp, ks_sb, ks_sh, vs_sp, vs_sb, vs_sh;
  int batch, queries, heads_kv, group, head_dim;
  int rows, tiles;   // queries * group rows of a KV head, in tiles of 16
  int page_size, block, num_pages, width, max_len;
  int box_keys;      // keys of a copy: the largest power of two, up to a stage, that divides a page
  int chunk, max_chunks, take_over, direct_o;
  float scale_log2;
};

// keys that query i of a sequence sees
__device__ __forceinline__ int visible(const Decode8Params& p, int len, int i) { return max(len - p.queries + 1 + i, 0); }
__device__ __forceinline__ int length_of(const Decode8Params& p, int b) { return min(max(p.lens[b], 0), p.max_len); }

// one work item as the producer hands it to the consumers
struct Decode8Item {
  int x, b, chunk_id;    // grid coordinates: KV head and row tile, sequence, chunk
  int c_begin, c_end;    // the keys that some row of the tile sees
  int len;
  int valid;             // 0: no more items
  int pad;
};

template <int DP>
struct Decode8Smem {
  static constexpr int kTileBytes = kStageKeys * DP;       // K or V of one stage
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kStages = DP == 128 ? 3 : 6;
  static constexpr int kQ = kStages * kStageBytes;         // the item's 16 query rows, fp16
  static constexpr int kQPitch = DP * 2 + 16;              // bytes
  static constexpr int kFold = kQ + kRowsTile * kQPitch;   // [4 warps][16 rows][32 columns] or [8][64], padded
  static constexpr int kFoldBytes = 4 * 16 * 36 * 4;
  static constexpr int kMl = kFold + kFoldBytes;           // row max and sum, [2][4 warps][16]
  static constexpr int kRowScale = kMl + 2 * 4 * 16 * 4;   // [16] what the query rows were divided by
  static constexpr int kScales = kRowScale + 64;           // [stage][unit] (ks, vs)
  static constexpr int kMask = kScales + kStages * kUnits * 8;   // [stage] units whose page is in the pool
  static constexpr int kItem = kMask + 32;
  static constexpr int kNext = kItem + 32;                 // response of the launch control (16 bytes)
  static constexpr int kBarOffset = kNext + 16;
  static constexpr int kBytes = kBarOffset + (2 * kStages + 3) * 8 + 16;
  static constexpr int kAlloc = kBytes + 1024;
  static_assert(kFold % 16 == 0 && kScales % 8 == 0 && kNext % 16 == 0 && kBarOffset % 8 == 0, "aligned");
  static_assert(kFoldBytes >= 4 * 8 * 68 * 4, "either form of the fold");
  static_assert(2 * (kAlloc + 1024) <= 228 * 1024, "two CTAs per SM");
};

__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, unsigned& r0, unsigned& r1, unsigned& r2, unsigned& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr));
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(addr));
  return r;
}
// barrier of the 128 consumer threads; true if `flag` is for any of them
__device__ __forceinline__ bool consumers_any(bool flag) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(flag ? 1u : 0u)
      : "memory");
  return r != 0;
}

__device__ __forceinline__ unsigned e4m3_pair(unsigned short x) {
  unsigned r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(x));
  return r;
}
// int8 -> fp16: the byte plus 128 under the exponent of 1024, minus 1152
__device__ __forceinline__ unsigned minus_1152(unsigned x) {
  unsigned r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(0x64806480u));
  return r;
}
// four numbers as two pairs: (0, 1) and (2, 3)
template <bool kE4M3>
__device__ __forceinline__ void neighbours(unsigned w, unsigned& lo, unsigned& hi) {
  if (kE4M3) {
    lo = e4m3_pair((unsigned short)(w & 0xffffu));
    hi = e4m3_pair((unsigned short)(w >> 16));
  } else {
    const unsigned x = w ^ 0x80808080u;
    lo = minus_1152(__byte_perm(x, 0x64646464u, 0x4140));
    hi = minus_1152(__byte_perm(x, 0x64646464u, 0x4342));
  }
}
// four numbers as two pairs: (0, 2) and (1, 3)
template <bool kE4M3>
__device__ __forceinline__ void alternates(unsigned w, unsigned& even, unsigned& odd) {
  if (kE4M3) {
    const unsigned a = e4m3_pair((unsigned short)(w & 0xffffu)), b = e4m3_pair((unsigned short)(w >> 16));
    even = __byte_perm(a, b, 0x5410);
    odd = __byte_perm(a, b, 0x7632);
  } else {
    const unsigned x = w ^ 0x80808080u;
    even = minus_1152(__byte_perm(x, 0x64646464u, 0x4240));
    odd = minus_1152(__byte_perm(x, 0x64646464u, 0x4341));
  }
}

// T: the type of q and o.  kRows: 8 or 16 query rows are in use.
template <typename T, bool kE4M3, int DP, int kRows>
__global__ void __launch_bounds__(160, 2)
decode_8bit_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                   const Decode8Params p) {
  using L = Decode8Smem<DP>;
  using namespace sm100;
  constexpr int kChunks16 = DP / 16;      // 16-byte pieces of a row
  constexpr int kQJ = DP / 64;            // pieces of a K row a lane takes
  constexpr int kNT = kRows / 8;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* sgen = smem_raw + (sbase - smem_u32(smem_raw));
  const uint32_t bars = sbase + L::kBarOffset;
  auto full = [&](int s) { return bars + 8 * s; };
  auto empty = [&](int s) { return bars + 8 * (L::kStages + s); };
  const uint32_t item_full = bars + 16 * L::kStages, item_empty = item_full + 8, next_full = item_full + 16;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sgen + L::kBarOffset + (2 * L::kStages + 3) * 8);
  volatile Decode8Item* item = reinterpret_cast<volatile Decode8Item*>(sgen + L::kItem);
  volatile float2* unit_scales = reinterpret_cast<volatile float2*>(sgen + L::kScales);
  volatile unsigned* unit_mask = reinterpret_cast<volatile unsigned*>(sgen + L::kMask);
  volatile float* row_scale = reinterpret_cast<volatile float*>(sgen + L::kRowScale);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // (set up under the tail of the kernel before this one; the combine kernel may be set up from here on)
  launch_dependents();
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < L::kStages; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 4); }
    mbar_init(item_full, 1);
    mbar_init(item_empty, 4);
    mbar_init(next_full, 1);
    fence_barrier_init();
    fence_proxy_async();
  }
  if (threadIdx.x == 128) { prefetch_tmap(&tmap_k); prefetch_tmap(&tmap_v); }
  grid_dependency_wait();
  __syncthreads();

  // A wait by a whole warp, answered alike in all of its lanes.
  auto warp_wait = [&](uint32_t bar, uint32_t parity) -> bool {
    const bool done = mbar_wait(bar, parity, abort_flag);
    return __all_sync(0xffffffffu, done);
  };
  if (warp == 4) {
    // ================================================================ producer
    int x = blockIdx.x, b = blockIdx.y, chunk_id = blockIdx.z;
    int issued = 0;                       // stages sent so far, over all items
    bool ok = true;
    for (int n_item = 0; ok; ++n_item) {
      bool asked = false;
      const int hk = x / p.tiles, tile = x - hk * p.tiles, row0 = tile * kRowsTile;
      const int len = length_of(p, b);
      const int n_vis = visible(p, len, (min(row0 + kRowsTile, p.rows) - 1) / p.group);
      const int c_begin = min(chunk_id * p.chunk, n_vis);
      const int c_end = min(n_vis, c_begin + p.chunk);
      const int n_stages = (c_end - c_begin + kStageKeys - 1) / kStageKeys;
      // Lane i looks after unit i of the next four stages: its page, asked for a batch ahead, and
      // its scales, asked for half a batch ahead.
      const int32_t* pages = p.table + (long long)b * p.width;
      auto page_of = [&](int t) -> int {
        if (t >= c_end) return -1;
        const int e = pages[t / p.page_size];
        return e >= 0 && e < p.num_pages ? e : -1;
      };
      auto scales_of = [&](int t, int page) -> float2 {
        if (page < 0) return make_float2(0.f, 0.f);
        const int blk = t % p.page_size / p.block;
        return make_float2(p.ks[page * p.ks_sp + blk * p.ks_sb + hk * p.ks_sh],
                           p.vs[page * p.vs_sp + blk * p.vs_sb + hk * p.vs_sh]);
      };
      int t_mine = c_begin + kUnitKeys * lane;
      int page = page_of(t_mine), page_nx = page_of(t_mine + 32 * kUnitKeys);
      float2 sc = scales_of(t_mine, page), sc_nx = make_float2(0.f, 0.f);
      // the item's query rows, and what they are divided by so that fp16 holds them
      constexpr int kVec = DP / 8;        // 16-byte pieces of a row
      uint4 qv[kRowsTile * kVec / 32];
#pragma unroll
      for (int i = 0; i < kRowsTile * kVec / 32; ++i) {
        const int r = row0 + (lane + 32 * i) / kVec, c = (lane + 32 * i) % kVec;
        qv[i] = make_uint4(0, 0, 0, 0);
        if (r < p.rows && 8 * c < p.head_dim)
          qv[i] = *reinterpret_cast<const uint4*>((const T*)p.q + b * p.q_sb + r / p.group * p.q_st +
                                                  (hk * p.group + r % p.group) * p.q_sh + 8 * c);
      }
      auto publish = [&]() -> bool {
        if (!warp_wait(item_empty, (n_item & 1) ^ 1)) return false;
#pragma unroll
        for (int i = 0; i < kRowsTile * kVec / 32; ++i) {
          const int r = (lane + 32 * i) / kVec, c = (lane + 32 * i) % kVec;
          uint4 v = qv[i];
          float up = 1.f;
          if (std::is_same<T, __nv_bfloat16>::value) {
            unsigned top = __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu),
                                    __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
#pragma unroll
            for (int o = 1; o < kVec; o <<= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, o));
            const unsigned e = min(max(max(top & 0xffffu, top >> 16) >> 7, 1u), 253u);   // bf16 exponent
            up = __uint_as_float(e << 23);
            const float down = __uint_as_float((254u - e) << 23);
            auto half2_of = [&](unsigned w) {
              return pack2<__half>(__uint_as_float(w << 16) * down, __uint_as_float(w & 0xffff0000u) * down);
            };
            v = make_uint4(half2_of(v.x), half2_of(v.y), half2_of(v.z), half2_of(v.w));
          }
          *reinterpret_cast<uint4*>(sgen + L::kQ + r * L::kQPitch + 16 * c) = v;
          if (c == 0) row_scale[r] = up;
        }
        if (lane == 0) {
          item->x = x; item->b = b; item->chunk_id = chunk_id;
          item->c_begin = c_begin; item->c_end = c_end; item->len = len; item->valid = 1;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(item_full);
        return true;
      };
      // The first item's copies leave before its query rows have arrived; later ones find the ring
      // full of the item before.
      const int publish_at = n_item == 0 ? min(n_stages, L::kStages) - 1 : -1;
      if (publish_at < 0) ok = publish();
      for (int st = 0; ok && st < max(n_stages, 1); ++st) {
        if (p.take_over && st == max(n_stages - 2, 0) && lane == 0) {   // what comes after this item
          mbar_expect_tx(next_full, 16);
          try_cancel_next_cta(sbase + L::kNext, next_full);
          asked = true;
        }
        if (n_stages == 0) break;
        if (st > 0 && (st & 3) == 0) {                                  // the next batch of units
          t_mine += 32 * kUnitKeys;
          page = page_nx; sc = sc_nx;
          page_nx = page_of(t_mine + 32 * kUnitKeys);
        }
        if ((st & 3) == 2) sc_nx = scales_of(t_mine + 32 * kUnitKeys, page_nx);
        const int s = issued % L::kStages;
        const int v0 = c_begin + st * kStageKeys;
        const int unit0 = kUnits * (st & 3);                            // the stage's first unit = its lane
        if (!warp_wait(empty(s), ((issued / L::kStages) & 1) ^ 1)) { ok = false; break; }
        const unsigned there = __ballot_sync(0xffffffffu, page >= 0) >> unit0 & ((1u << kUnits) - 1u);
        if (lane >= unit0 && lane < unit0 + kUnits) {
          unit_scales[s * kUnits + lane - unit0].x = sc.x;
          unit_scales[s * kUnits + lane - unit0].y = sc.y;
        }
        if (lane == 0) unit_mask[s] = there;
        // a lane per copy: its box's first unit's lane
        const int per_box = p.box_keys / kUnitKeys, u = lane - unit0;
        const bool mine = u >= 0 && u < kUnits && u % per_box == 0 && page >= 0;
        const unsigned copies = __popc(__ballot_sync(0xffffffffu, mine));
        __syncwarp();                                                   // (the scales before the arrival)
        if (lane == 0) mbar_expect_tx(full(s), copies * 2 * p.box_keys * DP);
        __syncwarp();
        if (mine) {
          const uint32_t kdst = sbase + s * L::kStageBytes + u * kUnitKeys * DP, vdst = kdst + L::kTileBytes;
          const int r = (v0 + u * kUnitKeys) % p.page_size;
          tma_load_4d(kdst, &tmap_k, full(s), 0, r, hk, page);
          tma_load_4d(vdst, &tmap_v, full(s), 0, r, hk, page);
        }
        __syncwarp();
        ++issued;
        if (st == publish_at) ok = publish();
      }
      // (the answer writes shared memory, so it is waited for whatever happened)
      asked = __shfl_sync(0xffffffffu, asked ? 1 : 0, 0) != 0;
      if (!ok || (p.take_over && !warp_wait(next_full, n_item & 1))) {
        if (asked) mbar_drain(next_full, n_item & 1);
        break;
      }
      if (!p.take_over || !next_cta(sbase + L::kNext, x, b, chunk_id)) {
        if (warp_wait(item_empty, n_item & 1)) {
          if (lane == 0) { item->valid = 0; mbar_arrive(item_full); }
        }
        break;
      }
      __syncwarp();
      fence_proxy_async();     // the answer has been read: the next request may overwrite it
    }
    // A wait gave up somewhere in the CTA: the consumers no longer wait for the stages, so
    // the copies still in flight are waited for here before the CTA may exit.
    if (*abort_flag)
      for (int i = max(issued - L::kStages, 0); i < issued; ++i) mbar_drain(full(i % L::kStages), (i / L::kStages) & 1);
    return;
  }

  // ================================================================== consumers
  const int gid = lane >> 2, tig = lane & 3;
  float* sm_fold = reinterpret_cast<float*>(sgen + L::kFold);
  float* sm_m = reinterpret_cast<float*>(sgen + L::kMl);               // [4][16]
  float* sm_l = sm_m + 4 * 16;
  // the 16-byte piece `c` of row `r` of a tile (64- or 128-byte swizzle of the copy engine)
  auto piece = [](int r, int c) -> uint32_t {
    return r * DP + ((DP == 128 ? c ^ (r & 7) : c ^ ((r >> 1) & 3)) << 4);
  };
  int used = 0;                            // stages read so far, over all items
  for (int n_item = 0;; ++n_item) {
    // (decided by all four warps together, here and below: a warp that left alone after a wait gave
    // up would be missing from the others' barriers)
    const bool got = mbar_wait(item_full, n_item & 1, abort_flag);
    if (consumers_any(!got)) break;
    if (!item->valid) break;
    const int x = item->x, b = item->b, chunk_id = item->chunk_id;
    const int c_begin = item->c_begin, c_end = item->c_end, len = item->len;
    const int n_stages = (c_end - c_begin + kStageKeys - 1) / kStageKeys;
    const int hk = x / p.tiles, row0 = (x - hk * p.tiles) * kRowsTile;
    const int rows_here = min(kRowsTile, p.rows - row0);
    const int query0 = row0 / p.group, query1 = (row0 + rows_here - 1) / p.group;
    unsigned qa[kQJ][4][2 * kNT];          // A operand of step m of piece j: rows gid (and gid + 8)
    float rsc[kNT];                        // what the scores of the lane's rows are multiplied by, but for ks
    int query[kNT], limit[kNT];            // the query of the row, the keys it sees
#pragma unroll
    for (int r = 0; r < kNT; ++r) {
#pragma unroll
      for (int j = 0; j < kQJ; ++j) {
        const uint32_t at = sbase + L::kQ + (gid + 8 * r) * L::kQPitch + 32 * (kQJ * tig + j);
        const uint4 a = lds128(at), c = lds128(at + 16);
        qa[j][0][r] = a.x; qa[j][0][kNT + r] = a.y; qa[j][1][r] = a.z; qa[j][1][kNT + r] = a.w;
        qa[j][2][r] = c.x; qa[j][2][kNT + r] = c.y; qa[j][3][r] = c.z; qa[j][3][kNT + r] = c.w;
      }
      rsc[r] = row_scale[gid + 8 * r] * p.scale_log2;
      query[r] = min(row0 + gid + 8 * r, p.rows - 1) / p.group;
      limit[r] = min(visible(p, len, query[r]), c_end);
    }
    const int limit0 = min(visible(p, len, query0), c_end);   // keys that every row of the tile sees
    __syncwarp();
    if (lane == 0) mbar_arrive(item_empty);
    float acc[kChunks16][kNT][4];
#pragma unroll
    for (int c = 0; c < kChunks16; ++c)
#pragma unroll
      for (int r = 0; r < kNT; ++r) acc[c][r][0] = acc[c][r][1] = acc[c][r][2] = acc[c][r][3] = 0.f;
    float m_run[kNT], l_run[kNT];
#pragma unroll
    for (int r = 0; r < kNT; ++r) { m_run[r] = -INFINITY; l_run[r] = 0.f; }

    for (int st = 0; st < n_stages; ++st, ++used) {
      const int s = used % L::kStages;
      if (!warp_wait(full(s), (used / L::kStages) & 1)) break;   // reported below
      const int v0 = c_begin + st * kStageKeys + kWarpKeys * warp;   // this warp's keys of the stage
      const unsigned there = unit_mask[s] >> (2 * warp) & 3u;
      if (v0 < c_end && there) {
        const uint32_t ktile = sbase + s * L::kStageBytes, vtile = ktile + L::kTileBytes;
        float ks[2], vs[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          ks[u] = unit_scales[s * kUnits + 2 * warp + u].x;
          vs[u] = unit_scales[s * kUnits + 2 * warp + u].y;
        }
        const bool whole = there == 3u && v0 + kWarpKeys <= limit0;   // every row sees every key
        // ---- S[row, key] = Q K^T for four 8-key tiles
        float sc[4][4];
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) {
          sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
#pragma unroll
          for (int j = 0; j < kQJ; ++j) {
            const uint4 k4 = lds128(ktile + piece(kWarpKeys * warp + 8 * nt + gid, kQJ * tig + j));
            const unsigned kw[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
            for (int m = 0; m < 4; ++m) {
              unsigned b0, b1;
              neighbours<kE4M3>(kw[m], b0, b1);
              if (kNT == 2) mma_16816<__half>(sc[nt], qa[j][m][0], qa[j][m][1], qa[j][m][kNT], qa[j][m][kNT + 1], b0, b1);
              else mma_16816<__half>(sc[nt], qa[j][m][0], 0u, qa[j][m][kNT], 0u, b0, b1);
            }
          }
        }
        // the lane's scores: keys 8 nt + 2 tig + {0, 1} of rows gid and gid + 8
        unsigned pb[kNT][4];
        float alpha[kNT];
#pragma unroll
        for (int r = 0; r < kNT; ++r) {
          float x8[8];
#pragma unroll
          for (int nt = 0; nt < 4; ++nt) {
            const float f = ks[nt >> 1] * rsc[r];
            x8[2 * nt] = sc[nt][2 * r] * f;
            x8[2 * nt + 1] = sc[nt][2 * r + 1] * f;
          }
          if (!whole) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int key = v0 + 8 * (i >> 1) + 2 * tig + (i & 1);
              if (key >= limit[r] || !((there >> (i >> 2)) & 1u)) x8[i] = -INFINITY;
            }
          }
          float mx = fmaxf(fmaxf(fmaxf(x8[0], x8[1]), fmaxf(x8[2], x8[3])), fmaxf(fmaxf(x8[4], x8[5]), fmaxf(x8[6], x8[7])));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float m_new = fmaxf(m_run[r], mx);
          const float m_use = (m_new == -INFINITY ? 0.f : m_new) - kPUp;
          alpha[r] = m_run[r] == m_new ? 1.f : exp2f(m_run[r] - kPUp - m_use);
          m_run[r] = m_new;
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) { x8[i] = exp2f(x8[i] - m_use); sum += x8[i]; }
          l_run[r] = l_run[r] * alpha[r] + sum;
#pragma unroll
          for (int i = 0; i < 4; ++i) pb[r][i] = pack2<__half>(x8[2 * i], x8[2 * i + 1]);   // B operand: units 0, 0, 1, 1
        }
        bool moved = alpha[0] != 1.f;
        if (kNT == 2) moved = moved || alpha[kNT - 1] != 1.f;
        if (__any_sync(0xffffffffu, moved)) {
          // (columns of the accumulators are rows 2 tig, 2 tig + 1 of the tile)
#pragma unroll
          for (int r = 0; r < kNT; ++r) {
            const float a0 = __shfl_sync(0xffffffffu, alpha[r], 8 * tig), a1 = __shfl_sync(0xffffffffu, alpha[r], 8 * tig + 4);
#pragma unroll
            for (int c = 0; c < kChunks16; ++c) {
              acc[c][r][0] *= a0; acc[c][r][1] *= a1; acc[c][r][2] *= a0; acc[c][r][3] *= a1;
            }
          }
        }
        // ---- O^T[d, row] += V^T P^T: 16 numbers of d (one piece of the rows) and 16 keys at a time
        const int mi = lane >> 3;
        const int vrow = kWarpKeys * warp + 8 * (mi & 1) + (lane & 7);
        if (whole) {
          const bool one_scale = vs[0] == vs[1];
#pragma unroll
          for (int c = 0; c < kChunks16; c += 2) {
            unsigned w0[4], w1[4];      // [piece c: keys 0-7, 8-15; piece c + 1: ...] of units 0 and 1
            ldmatrix_x4_trans(vtile + piece(vrow, c + (mi >> 1)), w0[0], w0[1], w0[2], w0[3]);
            ldmatrix_x4_trans(vtile + piece(vrow + kUnitKeys, c + (mi >> 1)), w1[0], w1[1], w1[2], w1[3]);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              unsigned a[4], e[4];
              alternates<kE4M3>(w0[2 * h], a[0], a[1]);
              alternates<kE4M3>(w0[2 * h + 1], a[2], a[3]);
              alternates<kE4M3>(w1[2 * h], e[0], e[1]);
              alternates<kE4M3>(w1[2 * h + 1], e[2], e[3]);
#pragma unroll
              for (int r = 0; r < kNT; ++r) {
                float t[4] = {0.f, 0.f, 0.f, 0.f};
                mma_16816<__half>(t, a[0], a[1], a[2], a[3], pb[r][0], pb[r][1]);
                if (!one_scale) {
#pragma unroll
                  for (int i = 0; i < 4; ++i) { acc[c + h][r][i] = fmaf(vs[0], t[i], acc[c + h][r][i]); t[i] = 0.f; }
                }
                mma_16816<__half>(t, e[0], e[1], e[2], e[3], pb[r][2], pb[r][3]);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[c + h][r][i] = fmaf(vs[1], t[i], acc[c + h][r][i]);
              }
            }
          }
        } else {
          // Some key is not there for some row.  What lies in its place may be anything, and 0 times
          // anything need not be 0: V is taken query by query, with what that query does not see cleared.
          int owner[kNT][2];     // the queries of the accumulators' columns
#pragma unroll
          for (int r = 0; r < kNT; ++r)
#pragma unroll
            for (int e = 0; e < 2; ++e) owner[r][e] = __shfl_sync(0xffffffffu, query[r], 8 * tig + 4 * e);
          for (int qi = query0; qi <= query1; ++qi) {
            const int lim = min(visible(p, len, qi), c_end);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const int n_real = lim - (v0 + kUnitKeys * u);
              if (n_real <= 0 || !((there >> u) & 1u)) continue;
              auto pair_mask = [&](int key) { return (key < n_real ? 0xffffu : 0u) | (key + 1 < n_real ? 0xffff0000u : 0u); };
              const unsigned m0 = pair_mask(2 * tig), m1 = pair_mask(2 * tig + 8);
#pragma unroll
              for (int c = 0; c < kChunks16; c += 2) {
                unsigned w[4];
                ldmatrix_x4_trans(vtile + piece(vrow + kUnitKeys * u, c + (mi >> 1)), w[0], w[1], w[2], w[3]);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  unsigned a[4];
                  alternates<kE4M3>(w[2 * h] & m0, a[0], a[1]);
                  alternates<kE4M3>(w[2 * h + 1] & m1, a[2], a[3]);
#pragma unroll
                  for (int r = 0; r < kNT; ++r) {
                    float t[4] = {0.f, 0.f, 0.f, 0.f};
                    const bool own = query[r] == qi;
                    mma_16816<__half>(t, a[0], a[1], a[2], a[3], own ? pb[r][2 * u] : 0u, own ? pb[r][2 * u + 1] : 0u);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                      if (owner[r][i & 1] == qi) acc[c + h][r][i] = fmaf(vs[u], t[i], acc[c + h][r][i]);
                  }
                }
              }
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty(s));
    }

    // ---- fold the four warps' sums, 32 or 64 columns at a time, through a buffer beside the ring
    constexpr int kCols = kRows == 8 ? 64 : 32, kPitch = kCols + 4;
#pragma unroll
    for (int r = 0; r < kNT; ++r) {
      l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 1);
      l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 2);
      if (tig == 0) {
        sm_m[warp * 16 + gid + 8 * r] = m_run[r];
        sm_l[warp * 16 + gid + 8 * r] = l_run[r];
      }
    }
    bool gave_up = false;
#pragma unroll
    for (int rd = 0; rd < DP / kCols; ++rd) {
#pragma unroll
      for (int i = 0; i < kCols / 16; ++i)
#pragma unroll
        for (int r = 0; r < kNT; ++r) {
          const float* a4 = acc[(kCols / 16) * rd + i][r];
          float* at = sm_fold + (warp * kRows + 8 * r + 2 * tig) * kPitch + 16 * i + 2 * gid;
          *reinterpret_cast<float2*>(at) = make_float2(a4[0], a4[2]);
          *reinterpret_cast<float2*>(at + kPitch) = make_float2(a4[1], a4[3]);
        }
      // (a bounded wait gave up: the chunk is reported as empty and the caller is told through the
      // status word)
      gave_up = consumers_any(*abort_flag != 0) || gave_up;
      for (int g = warp; g < rows_here; g += 4) {
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) M = fmaxf(M, sm_m[w * 16 + g]);
        const float Ms = (M == -INFINITY) ? 0.f : M;
        float f[4], Lsum = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          f[w] = exp2f(sm_m[w * 16 + g] - Ms);
          Lsum += sm_l[w * 16 + g] * f[w];
        }
        const bool some = Lsum != 0.f && !gave_up;
        const int row = row0 + g;
        const long long prow = ((long long)(b * p.heads_kv + hk) * p.rows + row) * p.max_chunks + chunk_id;
        T* orow = (T*)p.o + b * p.o_sb + row / p.group * p.o_st + (hk * p.group + row % p.group) * p.o_sh;
#pragma unroll
        for (int cc = 0; cc < kCols; cc += 32) {
          float O = 0.f;
#pragma unroll
          for (int w = 0; w < 4; ++w) O += sm_fold[(w * kRows + g) * kPitch + cc + lane] * f[w];
          const float v = some ? O / Lsum : 0.f;
          const int d = kCols * rd + cc + lane;
          if (d < p.head_dim) {
            if (p.direct_o) orow[d] = from_float<T>(v);
            else p.part_o[prow * p.head_dim + d] = v;
          }
        }
        if (rd == 0 && lane == 0 && !p.direct_o) p.part_lse[prow] = some ? Ms - kPUp + log2f(Lsum) : -INFINITY;
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
    }
    if (gave_up) break;
  }
  if (threadIdx.x == 0 && *abort_flag && p.status_word) atomicExch(p.status_word, 1);
}

// Phase 2: O = sum_c o_c * 2^(lse_c - lse), lse = log2 sum_c 2^lse_c.  Rows without visible keys give 0.
constexpr int kCombineWarps = 4;

template <typename T, int D>
__global__ void __launch_bounds__(32 * kCombineWarps) decode_8bit_combine_kernel(const Decode8Params p) {
  sm100::launch_dependents();
  sm100::grid_dependency_wait();
  constexpr int kLanes = D / 4;                     // lanes that hold 4 columns each
  const int hk = blockIdx.x / p.rows, row = blockIdx.x - hk * p.rows, b = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = visible(p, length_of(p, b), row / p.group);
  const int nchunk = (n + p.chunk - 1) / p.chunk;
  const long long row0 = ((long long)(b * p.heads_kv + hk) * p.rows + row) * p.max_chunks;
  const float* lse = p.part_lse + row0;
  float M = -INFINITY;
  for (int c = lane; c < nchunk; c += 32) M = fmaxf(M, lse[c]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  const float Ms = (M == -INFINITY) ? 0.f : M;
  float L = 0.f;
  for (int c = lane; c < nchunk; c += 32) L += exp2f(lse[c] - Ms);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
  const float inv = L != 0.f ? 1.f / L : 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (lane < kLanes) {
    const float4* rows = reinterpret_cast<const float4*>(p.part_o + row0 * D) + lane;
#pragma unroll 4
    for (int c = warp; c < nchunk; c += kCombineWarps) {
      const float w = exp2f(lse[c] - Ms) * inv;
      const float4 r = rows[(long long)c * kLanes];
      acc.x = fmaf(r.x, w, acc.x); acc.y = fmaf(r.y, w, acc.y);
      acc.z = fmaf(r.z, w, acc.z); acc.w = fmaf(r.w, w, acc.w);
    }
  }
  __shared__ float4 part[kCombineWarps][kLanes];
  if (lane < kLanes) part[warp][lane] = acc;
  __syncthreads();
  const int d = threadIdx.x;
  if (d < D) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kCombineWarps; ++w) s += reinterpret_cast<const float*>(part[w])[d];
    T* orow = (T*)p.o + b * p.o_sb + row / p.group * p.o_st + (hk * p.group + row % p.group) * p.o_sh;
    orow[d] = from_float<T>(s);
  }
}

// ---------------------------------------------------------------------------- host side
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
    if (s % 16 != 0 || s < 0) return B200ATTN_ERR_STRIDE;
  if (a->chunk_tokens < 0 || a->chunk_tokens % kStageKeys != 0) return B200ATTN_ERR_SHAPE;
  return B200ATTN_OK;
}

long long max_visible(const b200attn_paged_decode_8bit_args* a) {
  return std::min<long long>(a->max_seqlen, (long long)a->max_pages_per_seq * a->page_size);
}
long long rows_of(const b200attn_paged_decode_8bit_args* a) {
  return (long long)a->queries * (a->heads_q / a->heads_kv);
}

// Split size.
int chunk_of(const b200attn_paged_decode_8bit_args* a) {
  if (a->chunk_tokens > 0) return a->chunk_tokens;
  const long long units = a->batch * (long long)a->heads_kv * ((rows_of(a) + kRowsTile - 1) / kRowsTile);
  const long long keys = std::max<long long>(max_visible(a), 1);
  if (units >= 256) return 4096;
  const int sizes[8] = {16384, 8192, 4096, 2048, 1024, 512, 256, 128};
  for (int c : sizes)
    if (units * ((keys + c - 1) / c) >= 148) return c;
  return 128;
}
long long chunks_of(const b200attn_paged_decode_8bit_args* a) {
  const long long chunk = chunk_of(a), n = (max_visible(a) + chunk - 1) / chunk;
  return std::max<long long>(n, 1);
}

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return (EncodeFn)f;
  }();
  return fn;
}

// [D, tokens of a page, heads, pages] view of a pool, box = padded D x box_keys (columns past D read 0)
bool pool_map(CUtensorMap* m, const void* base, const b200attn_paged_decode_8bit_args* a, long long st, long long sh,
              long long sp, int dp, int box_keys) {
  EncodeFn enc = encode_fn();
  if (!enc) return false;
  if (a->heads_kv == 1) sh = st;       // (the stride of an axis of one may be anything)
  if (a->num_pages == 1) sp = st;
  cuuint64_t dims[4] = {(cuuint64_t)a->head_dim, (cuuint64_t)a->page_size, (cuuint64_t)a->heads_kv, (cuuint64_t)a->num_pages};
  cuuint64_t strides[3] = {(cuuint64_t)st, (cuuint64_t)sh, (cuuint64_t)sp};
  cuuint32_t box[4] = {(cuuint32_t)dp, (cuuint32_t)box_keys, 1, 1};
  cuuint32_t one[4] = {1, 1, 1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(base), dims, strides, box, one,
             CU_TENSOR_MAP_INTERLEAVE_NONE, dp == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, bool kE4M3, int DP, int kRows>
int launch_split(const b200attn_paged_decode_8bit_args* a, const Decode8Params& p, dim3 grid, cudaStream_t stream) {
  using L = Decode8Smem<DP>;
  auto kernel = decode_8bit_kernel<T, kE4M3, DP, kRows>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kAlloc) != cudaSuccess)
    return B200ATTN_ERR_CUDA;
  CUtensorMap tk, tv;
  if (!pool_map(&tk, a->k_pages, a, a->k_stride_t, a->k_stride_h, a->k_stride_page, DP, p.box_keys) ||
      !pool_map(&tv, a->v_pages, a, a->v_stride_t, a->v_stride_h, a->v_stride_page, DP, p.box_keys))
    return B200ATTN_ERR_CUDA;
  return launch_after(kernel, grid, dim3(160), L::kAlloc, stream, tk, tv, p) == cudaSuccess ? B200ATTN_OK
                                                                                            : B200ATTN_ERR_CUDA;
}
template <typename T, bool kE4M3>
int launch_split(const b200attn_paged_decode_8bit_args* a, const Decode8Params& p, dim3 grid, cudaStream_t stream) {
  if (a->head_dim <= 64)
    return p.rows <= 8 ? launch_split<T, kE4M3, 64, 8>(a, p, grid, stream) : launch_split<T, kE4M3, 64, 16>(a, p, grid, stream);
  return p.rows <= 8 ? launch_split<T, kE4M3, 128, 8>(a, p, grid, stream) : launch_split<T, kE4M3, 128, 16>(a, p, grid, stream);
}
template <typename T>
int launch(const b200attn_paged_decode_8bit_args* a, const Decode8Params& p, dim3 grid, cudaStream_t stream) {
  const int st = a->cache_dtype == B200ATTN_E4M3 ? launch_split<T, true>(a, p, grid, stream)
                                                 : launch_split<T, false>(a, p, grid, stream);
  if (st != B200ATTN_OK || p.direct_o) return st;
  const dim3 rows((unsigned)(p.heads_kv * p.rows), (unsigned)p.batch);
  auto go = [&](auto kernel) { return launch_after(kernel, rows, dim3(32 * kCombineWarps), 0, stream, p); };
  const cudaError_t e = a->head_dim == 32   ? go(decode_8bit_combine_kernel<T, 32>)
                        : a->head_dim == 64 ? go(decode_8bit_combine_kernel<T, 64>)
                        : a->head_dim == 96 ? go(decode_8bit_combine_kernel<T, 96>)
                                            : go(decode_8bit_combine_kernel<T, 128>);
  return e == cudaSuccess ? B200ATTN_OK : B200ATTN_ERR_CUDA;
}

}  // namespace

size_t paged_decode_8bit_workspace_bytes(const b200attn_paged_decode_8bit_args* a) {
  if (!a || a->batch <= 0 || a->queries <= 0 || a->heads_q <= 0 || a->heads_kv <= 0 || a->head_dim <= 0) return 0;
  const long long chunks = chunks_of(a);
  if (chunks == 1) return 16;          // phase 1 writes the result itself
  const size_t rows = (size_t)a->batch * a->queries * a->heads_q * chunks;
  return rows * a->head_dim * 4 + rows * 4;
}

int paged_decode_8bit_fwd(const b200attn_paged_decode_8bit_args* a, cudaStream_t stream) {
  int st = validate(a);
  if (st != B200ATTN_OK) return st;
  const long long rows = rows_of(a), tiles = (rows + kRowsTile - 1) / kRowsTile;
  const long long chunks = chunks_of(a);
  if (a->heads_kv * rows > INT_MAX || chunks > 65535 || max_visible(a) > INT_MAX - 65536) return B200ATTN_ERR_TOO_LARGE;
  if (!a->workspace || a->workspace_bytes < paged_decode_8bit_workspace_bytes(a)) return B200ATTN_ERR_WORKSPACE;
  if ((uintptr_t)a->workspace & 15) return B200ATTN_ERR_ALIGN;
  const DeviceInfo* di = nullptr;
  if ((st = device_info(&di)) != B200ATTN_OK) return st;
  Decode8Params p;
  p.q = a->q; p.ks = a->k_scales; p.vs = a->v_scales; p.o = a->o;
  p.table = a->page_table; p.lens = a->seqlens; p.status_word = a->status_word;
  p.q_sb = a->q_stride_b; p.q_st = a->q_stride_t; p.q_sh = a->q_stride_h;
  p.o_sb = a->o_stride_b; p.o_st = a->o_stride_t; p.o_sh = a->o_stride_h;
  p.ks_sp = a->ks_stride_page; p.ks_sb = a->ks_stride_blk; p.ks_sh = a->ks_stride_h;
  p.vs_sp = a->vs_stride_page; p.vs_sb = a->vs_stride_blk; p.vs_sh = a->vs_stride_h;
  p.batch = a->batch; p.queries = a->queries; p.heads_kv = a->heads_kv;
  p.group = a->heads_q / a->heads_kv; p.head_dim = a->head_dim;
  p.rows = (int)rows; p.tiles = (int)tiles;
  p.page_size = a->page_size; p.block = a->block_tokens; p.num_pages = a->num_pages; p.width = a->max_pages_per_seq;
  p.max_len = (int)max_visible(a);
  p.box_keys = std::min(a->page_size & -a->page_size, kStageKeys);
  p.chunk = chunk_of(a); p.max_chunks = (int)chunks;
  p.direct_o = chunks == 1;
  p.take_over = a->heads_kv * tiles * a->batch * chunks > 2LL * di->sm_count;
  p.scale_log2 = a->softmax_scale * 1.4426950408889634f;
  p.part_o = (float*)a->workspace;
  p.part_lse = p.part_o + (size_t)a->batch * a->queries * a->heads_q * chunks * a->head_dim;
  const dim3 grid((unsigned)(a->heads_kv * tiles), (unsigned)a->batch, (unsigned)chunks);
  st = a->dtype == B200ATTN_F16 ? launch<__half>(a, p, grid, stream) : launch<__nv_bfloat16>(a, p, grid, stream);
  if (st != B200ATTN_OK) return st;
  set_launch_count(p.direct_o ? 1 : 2);
  return cudaGetLastError() == cudaSuccess ? B200ATTN_OK : B200ATTN_ERR_CUDA;
}

}  // namespace b200attn
