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
// Measured on B200, 8 KV heads of 128, one token: 64 sequences of 4096 keys 90 us, 0.92 of a copy; 64 of 1024
// to 8192 118 us, 0.80 (the end of an uneven batch); four of 90001 to 131072, int8, scales of 16 keys, 171 us,
// 0.85.  Up to 8 query rows the memory bounds it.  With 16 the warps' own chain does (43 % of the issue slots,
// two warps a scheduler, 168 registers): 32 sequences of 4096 keys take 87 us against 42 us for their bytes,
// and more rows take another pass (20 rows: 140 us).  24 rows at once with Q in shared memory spilled: 174 us.
// The products take 16-bit operands, and of the types fp16 holds the cached numbers exactly, so the other
// operand is rounded to its 11 bits too (the rest of either would be a second product for each):
//   * Q: fp16 rows as they are; bf16 rows (8 bits) times a power of two per row, exact but for what lies below
//     2^-14 of the row's largest element, which is rounded to 2^-25 of that.
//   * P, 2^10 times the weight, which keeps weights down to 2^-24 of the largest one out of fp16's
//     subnormals: relative 2^-11 of a weight; the sum of weights is of the unrounded ones, in fp32.  The
//     outputs' relative error against 64 bits is 2.1e-4 (fp16, 333 keys) and 2.2e-4 (20 rows of drafts), where
//     32-bit arithmetic has 2.0e-4 and 2.1e-4; 1.7e-3 either way for bf16 outputs, whose own rounding that is.
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

// CTAs per SM: 192 KB are in flight either way.  With heads of up to 64 and up to 8 rows the copies' issue and the
// warps' chains bound, of which three CTAs have more under way: 64 sequences of 4096 keys, D = 64, 107 us -> 81 in
// pages of 16 keys, 67 -> 60 in pages of 64; two of 60000, 62 -> 49 and 43 -> 40; 128 of 100 to 2000, 68 -> 66 and
// 44 -> 47.  The registers that three leave are few for 16 rows (D = 64: 20 rows, 24 sequences of 300 to 6000, 81 us ->
// 92; D = 128: 32 of 4096, 87 -> 118), and with D = 128 two stages are few for the memory (92 -> 104 with one row).
__host__ __device__ constexpr int ctas_per_sm(int head_dim, int rows) { return head_dim <= 64 && rows <= 8 ? 3 : 2; }

// n / d for 0 <= n < 2^31 by a multiplication (a division by a run-time number takes the producer
// warp longer than the copy it prepares)
struct Divisor {
  unsigned mul;
  int shift, d;
  __device__ __forceinline__ int quotient(int n) const { return (int)(((unsigned long long)(unsigned)n * mul) >> shift); }
  __device__ __forceinline__ int remainder(int n) const { return n - quotient(n) * d; }
};
Divisor divisor(int d) {      // mul = ceil(2^shift / d) < 2^32, exact for n < 2^31 as 2^31 * (mul * d - 2^shift) <= 2^shift
  int bits = 0;
  while ((1LL << bits) < d) ++bits;
  return {(unsigned)(((1ULL << (31 + bits)) + d - 1) / d), 31 + bits, d};
}

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
  Divisor by_page, by_group, by_tiles;
  int block_shift, num_pages, width, max_len;
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

constexpr int kConsumers = kStageKeys / kWarpKeys;   // warps
constexpr int kDecode8Threads = 32 * kConsumers + 32;

template <int DP, int kRows>
struct Decode8Smem {
  static constexpr int kTileBytes = kStageKeys * DP;       // K or V of one stage
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kStages = 192 * 1024 / ctas_per_sm(DP, kRows) / kStageBytes;
  static constexpr int kQ = kStages * kStageBytes;         // the item's 16 query rows, fp16
  static constexpr int kQPitch = DP * 2 + 16;              // bytes
  static constexpr int kMl = kQ + kRowsTile * kQPitch;     // row max and sum, [2][warps][16]
  static constexpr int kRowScale = kMl + 2 * kConsumers * 16 * 4;   // [16] what the query rows were divided by
  static constexpr int kScales = kRowScale + 64;           // [stage][unit] (ks, vs)
  static constexpr int kMask = kScales + kStages * kUnits * 8;   // [stage] units whose page is in the pool
  static constexpr int kItem = kMask + 32;
  static constexpr int kNext = kItem + 32;                 // response of the launch control (16 bytes)
  static constexpr int kBarOffset = kNext + 16;
  static constexpr int kBytes = kBarOffset + (2 * kStages + 3) * 8 + 16;
  static constexpr int kAlloc = kBytes + 1024;
  static_assert(kScales % 8 == 0 && kNext % 16 == 0 && kBarOffset % 8 == 0, "aligned");
  static_assert(kStageBytes == kConsumers * 16 * DP * 4, "the warps' sums of 16 rows fold in the buffer of a stage");
  static_assert(ctas_per_sm(DP, kRows) * (kAlloc + 1024) <= 228 * 1024, "resident together");
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
__global__ void __launch_bounds__(kDecode8Threads, ctas_per_sm(DP, kRows))
decode_8bit_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                   const Decode8Params p) {
  using L = Decode8Smem<DP, kRows>;
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
    for (int s = 0; s < L::kStages; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), kConsumers); }
    mbar_init(item_full, 1);
    mbar_init(item_empty, kConsumers);
    mbar_init(next_full, 1);
    fence_barrier_init();
    fence_proxy_async();
  }
  if (threadIdx.x == 32 * kConsumers) { prefetch_tmap(&tmap_k); prefetch_tmap(&tmap_v); }
  grid_dependency_wait();
  __syncthreads();

  // A wait by a whole warp, answered alike in all of its lanes.
  auto warp_wait = [&](uint32_t bar, uint32_t parity) -> bool {
    const bool done = mbar_wait(bar, parity, abort_flag);
    return __all_sync(0xffffffffu, done);
  };
  if (warp == kConsumers) {
    // ================================================================ producer
    // Everything small that a copy needs is asked for long before it: behind full rings (192 KB
    // per SM) a load takes as long as those bytes take to arrive, 3 to 4 us.  So nothing below
    // computes with a loaded value until stages later: a batch of units' page-table entries are asked
    // for two batches ahead and its scales one, the next item while this one's last eight stages leave.
    constexpr int kVec = DP / 8;        // 16-byte pieces of a query row
    constexpr int kQRows = 8 * kNT;
    constexpr int kBatch = 32 * kUnitKeys;   // keys of a batch of units, one per lane: four stages
    struct Head {
      int x, b, chunk_id;
      int len;                          // as it stands in memory
      int entry, entry_nx;              // page-table entries of the lane's units of the first two batches
      float2 sc;                        // scales of its unit of the first one
      uint4 q[kQRows * kVec / 32];
    };
    auto fetch = [&](Head& h) {
      const int32_t* pages = p.table + (long long)h.b * p.width;
      const int t = h.chunk_id * p.chunk + kUnitKeys * lane;      // (the row has an entry there, if perhaps not a page)
      h.entry = h.entry_nx = -1;
      if (t < p.max_len) h.entry = pages[p.by_page.quotient(t)];
      if (t + kBatch < p.max_len) h.entry_nx = pages[p.by_page.quotient(t + kBatch)];
      h.len = p.lens[h.b];
      const int hk = p.by_tiles.quotient(h.x), row0 = p.by_tiles.remainder(h.x) * kRowsTile;
#pragma unroll
      for (int i = 0; i < kQRows * kVec / 32; ++i) {
        const int r = row0 + (lane + 32 * i) / kVec, c = (lane + 32 * i) % kVec;
        h.q[i] = make_uint4(0, 0, 0, 0);
        if (r < p.rows && 8 * c < p.head_dim)
          h.q[i] = *reinterpret_cast<const uint4*>((const T*)p.q + h.b * p.q_sb + p.by_group.quotient(r) * p.q_st +
                                                   (hk * p.group + p.by_group.remainder(r)) * p.q_sh + 8 * c);
      }
    };
    // scales of the unit at key t, whose page-table entry is e (whether or not the sequence has that key)
    auto scales_of = [&](int hk, int t, int e) -> float2 {
      float2 r = make_float2(0.f, 0.f);
      if (e >= 0 && e < p.num_pages) {
        const int blk = p.by_page.remainder(t) >> p.block_shift;
        r.x = p.ks[e * p.ks_sp + blk * p.ks_sb + hk * p.ks_sh];
        r.y = p.vs[e * p.vs_sp + blk * p.vs_sb + hk * p.vs_sh];
      }
      return r;
    };
    auto first_scales = [&](Head& h) {
      h.sc = scales_of(p.by_tiles.quotient(h.x), h.chunk_id * p.chunk + kUnitKeys * lane, h.entry);
    };
    int issued = 0;                       // stages sent so far, over all items
    bool ok = true;
    Head head;
    head.x = blockIdx.x; head.b = blockIdx.y; head.chunk_id = blockIdx.z;
    fetch(head);
    first_scales(head);
    for (int n_item = 0; ok; ++n_item) {
      bool asked = false, known = !p.take_over, more = false, scaled = !p.take_over;   // of the next item
      Head next;
      const int hk = p.by_tiles.quotient(head.x), row0 = p.by_tiles.remainder(head.x) * kRowsTile;
      const int len = min(max(head.len, 0), p.max_len);
      const int n_vis = visible(p, len, p.by_group.quotient(min(row0 + kRowsTile, p.rows) - 1));
      const int c_begin = min(head.chunk_id * p.chunk, n_vis);
      const int c_end = c_begin + min(n_vis - c_begin, p.chunk);
      const int n_stages = (c_end - c_begin + kStageKeys - 1) / kStageKeys;
      const int ask_at = max(n_stages - 8, 0), fetch_at = max(n_stages - 5, 1), scales_at = max(n_stages - 2, 2);
      // lane i looks after unit i of four stages
      const int32_t* pages = p.table + (long long)head.b * p.width;
      int t_mine = head.chunk_id * p.chunk + kUnitKeys * lane;
      int entry = head.entry, entry_nx = head.entry_nx, entry_nx2 = -1, page = -1, row_mine = 0;
      float2 sc = make_float2(0.f, 0.f), sc_nx = head.sc;
      auto publish = [&]() -> bool {
        if (!warp_wait(item_empty, (n_item & 1) ^ 1)) return false;
        // (bf16 rows are divided by a power of two so that fp16 holds them)
#pragma unroll
        for (int i = 0; i < kQRows * kVec / 32; ++i) {
          const int r = (lane + 32 * i) / kVec, c = (lane + 32 * i) % kVec;
          uint4 v = head.q[i];
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
          item->x = head.x; item->b = head.b; item->chunk_id = head.chunk_id;
          item->c_begin = c_begin; item->c_end = c_end; item->len = len; item->valid = 1;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(item_full);
        return true;
      };
      // the item that comes after this one, and its loads
      auto look_ahead = [&]() -> bool {
        if (!warp_wait(next_full, n_item & 1)) return false;
        known = true;
        more = next_cta(sbase + L::kNext, next.x, next.b, next.chunk_id);
        __syncwarp();
        fence_proxy_async();     // the answer has been read: the next request may overwrite it
        if (more) fetch(next);
        else scaled = true;
        return true;
      };
      // The first item's copies leave before its query rows have arrived; later items have the
      // consumers at work on the one before.
      const int publish_at = n_item == 0 ? min(n_stages, L::kStages) - 1 : min(n_stages, 1) - 1;
      if (publish_at < 0) ok = publish();
      for (int st = 0; ok && st < max(n_stages, 1); ++st) {
        if (p.take_over && st == ask_at && lane == 0) {                 // what comes after this item
          mbar_expect_tx(next_full, 16);
          try_cancel_next_cta(sbase + L::kNext, next_full);
          asked = true;
        }
        if (n_stages == 0) break;
        if ((st & 3) == 0) {                                            // the next batch of units
          if (st > 0) { t_mine += kBatch; entry = entry_nx; entry_nx = entry_nx2; }
          sc = sc_nx;
          page = t_mine < c_end && entry >= 0 && entry < p.num_pages ? entry : -1;
          row_mine = p.by_page.remainder(t_mine);
          entry_nx2 = -1;
          if (t_mine + 2 * kBatch < c_end) entry_nx2 = pages[p.by_page.quotient(t_mine + 2 * kBatch)];
          sc_nx = make_float2(0.f, 0.f);
          if (t_mine + kBatch < c_end) sc_nx = scales_of(hk, t_mine + kBatch, entry_nx);
        }
        const int s = issued % L::kStages;
        const int unit0 = kUnits * (st & 3);                            // the stage's first unit = its lane
        const unsigned there = __ballot_sync(0xffffffffu, page >= 0) >> unit0 & ((1u << kUnits) - 1u);
        if (!warp_wait(empty(s), ((issued / L::kStages) & 1) ^ 1)) { ok = false; break; }
        if (lane >= unit0 && lane < unit0 + kUnits) {
          unit_scales[s * kUnits + lane - unit0].x = sc.x;
          unit_scales[s * kUnits + lane - unit0].y = sc.y;
        }
        __syncwarp();                                                   // (the scales before the arrival)
        // One lane issues, from registers that hold every box: copies of several lanes go out one by one
        // all the same, and a shuffle between two copies costs as much as a copy.
        auto copy_stage = [&](auto units) {
          constexpr int kPer = decltype(units)::value, kBoxes = kUnits / kPer;
          int pg[kBoxes], row[kBoxes], n = 0;
#pragma unroll
          for (int i = 0; i < kBoxes; ++i) {
            pg[i] = __shfl_sync(0xffffffffu, page, unit0 + i * kPer);
            row[i] = __shfl_sync(0xffffffffu, row_mine, unit0 + i * kPer);
            n += pg[i] >= 0;
          }
          if (lane == 0) {
            unit_mask[s] = there;
            mbar_expect_tx(full(s), n * 2 * kPer * kUnitKeys * DP);
            const uint32_t kdst = sbase + s * L::kStageBytes, vdst = kdst + L::kTileBytes;
#pragma unroll
            for (int i = 0; i < kBoxes; ++i)
              if (pg[i] >= 0) {
                tma_load_4d(kdst + i * kPer * kUnitKeys * DP, &tmap_k, full(s), 0, row[i], hk, pg[i]);
                tma_load_4d(vdst + i * kPer * kUnitKeys * DP, &tmap_v, full(s), 0, row[i], hk, pg[i]);
              }
          }
        };
        switch (p.box_keys) {
          case 16: copy_stage(std::integral_constant<int, 1>()); break;
          case 32: copy_stage(std::integral_constant<int, 2>()); break;
          case 64: copy_stage(std::integral_constant<int, 4>()); break;
          default: copy_stage(std::integral_constant<int, 8>()); break;
        }
        __syncwarp();
        ++issued;
        if (st == publish_at) ok = publish();
        if (ok && !known && st >= fetch_at) ok = look_ahead();
        else if (known && !scaled && st >= scales_at) { first_scales(next); scaled = true; }
      }
      if (ok && !known) ok = look_ahead();
      if (ok && !scaled) first_scales(next);
      // (the answer writes shared memory, so it is waited for whatever happened)
      asked = __shfl_sync(0xffffffffu, asked ? 1 : 0, 0) != 0;
      if (!ok) {
        if (asked) mbar_drain(next_full, n_item & 1);
        break;
      }
      if (!more) {
        if (warp_wait(item_empty, n_item & 1)) {
          if (lane == 0) { item->valid = 0; mbar_arrive(item_full); }
        }
        break;
      }
      head = next;
    }
    // A wait gave up somewhere in the CTA: the consumers no longer wait for the stages, so
    // the copies still in flight are waited for here before the CTA may exit.
    if (*abort_flag)
      for (int i = max(issued - L::kStages, 0); i < issued; ++i) mbar_drain(full(i % L::kStages), (i / L::kStages) & 1);
    return;
  }

  // ================================================================== consumers
  const int gid = lane >> 2, tig = lane & 3;
  float* sm_m = reinterpret_cast<float*>(sgen + L::kMl);               // [warps][16]
  float* sm_l = sm_m + kConsumers * 16;
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
    const int hk = p.by_tiles.quotient(x), row0 = p.by_tiles.remainder(x) * kRowsTile;
    const int rows_here = min(kRowsTile, p.rows - row0);
    const int query0 = p.by_group.quotient(row0), query1 = p.by_group.quotient(row0 + rows_here - 1);
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
      query[r] = p.by_group.quotient(min(row0 + gid + 8 * r, p.rows - 1));
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
        for (int nt = 0; nt < 4; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
#pragma unroll
        for (int j = 0; j < kQJ; ++j) {
          uint4 k4[4];
#pragma unroll
          for (int nt = 0; nt < 4; ++nt) k4[nt] = lds128(ktile + piece(kWarpKeys * warp + 8 * nt + gid, kQJ * tig + j));
#pragma unroll
          for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) {     // (four sums at a time: each waits for its own last product)
              unsigned b0, b1;
              neighbours<kE4M3>(m == 0 ? k4[nt].x : m == 1 ? k4[nt].y : m == 2 ? k4[nt].z : k4[nt].w, b0, b1);
              if (kNT == 2) mma_16816<__half>(sc[nt], qa[j][m][0], qa[j][m][1], qa[j][m][kNT], qa[j][m][kNT + 1], b0, b1);
              else mma_16816<__half>(sc[nt], qa[j][m][0], 0u, qa[j][m][kNT], 0u, b0, b1);
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
      if (lane == 0 && st + 1 < n_stages) mbar_arrive(empty(s));
    }

    // ---- fold the warps' sums in the buffer of the item's last stage, which is given back only then
    // (the producer is filling the others for the next item)
#pragma unroll
    for (int r = 0; r < kNT; ++r) {
      l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 1);
      l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 2);
      if (tig == 0) {
        sm_m[warp * 16 + gid + 8 * r] = m_run[r];
        sm_l[warp * 16 + gid + 8 * r] = l_run[r];
      }
    }
    const int last = (used + L::kStages - 1) % L::kStages;
    float* sm_fold = reinterpret_cast<float*>(sgen + last * L::kStageBytes);   // [warps][rows][DP]
    // (a bounded wait gave up: the chunk is reported as empty and the caller is told through the status word)
    const bool gave_up = consumers_any(*abort_flag != 0);        // (and everyone has read the stage)
    const bool sums = n_stages > 0 && !gave_up;
    if (sums) {
      // the columns of rows 2 tig and 2 tig + 1 are moved by 8 tig, so that a store's four row pairs
      // lie in banks of their own
#pragma unroll
      for (int c = 0; c < kChunks16; ++c)
#pragma unroll
        for (int r = 0; r < kNT; ++r) {
          float* at = sm_fold + (warp * kRows + 8 * r + 2 * tig) * DP + ((16 * c + 2 * gid) ^ (8 * tig));
          *reinterpret_cast<float2*>(at) = make_float2(acc[c][r][0], acc[c][r][2]);
          *reinterpret_cast<float2*>(at + DP) = make_float2(acc[c][r][1], acc[c][r][3]);
        }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(32 * kConsumers) : "memory");
    // a thread takes four columns of a row
    constexpr int kLanes = DP / 4;
    for (int i = threadIdx.x; i < rows_here * kLanes; i += 32 * kConsumers) {
      const int g = i / kLanes, d = 4 * (i % kLanes);
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < kConsumers; ++w) M = fmaxf(M, sm_m[w * 16 + g]);
      const float Ms = (M == -INFINITY) ? 0.f : M;
      float Lsum = 0.f;
      float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kConsumers; ++w) {
        const float f = exp2f(sm_m[w * 16 + g] - Ms);
        Lsum += sm_l[w * 16 + g] * f;
        if (sums) {
          const float4 v = *reinterpret_cast<const float4*>(sm_fold + (w * kRows + g) * DP + (d ^ (8 * ((g & 7) >> 1))));
          O.x += v.x * f; O.y += v.y * f; O.z += v.z * f; O.w += v.w * f;
        }
      }
      const bool some = Lsum != 0.f && sums;
      O = some ? make_float4(O.x / Lsum, O.y / Lsum, O.z / Lsum, O.w / Lsum) : make_float4(0.f, 0.f, 0.f, 0.f);
      const int row = row0 + g;
      const long long prow = ((long long)(b * p.heads_kv + hk) * p.rows + row) * p.max_chunks + chunk_id;
      if (d < p.head_dim) {
        if (p.direct_o) {
          T* at = (T*)p.o + b * p.o_sb + p.by_group.quotient(row) * p.o_st +
                  (hk * p.group + p.by_group.remainder(row)) * p.o_sh + d;
          at[0] = from_float<T>(O.x); at[1] = from_float<T>(O.y);
          at[2] = from_float<T>(O.z); at[3] = from_float<T>(O.w);
        } else {
          *reinterpret_cast<float4*>(p.part_o + prow * p.head_dim + d) = O;
        }
      }
      if (d == 0 && !p.direct_o) p.part_lse[prow] = some ? Ms - kPUp + log2f(Lsum) : -INFINITY;
    }
    if (gave_up) break;
    fence_proxy_async();       // the plain accesses to the stage come before the copy engine's next write
    __syncwarp();
    if (lane == 0 && n_stages > 0) mbar_arrive(empty(last));
  }
  if (threadIdx.x == 0 && *abort_flag && p.status_word) atomicExch(p.status_word, 1);
}

// Phase 2: O = sum_c o_c * 2^(lse_c - lse), lse = log2 sum_c 2^lse_c.  Rows without visible keys give 0.
constexpr int kCombineWarps = 4;

template <typename T, int D>
__global__ void __launch_bounds__(32 * kCombineWarps) decode_8bit_combine_kernel(const Decode8Params p) {
  // (no kernel may start before this one ends: one that has started keeps what it has read of the partial
  // sums' memory, which the next call writes again)
  sm100::grid_dependency_wait();
  constexpr int kLanes = D / 4;                     // lanes that hold 4 columns each
  const int hk = blockIdx.x / p.rows, row = blockIdx.x - hk * p.rows, b = blockIdx.y;
  const int query = p.by_group.quotient(row), head = p.by_group.remainder(row);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = visible(p, length_of(p, b), query);
  const int nchunk = n > 0 ? (n - 1) / p.chunk + 1 : 0;
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
    T* orow = (T*)p.o + b * p.o_sb + query * p.o_st + (hk * p.group + head) * p.o_sh;
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
  if (((uintptr_t)a->o & 1) || !aligned4({a->k_scales, a->v_scales, a->page_table, a->seqlens, a->status_word}))
    return B200ATTN_ERR_ALIGN;
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

// Split size: the one with the least waves x (stages of a chunk + 4) + half a chunk + 4 where there is
// more than one chunk, all lengths taken as the largest.  Four stages are a chunk's own cost (look-ups
// behind a full ring, the fold), half a chunk the uneven end of a ragged batch, four the second kernel
// and its launch.
// Measured on B200, 8 KV heads, D = 128, us: 64 sequences of 4096 keys 90.5 in one chunk, 96 in 1024; of
// 1024-8192 118.7 in 2048, 125 in 1024, 132 in one; 16 of 1024-8192 47.3 in 2048, 44.0 in 1536, 49.6 in
// 4096; 12 of 4096 26.0 in 1536, 28.6 in 2048; 8 of 2048 13.5 in 512, 15.3 in 768; four of 90001-131072
// 156.6 in 2048, 151 in 4096, 182 in 8192; one of 8192 10.9 in 256, 13.4 in 128.
int chunk_of(const b200attn_paged_decode_8bit_args* a) {
  if (a->chunk_tokens > 0) return a->chunk_tokens;
  const long long units = a->batch * (long long)a->heads_kv * ((rows_of(a) + kRowsTile - 1) / kRowsTile);
  const long long stages = std::max<long long>((max_visible(a) + kStageKeys - 1) / kStageKeys, 1);
  // (148: the chip's SMs.  The workspace follows from the split and can be asked for without a device.)
  const long long slots = 148 * ctas_per_sm(a->head_dim, (int)std::min<long long>(rows_of(a), kRowsTile));
  long long best = 0, least = 0;
  auto consider = [&](long long per) {
    const long long n = (stages + per - 1) / per;
    const long long cost = 2 * ((units * n + slots - 1) / slots) * (per + 4) + per + (n > 1 ? 8 : 0);
    if (!best || cost < least) { best = per; least = cost; }
  };
  const int sizes[10] = {1, 2, 3, 4, 6, 8, 12, 16, 32, 64};
  for (int per : sizes)
    if (per < stages) consider(per);
  if (stages <= 64 || !best) consider(stages);
  return (int)(best * kStageKeys);
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
  using L = Decode8Smem<DP, kRows>;
  auto kernel = decode_8bit_kernel<T, kE4M3, DP, kRows>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kAlloc) != cudaSuccess)
    return B200ATTN_ERR_CUDA;
  CUtensorMap tk, tv;
  if (!pool_map(&tk, a->k_pages, a, a->k_stride_t, a->k_stride_h, a->k_stride_page, DP, p.box_keys) ||
      !pool_map(&tv, a->v_pages, a, a->v_stride_t, a->v_stride_h, a->v_stride_page, DP, p.box_keys))
    return B200ATTN_ERR_CUDA;
  return launch_after(kernel, grid, dim3(kDecode8Threads), L::kAlloc, stream, tk, tv, p) == cudaSuccess ? B200ATTN_OK
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
  if (chunks == 1) return 0;           // phase 1 writes the result itself
  const size_t rows = (size_t)a->batch * a->queries * a->heads_q * chunks;
  return rows * a->head_dim * 4 + rows * 4;
}

int paged_decode_8bit_fwd(const b200attn_paged_decode_8bit_args* a, cudaStream_t stream) {
  int st = validate(a);
  if (st != B200ATTN_OK) return st;
  const long long rows = rows_of(a), tiles = (rows + kRowsTile - 1) / kRowsTile;
  const long long chunks = chunks_of(a);
  if (a->heads_kv * rows > INT_MAX || chunks > 65535 || max_visible(a) > INT_MAX - 65536) return B200ATTN_ERR_TOO_LARGE;
  if (const size_t need = paged_decode_8bit_workspace_bytes(a))
    if (!a->workspace || a->workspace_bytes < need) return B200ATTN_ERR_WORKSPACE;
  if ((uintptr_t)a->workspace & 15) return B200ATTN_ERR_ALIGN;
  auto meets = [](long long extent, long long stride) { return extent > 1 && stride == 0; };
  if (meets(a->num_pages, a->k_stride_page) || meets(a->num_pages, a->v_stride_page) || meets(a->page_size, a->k_stride_t) ||
      meets(a->page_size, a->v_stride_t) || meets(a->heads_kv, a->k_stride_h) || meets(a->heads_kv, a->v_stride_h))
    return B200ATTN_ERR_STRIDE;
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
  p.by_page = divisor(a->page_size); p.by_group = divisor(p.group); p.by_tiles = divisor((int)tiles);
  p.block_shift = a->block_tokens == 16 ? 4 : a->block_tokens == 32 ? 5 : a->block_tokens == 64 ? 6 : 7;
  p.num_pages = a->num_pages; p.width = a->max_pages_per_seq;
  p.max_len = (int)max_visible(a);
  p.box_keys = std::min(a->page_size & -a->page_size, kStageKeys);
  p.chunk = chunk_of(a); p.max_chunks = (int)chunks;
  p.direct_o = chunks == 1;
  p.take_over = a->heads_kv * tiles * a->batch * chunks > (long long)ctas_per_sm(a->head_dim, p.rows) * di->sm_count;
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
