// paged_attention_tc.cu — attention over a paged cache for chunks of many new tokens, on tcgen05.
//
// A chunk's rows times the cached keys are two matrix products of 2 head_dim operations a pair each, with a softmax between: the
// tensor cores bound it, and the exponentials come close behind (16 of them a cycle and SM against 128 x 128 x 128 products in
// 512 cycles).  A CTA owns 256 (token, head of the group) rows of one key head in two tiles of 128 and walks the keys in tiles of
// 128, so that one tile's softmax runs while the tensor cores work on the other:
//   warps 0-3, 4-7   softmax of row tile 0 and 1: a thread has a row, reads its 128 scores from tensor memory and writes the probabilities
//                    back over them as 16-bit pairs, from where P V reads them (A operand in tensor memory)
//   warp 8           issues the tensor instructions: per key tile P_0 V, Q_0 K', P_1 V, Q_1 K' (K' the next tile)
//   warps 9-11       bring K and V tiles out of the pages into a ring: by TMA, a box of a page's slots a lane (copies a thread each took 6300
//                    cycles a key tile, twice what everything else did); 8-bit codes through the registers of seven warps, as halves
// Heads of over 128 elements have one tile of 128 rows (O takes 256 columns of tensor memory) and two score tiles that alternate.  So have
// queries of fp32, which are two halves a value (22 bits) and whose probabilities are, over all 128 columns of the scores.  For them O holds the
// products of two key tiles only, and what these come to is added in fp32 to a sum in the rest of tensor memory: the tensor core's accumulation
// truncates, which over 16 K keys came to 2.3e-4 of rows whose probability was on the first 64.
// K and V tiles lie in the same layout, [64 elements][key] rows of 128 swizzled bytes: K-major for Q K^T, MN-major for P V.
// The running maximum is raised only when a score outgrows it by 2^8, so O in tensor memory is rescaled a few times a row.
// Probabilities of a bfloat16 cache are rounded to bfloat16 (8 bits, relative to each probability), else to half (11 bits); their sum is
// of the unrounded ones, in fp32.  Scores, maxima, sums and O are fp32.
// Four chunks of 1.6 to 2 K tokens behind up to 8 K keys, 32 heads of 128 over 8 key heads, bfloat16: 606 us, 1.19 PFLOP/s; the products alone 465.
#include <cmath>
#include <type_traits>

#include "common.h"
#include "launch.cuh"
#include "paged.cuh"
#include "paged_attention.cuh"
#include "sm100_ptx.cuh"

namespace mb {
namespace {

constexpr int TC_TMEM = 512;
constexpr int TC_POLY = 6;  // of eight exponentials the last two go to the FMA lanes (none: 2 % more time, of four the last two: 9 %)

template <int DP, int CT, int NQ>  // NQ: terms of a query and of a probability
struct TcShape {
  static constexpr bool BF = CT == MIMIR_B200_T_BF16, CODED = CT == MIMIR_B200_T_I8 || CT == MIMIR_B200_T_E4M3;
  static constexpr int NT = DP <= 128 && NQ == 1 ? 2 : 1;  // row tiles
  static constexpr int SUB = DP / 64;                  // 64-element columns of a tile
  static constexpr int TILE = SUB * TC_KEYS * 128;     // bytes of a K or V tile, and of a Q tile
  static constexpr int NS = DP == 64 ? 6 : DP == 128 ? 4 : 2;
  static constexpr int SCALES = CODED ? NS / 2 * 2 * TC_KEYS * 4 : 0;  // [V stage][key, value][key]
  // fp32 results: key tiles whose products the tensor core adds up, truncating; what they come to is added to a sum beside them, rounded.  Four
  // chunks of 1.6 to 2 K tokens behind up to 8 K keys of half, heads of 128: 1078 us without, 1124 by two (1175 by one, 1083 by four); heads of 64
  // over e4m3 1350 and 1487.
  static constexpr int GROUP = NQ == 2 ? 2 : 0;
  static_assert((GROUP & (GROUP - 1)) == 0 && (GROUP == 0 || 2 * TC_KEYS + 2 * DP <= TC_TMEM), "tensor memory");
  static constexpr int OFFS = 2 * TC_KEYS * 8;         // where the rows of a key tile lie, two tiles
  static constexpr int SMEM = NT * NQ * TILE + NS * TILE + SCALES + OFFS + 512;
  // halves: probabilities of up to 2^6, by the maximum that may be 2^8 too low 2^14, are exact to 2^-31 of the largest where 2^-25 would be
  static constexpr float ROOM = BF ? 0.0f : 6.0f;
  static constexpr int LOADERS = CODED ? 224 : 96;     // threads that bring tiles
  static constexpr int THREADS = NT * 128 + 32 + LOADERS;
  // 8-bit codes take seven loader warps, which leave registers to the softmax warps: the shares add up to the launch's
  static constexpr int SOFT_REGS = NT == 2 ? 168 : 232, LOAD_REGS = NT == 2 ? 88 : 136, LAUNCH_REGS = NT == 2 ? 128 : 168;
  static_assert(!CODED || NT * 128 * SOFT_REGS + 256 * LOAD_REGS == THREADS * LAUNCH_REGS, "register shares");
};

// (not a number where one of them is: it decides which exponentials a tile gets)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// (64 elements, slots, head, page)
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}

// pairs of fp32 in one instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
// 2^x on the FMA lanes, for x of at most 127 (below -126: 2^-126): x = n + f, |f| <= 1/2, and the polynomial of fourth degree in f whose
// largest relative error is least (2.6e-6, by Remez' exchange); n goes into the exponent.  A share of the exponentials done so leaves the
// special-function lanes, 16 a cycle and SM, less to do.  What is not a number may come out as one: callers do without it then.
__device__ __forceinline__ float2 exp2_poly(float2 x) {
  x = make_float2(fmaxf(x.x, -126.0f), fmaxf(x.y, -126.0f));
  const float2 m = add2(x, make_float2(12582912.0f, 12582912.0f));  // 1.5 * 2^23: n in the low bits
  const float2 n = add2(m, make_float2(-12582912.0f, -12582912.0f));
  const float2 f = fma2(n, make_float2(-1.0f, -1.0f), x);
  float2 p = fma2(f, make_float2(9.5701021e-3f, 9.5701021e-3f), make_float2(5.5917859e-2f, 5.5917859e-2f));
  p = fma2(p, f, make_float2(0.24024744f, 0.24024744f));
  p = fma2(p, f, make_float2(0.69312179f, 0.69312179f));
  p = fma2(p, f, make_float2(0.99999928f, 0.99999928f));
  return make_float2(__uint_as_float(__float_as_uint(p.x) + (__float_as_uint(m.x) << 23)), __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(m.y) << 23)));
}

// MN-major operand of 64-element columns `column` bytes apart, 16 keys (two groups of eight 128-byte rows) an instruction
__device__ __forceinline__ uint64_t desc_mn(uint32_t saddr, uint32_t column) {
  return static_cast<uint64_t>((saddr & 0x3FFFF) >> 4) | (static_cast<uint64_t>(column >> 4) << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}

// Tensor maps of the pages for 16-bit caches: boxes of `slots` slots, a power of two that divides a page, and of one.
struct PageMaps {
  CUtensorMap k, v, v_row;
  int slots;
};

template <int DP, int CT, int NQ>
__global__ void __launch_bounds__(TcShape<DP, CT, NQ>::THREADS, 1)
paged_attention_tc_kernel(const __grid_constant__ AttendArgs a, const __grid_constant__ PageMaps maps) {
  using S = TcShape<DP, CT, NQ>;
  constexpr bool BF = S::BF, CODED = S::CODED;
  constexpr int NT = S::NT, NS = S::NS, TILE = S::TILE, SUB = S::SUB, GROUP = S::GROUP;
  constexpr float LOG2E = 1.4426950408889634f;
  extern __shared__ __align__(1024) uint8_t smem[];
  if ((smem_u32(smem) & 1023u) != 0) {  // the swizzled tiles need it
    if (threadIdx.x == 0) atomicExch(a.err_word, 60);
    return;
  }
  uint8_t* sq = smem;
  uint8_t* ring = sq + NT * NQ * TILE;  // (after the queries' terms)
  float* scales = reinterpret_cast<float*>(ring + NS * TILE);
  long long* offs = reinterpret_cast<long long*>(ring + NS * TILE + S::SCALES);
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + NS * TILE + S::SCALES + S::OFFS);
  uint64_t *kv_full = bars, *kv_empty = bars + NS, *s_full = bars + 2 * NS /*[2]*/, *p_full = s_full + 2 /*[2]*/, *pv_done = s_full + 4 /*[2]*/, *drained = s_full + 6;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_full + 7);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* missing = abort_flag + 1;  // the loaders met a page outside the cache

  const PagedView& p = a.p;
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int split = static_cast<int>(blockIdx.x) % a.splits, unit = static_cast<int>(blockIdx.x) / a.splits;
  const ChunkUnit mine = chunk_unit(a, unit);
  if (mine.s < 0) return;
  const PagedSeq seq = mine.seq;
  const int s = mine.s, head = mine.head, n_rows = seq.rows * a.group, r0 = mine.tile * NT * TC_ROWS;
  const int r_end = min(r0 + NT * TC_ROWS, n_rows), tiles_here = (r_end - r0 + TC_ROWS - 1) / TC_ROWS;
  const int pos0 = seq.kv - seq.rows;
  const int pos_first = pos0 + r0 / a.group, pos_last = pos0 + (r_end - 1) / a.group;
  const int k_end = a.causal ? min(seq.kv, pos_last + 1) : seq.kv;
  const int k_begin = a.window > 0 ? max(0, pos_first - a.window + 1) : 0;
  const int t_first = k_begin / TC_KEYS, t_all = k_end > k_begin ? (k_end + TC_KEYS - 1) / TC_KEYS - t_first : 0;
  const int kt0 = t_first + static_cast<int>(static_cast<long long>(t_all) * split / a.splits);
  const int n_kt = t_first + static_cast<int>(static_cast<long long>(t_all) * (split + 1) / a.splits) - kt0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(kv_full + i, CODED ? S::LOADERS : 1);
      mbar_init(kv_empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(p_full + i, 4);
      mbar_init(pv_done + i, 1);
    }
    mbar_init(drained, 1);
    *abort_flag = 0;
    *missing = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == NT * 4) {
    tmem_alloc(tmem_slot, TC_TMEM);
    tmem_relinquish();
  }

  // ---- queries: a softmax thread lays its row out, 8 elements to a 16-byte chunk ---------------------------------------------------------
  float c2 = 0.0f;
  const int t = warp >> 2, r_local = static_cast<int>(threadIdx.x) & 127, r = r0 + t * TC_ROWS + r_local;
  const int tok = r / a.group;
  if (t < NT) {
    const int h = head * a.group + r - tok * a.group;
    const bool there = r < r_end;
    const char* src = static_cast<const char*>(a.q) + ((seq.row0 + tok) * a.q_row + h * a.q_head) * (NQ == 2 ? 4 : 2);
    const bool from_bf = a.type == MIMIR_B200_T_BF16, scaled = NQ == 2 || (!BF && from_bf);
    auto read = [&](int c, float (&f)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = 0.0f;
      if (there && 8 * c < p.head_dim) {
        if constexpr (NQ == 2) unpack8<MIMIR_B200_T_F32>(load8<MIMIR_B200_T_F32>(src + 32 * c), f);
        else if (from_bf) unpack8<MIMIR_B200_T_BF16>(load8<MIMIR_B200_T_BF16>(src + 16 * c), f);
        else unpack8<MIMIR_B200_T_F16>(load8<MIMIR_B200_T_F16>(src + 16 * c), f);
      }
    };
    // bfloat16 and fp32 as halves: the row times a power of two that brings its largest to [1, 2) (bits below 2^-24 of that are lost)
    float up = 1.0f, down = 1.0f;
    if (scaled) {
      float top = 0.0f;
      for (int c = 0; c < DP / 8; ++c) {
        float f[8];
        read(c, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(f[e]));
      }
      const int e2 = min(252, max(1, static_cast<int>(__float_as_uint(top) >> 23)));
      up = __uint_as_float(static_cast<uint32_t>(e2) << 23);
      down = __uint_as_float(static_cast<uint32_t>(254 - e2) << 23);
    }
    // (fp32: the tensor core's sums are low by 1.5e-8 of their value an instruction)
    c2 = fabsf(a.scale) * LOG2E * up * (NQ == 2 ? 1.0f + 1.5e-8f * (DP / 8) : 1.0f);
    c2 = fmaxf(c2, 0x1p-149f);  // (masked scores are -infinity before they are multiplied: a scale of zero would make them no numbers)
    if (a.scale < 0.0f) down = -down;  // (the largest product is then the smallest score's)
    for (int c = 0; c < DP / 8; ++c) {
      float f[8];
      read(c, f);
      uint32_t w[4], l[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) split2<BF>(f[2 * e] * down, f[2 * e + 1] * down, w[e], l[e]);
      uint8_t* to = sq + t * TILE + (c >> 3) * (TC_ROWS * 128) + r_local * 128 + (((c & 7) ^ (r_local & 7)) << 4);
      *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
      if constexpr (NQ == 2) *reinterpret_cast<uint4*>(to + TILE) = make_uint4(l[0], l[1], l[2], l[3]);
    }
    fence_proxy_async_smem();
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  pdl_launch_dependents();  // sequences of few rows, another kernel's, may start on SMs that come free
  const uint32_t tmem = *tmem_slot;
  const uint32_t tmem_o = tmem + 2 * TC_KEYS;  // tile t at + t * DP
  const uint32_t tmem_sum = tmem_o + DP;       // GROUP > 0: of the groups of key tiles before the present one

  if constexpr (CODED) {
    if (warp < NT * 4) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::SOFT_REGS));
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::LOAD_REGS));
  }
  if (warp > NT * 4) {
    // ---- loaders -----------------------------------------------------------------------------------------------------------------------------
    const int id = static_cast<int>(threadIdx.x) - (NT * 128 + 32);
    const uint32_t ring_at = smem_u32(ring);
    if constexpr (!CODED) {
      // one warp brings keys, one values; box x of a tile is (slots of a page, 64 elements)
      const int kv = warp - (NT * 4 + 1), boxes = TC_KEYS / maps.slots;
      int issued = 0;
      for (int j = 0; j < n_kt && kv < 2; ++j) {
        const int i = 2 * j + kv, st = i % NS, key0 = (kt0 + j) * TC_KEYS;
        constexpr int ROUNDS = SUB > 2 ? SUB / 2 : 1;  // (boxes * SUB <= 16 * SUB)
        int page[ROUNDS], slot[ROUNDS];
#pragma unroll
        for (int n = 0; n < ROUNDS; ++n) {
          const int x = n * 32 + lane, key = key0 + x % boxes * maps.slots;
          page[n] = p.n_pages, slot[n] = 0;  // (outside the map: zeros)
          if (x < boxes * SUB && key < k_end && key + maps.slots > k_begin) {
            const int pi = p.by_page.div(key), found = paged_page(p, s, pi);
            slot[n] = key - pi * p.page_size;
            if (found >= 0) page[n] = found;
            else *missing = 1;
          }
        }
        if (!mbar_wait_warp(kv_empty + st, static_cast<uint32_t>((i / NS) & 1) ^ 1, abort_flag, a.err_word, 61)) break;
        if (lane == 0) mbar_expect_tx(kv_full + st, TILE);
        __syncwarp();
#pragma unroll
        for (int n = 0; n < ROUNDS; ++n) {
          const int x = n * 32 + lane, bx = x % boxes, sub = x / boxes, key = key0 + bx * maps.slots;
          if (x >= boxes * SUB) continue;
          const uint32_t dst = ring_at + st * TILE + sub * (TC_KEYS * 128) + bx * maps.slots * 128;
          if (kv == 0) {
            tma_load_4d(dst, &maps.k, kv_full + st, 64 * sub, slot[n], head, page[n]);
          } else if (page[n] == p.n_pages || (key >= k_begin && key + maps.slots <= k_end)) {
            tma_load_4d(dst, &maps.v, kv_full + st, 64 * sub, slot[n], head, page[n]);
          } else {  // (a value that no row sees must be zero whatever its slot holds)
            for (int r = 0; r < maps.slots; ++r)
              tma_load_4d(dst + r * 128, &maps.v_row, kv_full + st, 64 * sub, slot[n] + r, head, key + r >= k_begin && key + r < k_end ? page[n] : p.n_pages);
          }
        }
        __syncwarp();
        issued = j + 1;
      }
      if (*abort_flag && kv < 2) {  // a wait gave up: nothing may still be on its way into shared memory when the block ends
        int still = 0;
        for (int j = max(0, issued - NS / 2); j < issued; ++j)
          mbar_wait_warp(kv_full + (2 * j + kv) % NS, static_cast<uint32_t>(((2 * j + kv) / NS) & 1), &still, a.err_word, 61);
      }
    } else {
      // a tile's codes are on their way in registers while the one before it becomes halves
      constexpr int N = (TC_KEYS * (DP / 8) + S::LOADERS - 1) / S::LOADERS;
      Raw8<CT> raw[N];
      long long scale_at[2] = {-1, -1};
      auto find_rows = [&](int j) {
        const int key0 = (kt0 + j) * TC_KEYS;
        long long* at = offs + (j & 1) * TC_KEYS;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int k = id + i * S::LOADERS, key = key0 + k;
          scale_at[i] = -1;
          if (k < TC_KEYS) {
            long long where = -1;
            if (key >= k_begin && key < k_end) {
              const int pi = p.by_page.div(key), slot = key - pi * p.page_size, page = paged_page(p, s, pi);
              if (page >= 0) {
                where = page * p.page_stride + slot * p.slot_stride + head * p.head_stride;
                scale_at[i] = (static_cast<long long>(page) * p.kv_heads + head) * p.page_size + slot;
              } else {
                *missing = 1;
              }
            }
            at[k] = where;
          }
        }
        __syncwarp();
        asm volatile("barrier.sync 1, %0;" ::"n"(S::LOADERS) : "memory");
      };
      auto fetch = [&](int j, int kv) {
        const long long* at = offs + (j & 1) * TC_KEYS;
        const char* src = static_cast<const char*>(kv ? p.v : p.k);
#pragma unroll
        for (int n = 0; n < N; ++n) {
          const int x = id + n * S::LOADERS, k = x / (DP / 8), c = x % (DP / 8);
          raw[n].w[0] = raw[n].w[1] = 0;
          if (k < TC_KEYS && at[k] >= 0 && 8 * c < p.head_dim) raw[n] = load8<CT>(src + at[k] + 8 * c);
        }
      };
      bool ok = true;
      if (n_kt > 0) {
        find_rows(0);
        fetch(0, 0);
      }
      for (int j = 0; j < n_kt; ++j) {  // (a thread whose wait gave up keeps coming to the barrier)
        float* sc = scales + (j % (NS / 2)) * 2 * TC_KEYS;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const int i = 2 * j + kv, st = i % NS;
          if (ok) ok = mbar_wait(kv_empty + st, static_cast<uint32_t>((i / NS) & 1) ^ 1, abort_flag, a.err_word, 61);
          if (ok) {
#pragma unroll
            for (int n = 0; n < N; ++n) {
              const int x = id + n * S::LOADERS, k = x / (DP / 8), c = x % (DP / 8);
              uint32_t hi[4];
              to_pairs<CT>(raw[n], hi);
              if (k < TC_KEYS)
                *reinterpret_cast<uint4*>(ring + st * TILE + (c >> 3) * (TC_KEYS * 128) + k * 128 + (((c & 7) ^ (k & 7)) << 4)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            }
            if (kv) {  // both scales with the values, whose stage is let go of last
#pragma unroll
              for (int n = 0; n < 2; ++n) {
                const int k = id + n * S::LOADERS;
                if (k < TC_KEYS) {
                  sc[k] = scale_at[n] >= 0 ? __ldg(p.k_scale + scale_at[n]) : 0.0f;
                  sc[TC_KEYS + k] = scale_at[n] >= 0 ? __ldg(p.v_scale + scale_at[n]) : 0.0f;
                }
              }
            }
            fence_proxy_async_smem();
            mbar_arrive(kv_full + st);
          }
          if (kv == 0) {
            fetch(j, 1);
          } else if (j + 1 < n_kt) {
            find_rows(j + 1);
            fetch(j + 1, 0);
          }
        }
      }
    }
  } else if (warp == NT * 4) {
    // ---- tensor instructions -------------------------------------------------------------------------------------------------------------------
    const uint32_t idesc_s = make_idesc(TC_ROWS, TC_KEYS, BF ? 0 : 1), idesc_o = make_idesc(TC_ROWS, DP, BF ? 0 : 1) | (1u << 16);
    const uint32_t q_at = smem_u32(sq), ring_at = smem_u32(ring);
    auto scores = [&](int tt, int j) {  // S = Q_tt K_j^T
      const uint32_t k_at = ring_at + ((2 * j) % NS) * TILE, d = tmem + (NT == 2 ? tt : (j & 1)) * TC_KEYS;
      const uint64_t q_desc = make_smem_desc(q_at + tt * TILE, 128), k_desc = make_smem_desc(k_at, 128);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          const uint64_t o = ((k >> 2) * (TC_KEYS * 128) + (k & 3) * 32) >> 4;
          umma_bf16(d, q_desc + o, k_desc + o, idesc_s, k != 0 ? 1u : 0u);
          if constexpr (NQ == 2) umma_bf16(d, q_desc + (TILE >> 4) + o, k_desc + o, idesc_s, 1u);
        }
        umma_commit(s_full + (NT == 2 ? tt : (j & 1)));
      }
      __syncwarp();
    };
    auto values = [&](int tt, int j) {  // O_tt (+)= P V_j
      const uint32_t v_at = ring_at + ((2 * j + 1) % NS) * TILE, pa = tmem + (NT == 2 ? tt : (j & 1)) * TC_KEYS, d = tmem_o + tt * DP;
      const uint64_t v_desc = desc_mn(v_at, TC_KEYS * 128);
      const int first = GROUP > 0 ? j & (GROUP - 1) : j;
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < TC_KEYS / 16; ++k) {
          umma_f16_ts(d, pa + 8 * k, v_desc + ((k * 2048) >> 4), idesc_o, (first | k) != 0 ? 1u : 0u);
          if constexpr (NQ == 2) umma_f16_ts(d, pa + TC_KEYS / 2 + 8 * k, v_desc + ((k * 2048) >> 4), idesc_o, 1u);
        }
        umma_commit(pv_done + tt);
      }
      __syncwarp();
    };
    auto release = [&](int i) {
      if (elect_one()) umma_commit(kv_empty + i % NS);
      __syncwarp();
    };
    auto full = [&](int i, int where) {
      const bool ok = mbar_wait_warp(kv_full + i % NS, static_cast<uint32_t>((i / NS) & 1), abort_flag, a.err_word, where);
      tcgen05_fence_after();
      return ok;
    };
    auto ready = [&](int tt, int j) {
      const bool ok = mbar_wait_warp(p_full + (NT == 2 ? tt : (j & 1)), static_cast<uint32_t>((NT == 2 ? j : j >> 1) & 1), abort_flag, a.err_word, 64);
      tcgen05_fence_after();
      return ok;
    };
    bool ok = n_kt > 0 && full(0, 62);
    if (ok) {
      for (int tt = 0; tt < tiles_here; ++tt) scores(tt, 0);
      release(0);
    }
    for (int j = 0; j < n_kt && ok; ++j) {
      const bool more = j + 1 < n_kt;
      if constexpr (NT == 2) {
        for (int tt = 0; tt < tiles_here && ok; ++tt) {
          ok = (tt > 0 || full(2 * j + 1, 63)) && ready(tt, j);
          if (!ok) break;
          values(tt, j);
          if (tt == tiles_here - 1) release(2 * j + 1);
          if (more) {
            if (tt == 0) ok = full(2 * j + 2, 62);
            if (!ok) break;
            scores(tt, j + 1);
            if (tt == tiles_here - 1) release(2 * j + 2);
          }
        }
      } else {
        if (more) {
          ok = full(2 * j + 2, 62);
          if (!ok) break;
          scores(0, j + 1);
          release(2 * j + 2);
        }
        ok = full(2 * j + 1, 63) && ready(0, j);
        if (!ok) break;
        values(0, j);
        release(2 * j + 1);
      }
    }
    // everything issued has finished before tensor memory is let go of
    if (elect_one()) umma_commit(drained);
    __syncwarp();
    int drain_abort = 0;
    mbar_wait_warp(drained, 0, &drain_abort, a.err_word, 65);
  } else if (t < tiles_here) {
    // ---- softmax: a thread a row -------------------------------------------------------------------------------------------------------------------
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const int pos = pos0 + min(tok, (r_end - 1) / a.group);
    const int lim_hi = a.causal ? min(seq.kv, pos + 1) : seq.kv, lim_lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    // of all of this warp's rows: keys that every row sees (positions ascend with the rows)
    const int w_first = __shfl_sync(0xffffffffu, pos, 0), w_last = __shfl_sync(0xffffffffu, pos, 31);
    const int all_hi = a.causal ? min(seq.kv, w_first + 1) : seq.kv, all_lo = a.window > 0 ? max(0, w_last - a.window + 1) : 0;
    float base = -INFINITY, sum = 0.0f;
    float sum_f = 1.0f, o_f = 1.0f;  // GROUP > 0: what the sum of the earlier groups, and O where it is complete, are still to be multiplied by
    float v_unit = 0.0f;  // codes: the power of two that O's values are in
    if constexpr (GROUP > 0) {  // (a sum that starts from zero has one form of addition; with a first one of its own 1 to 6 % more time)
      uint32_t none[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) none[i] = 0;
#pragma unroll 1
      for (int c = 0; c < DP / 32; ++c) tmem_st_32x32(tmem_sum + lanes + 32 * c, none);
      tmem_wait_st();
    }
    bool alive = true;
    for (int j = 0; j < n_kt; ++j) {
      const int buf = NT == 2 ? t : (j & 1);
      const uint32_t ts = tmem + buf * TC_KEYS + lanes;
      alive = mbar_wait_warp(s_full + buf, static_cast<uint32_t>((NT == 2 ? j : j >> 1) & 1), abort_flag, a.err_word, 66);
      const float* sc = scales + (j % (NS / 2)) * 2 * TC_KEYS;
      if (CODED && alive) alive = mbar_wait_warp(kv_full + (2 * j + 1) % NS, static_cast<uint32_t>(((2 * j + 1) / NS) & 1), abort_flag, a.err_word, 67);
      if (!alive) break;
      tcgen05_fence_after();
      const int key0 = (kt0 + j) * TC_KEYS;
      const bool masked = key0 < all_lo || key0 + TC_KEYS > all_hi || *missing;
      // 32 scores of the row, times their keys' scales, with what the row does not see at -infinity
      auto read_scores = [&](int c, uint32_t (&w)[32]) {
        tmem_ld_32x32_nowait(ts + 32 * c, w);
        tmem_wait_ld_regs(w);
        if constexpr (CODED) {
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 k4 = *reinterpret_cast<const float4*>(sc + 32 * c + i);
            w[i] = __float_as_uint(__uint_as_float(w[i]) * k4.x);
            w[i + 1] = __float_as_uint(__uint_as_float(w[i + 1]) * k4.y);
            w[i + 2] = __float_as_uint(__uint_as_float(w[i + 2]) * k4.z);
            w[i + 3] = __float_as_uint(__uint_as_float(w[i + 3]) * k4.w);
          }
        }
        if (masked) {
          const int lo = lim_lo - key0 - 32 * c, hi = lim_hi - key0 - 32 * c;
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (i < lo || i >= hi) w[i] = 0xff800000u;
          if (*missing) {  // a page of this sequence is none of the cache's: which keys are out is looked up again
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              const int key = key0 + 32 * c + i;
              if (key + 7 >= k_begin && key < k_end && paged_page(p, s, p.by_page.div(key)) < 0) {
#pragma unroll
                for (int e = 0; e < 8; ++e) w[i + e] = 0xff800000u;
              }
            }
          }
        }
      };
      auto largest = [&](const uint32_t (&w)[32], float m) {
        float m4[4] = {m, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 32; i += 2) m4[(i >> 1) & 3] = max3(m4[(i >> 1) & 3], __uint_as_float(w[i]), __uint_as_float(w[i + 1]));
        return max3(max3(m4[0], m4[1], m4[2]), m4[3], m4[3]);
      };
      float grow = 0.0f;
      if constexpr (CODED) {
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(sc[TC_KEYS + 32 * i + lane]));
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const int e2 = min(240, max(14, static_cast<int>(__float_as_uint(top) >> 23)));
        grow = __uint_as_float(static_cast<uint32_t>(e2) << 23);
      }
      const bool complete = GROUP > 0 && j > 0 && (j & (GROUP - 1)) == 0;  // O is a group's: the next product starts another
      // another maximum, and O with it
      auto rescale = [&](float mx) {
        const float nb = fmaxf(base, mx - S::ROOM);
        float f = base == -INFINITY ? 0.0f : ex2f(base - nb);
        sum *= f;
        base = nb;
        if constexpr (CODED) {
          const float nu = fmaxf(v_unit, grow);
          f *= v_unit / nu;
          v_unit = nu;
        }
        sum_f *= f;
        if (complete) o_f *= f;
        if (j == 0 || complete) return true;
        if (!mbar_wait_warp(pv_done + (NT == 2 ? t : 0), static_cast<uint32_t>(j - 1) & 1, abort_flag, a.err_word, 68)) return false;
        tcgen05_fence_after();
#pragma unroll 1
        for (int c = 0; c < DP / 32; ++c) {
          uint32_t o[32];
          tmem_ld_32x32_nowait(tmem_o + t * DP + lanes + 32 * c, o);
          tmem_wait_ld_regs(o);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
          tmem_st_32x32(tmem_o + t * DP + lanes + 32 * c, o);
        }
        return true;
      };
      uint32_t pk[4][16], pl[4][16];  // (pl: what the rounding leaves, for fp32)
      float2 part[2];
      // the probabilities by the present maximum, packed; the largest score on the way
      auto weigh_keys = [&](auto few_special) {
        const float sub = base == -INFINITY ? 0.0f : base, inv_unit = CODED ? 1.0f / v_unit : 1.0f;
        const float2 cc = make_float2(c2, c2), ss = make_float2(-sub, -sub);
        part[0] = part[1] = make_float2(0.0f, 0.0f);
        float mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t w[32];
          read_scores(c, w);
          mx = largest(w, mx);
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float2 x = fma2(make_float2(__uint_as_float(w[i]), __uint_as_float(w[i + 1])), cc, ss);
            // (keys behind a mask need an exact zero: they take the special function)
            float2 e = decltype(few_special)::value && (i & TC_POLY) == TC_POLY ? exp2_poly(x) : make_float2(ex2f(x.x), ex2f(x.y));
            part[(i >> 1) & 1] = add2(part[(i >> 1) & 1], e);
            if constexpr (CODED) {
              const float2 v2 = *reinterpret_cast<const float2*>(sc + TC_KEYS + 32 * c + i);
              e.x *= v2.x * inv_unit, e.y *= v2.y * inv_unit;
            }
            if constexpr (NQ == 2) split2<BF>(e.x, e.y, pk[c][i / 2], pl[c][i / 2]);
            else pk[c][i / 2] = pack2<BF>(e.x, e.y);
          }
        }
        return mx * c2;
      };
      // a first maximum where a row of the warp has none yet; after that the present one is used at once, and only where a score outgrows it
      // by more than 2^8 (a few times a row), or is not a number, are the tile's probabilities computed again by a new one and without polynomials
      if (__any_sync(0xffffffffu, base == -INFINITY) || (CODED && grow > v_unit)) {
        float mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t w[32];
          read_scores(c, w);
          mx = largest(w, mx);
        }
        if (!rescale(mx * c2)) { alive = false; break; }
      }
      const float mx = masked ? weigh_keys(std::false_type()) : weigh_keys(std::integral_constant<bool, NQ == 1>());
      if (__any_sync(0xffffffffu, !(mx <= base + (8.0f + S::ROOM)))) {
        if (!rescale(mx)) { alive = false; break; }
        weigh_keys(std::false_type());
      }
      sum += (part[0].x + part[0].y) + (part[1].x + part[1].y);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        tmem_st_32x16(ts + 16 * c, pk[c]);
        if constexpr (NQ == 2) tmem_st_32x16(ts + TC_KEYS / 2 + 16 * c, pl[c]);
      }
      if (GROUP > 0 && complete) {
        alive = mbar_wait_warp(pv_done, static_cast<uint32_t>(j - 1) & 1, abort_flag, a.err_word, 70);
        if (!alive) break;
        tcgen05_fence_after();
#pragma unroll 1
        for (int c = 0; c < DP / 32; ++c) {
          uint32_t o[32], old[32];
          tmem_ld_32x32_nowait(tmem_o + lanes + 32 * c, o);
          tmem_ld_32x32_nowait(tmem_sum + lanes + 32 * c, old);
          tmem_wait_ld_regs(o);
          tmem_wait_ld_regs(old);
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float v = __uint_as_float(o[i]) * o_f;
            o[i] = __float_as_uint(fmaf(__uint_as_float(old[i]), sum_f, v));
          }
          tmem_st_32x32(tmem_sum + lanes + 32 * c, o);
        }
        sum_f = o_f = 1.0f;
      }
      tmem_wait_st();
      tcgen05_fence_before();
      // With two score tiles the last product's wait, below, comes while the one before it may still run, and a barrier two phases behind looks
      // complete.  So that one is waited for first; here, where the last cannot be through yet: two phases ahead looks incomplete for good.
      if (NT == 1 && j > 0 && j + 1 == n_kt) {
        alive = mbar_wait_warp(pv_done, static_cast<uint32_t>(j - 1) & 1, abort_flag, a.err_word, 69);
        if (!alive) break;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full + buf);
    }
    if (alive && n_kt > 0) alive = mbar_wait_warp(pv_done + (NT == 2 ? t : 0), static_cast<uint32_t>(n_kt - 1) & 1, abort_flag, a.err_word, 69);
    if (alive) {
      tcgen05_fence_after();
      const bool there = r < r_end;
      // fp32: a group's products, two instructions for 16 keys that the row sees, are low by 1.5e-8 an instruction where these weigh alike, by
      // nothing or twice that where the last or the first have all the weight
      const int keys_seen = max(0, min(lim_hi, (kt0 + n_kt) * TC_KEYS) - max(lim_lo, kt0 * TC_KEYS));
      const float unit_v = (CODED ? v_unit : 1.0f) * (GROUP > 0 ? 1.0f + 1.5e-8f * (min(keys_seen, GROUP * TC_KEYS) / 8) : 1.0f);
      const float inv = a.splits > 1 ? unit_v : sum == 0.0f ? 0.0f : unit_v / sum;
      const int h = head * a.group + r - tok * a.group;
      const long long part_row = static_cast<long long>(blockIdx.x) * (NT * TC_ROWS) + t * TC_ROWS + r_local;
      char* dst = static_cast<char*>(a.out) + ((seq.row0 + tok) * a.o_row + h * a.o_head) * (NQ == 2 ? 4 : 2);
#pragma unroll 1
      for (int c = 0; c < DP / 32; ++c) {
        uint32_t o[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = 0;
        if (n_kt > 0) {
          tmem_ld_32x32_nowait(tmem_o + t * DP + lanes + 32 * c, o);
          tmem_wait_ld_regs(o);
          if (GROUP > 0 && n_kt > GROUP) {
            uint32_t old[32];
            tmem_ld_32x32_nowait(tmem_sum + lanes + 32 * c, old);
            tmem_wait_ld_regs(old);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(fmaf(__uint_as_float(old[i]), sum_f, __uint_as_float(o[i])));
          }
        }
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          const int d = 32 * c + i;
          if (!there || d >= p.head_dim) continue;
          float f[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(o[i + e]) * inv;
          if (a.splits > 1) {
            store8<MIMIR_B200_T_F32>(a.part_o + part_row * p.head_dim + d, pack8<MIMIR_B200_T_F32>(f));
          } else if constexpr (NQ == 2) {
            store8<MIMIR_B200_T_F32>(dst + 4 * d, pack8<MIMIR_B200_T_F32>(f));
          } else if (a.type == MIMIR_B200_T_BF16) {
            store8<MIMIR_B200_T_BF16>(dst + 2 * d, pack8<MIMIR_B200_T_BF16>(f));
          } else {
            store8<MIMIR_B200_T_F16>(dst + 2 * d, pack8<MIMIR_B200_T_F16>(f));
          }
        }
        __syncwarp();
      }
      if (there) {
        if (a.splits > 1) a.part_ml[part_row] = make_float2(base, sum);
        else store_lse(a, seq.row0, r, head, base, sum);
      }
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == NT * 4) {
    tcgen05_fence_after();
    tmem_dealloc(tmem, TC_TMEM);
  }
}

// 4-D map over the pages of a 16-bit cache: (element, slot, head, page), boxes of 64 elements and `slots` slots, 128-byte swizzle
int make_page_map(CUtensorMap* map, const PagedView& p, const void* base, int slots) {
  using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static EncodeFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) f = nullptr;
    return reinterpret_cast<EncodeFn>(f);
  }();
  if (!fn) return fail(MIMIR_B200_E_CUDA, "cuTensorMapEncodeTiled entry point not available");
  auto bytes = [](int extent, long long stride) { return static_cast<cuuint64_t>(extent > 1 ? stride * 2 : 16); };  // (one of a kind has no stride)
  cuuint64_t dims[4] = {static_cast<cuuint64_t>(p.head_dim), static_cast<cuuint64_t>(p.page_size), static_cast<cuuint64_t>(p.kv_heads), static_cast<cuuint64_t>(p.n_pages)};
  cuuint64_t strides[3] = {bytes(p.page_size, p.slot_stride), bytes(p.kv_heads, p.head_stride), bytes(p.n_pages, p.page_stride)};
  cuuint32_t box[4] = {64, static_cast<cuuint32_t>(slots), 1, 1};
  cuuint32_t step[4] = {1, 1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(MIMIR_B200_E_UNSUPPORTED, "paged_attention: no tensor map over these pages (%d)", static_cast<int>(r));
  return MIMIR_B200_OK;
}

template <int DP, int CT, int NQ>
int launch_tc_as(const AttendArgs& a, long long grid, cudaStream_t st) {
  using S = TcShape<DP, CT, NQ>;
  static PerDeviceOnce once;
  MB_TRY(once.run([]() -> int {
    MB_CUDA(cudaFuncSetAttribute(paged_attention_tc_kernel<DP, CT, NQ>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
    if (S::CODED) {  // (setmaxnreg waits for registers of the launch's own: with fewer than the shares add up to it would wait for good)
      cudaFuncAttributes at;
      MB_CUDA(cudaFuncGetAttributes(&at, paged_attention_tc_kernel<DP, CT, NQ>));
      if (at.numRegs < S::LAUNCH_REGS) return fail(MIMIR_B200_E_UNSUPPORTED, "paged_attention: compiled with %d registers a thread, %d are shared out", at.numRegs, S::LAUNCH_REGS);
    }
    return MIMIR_B200_OK;
  }));
  PageMaps maps = {};
  if constexpr (!S::CODED) {
    maps.slots = 8;
    while (maps.slots < TC_KEYS && a.p.page_size % (2 * maps.slots) == 0) maps.slots *= 2;
    MB_TRY(make_page_map(&maps.k, a.p, a.p.k, maps.slots));
    MB_TRY(make_page_map(&maps.v, a.p, a.p.v, maps.slots));
    MB_TRY(make_page_map(&maps.v_row, a.p, a.p.v, 1));
  }
  paged_attention_tc_kernel<DP, CT, NQ><<<static_cast<unsigned>(grid), S::THREADS, S::SMEM, st>>>(a, maps);
  MB_CUDA(cudaGetLastError());
  count_launch();
  return MIMIR_B200_OK;
}
template <int CT>
int launch_tc_dim(const AttendArgs& a, long long grid, cudaStream_t st) {
  if constexpr (CT != MIMIR_B200_T_BF16) {
    if (a.type == MIMIR_B200_T_F32) return a.p.head_dim <= 64 ? launch_tc_as<64, CT, 2>(a, grid, st) : launch_tc_as<128, CT, 2>(a, grid, st);
  }
  if (a.p.head_dim <= 64) return launch_tc_as<64, CT, 1>(a, grid, st);
  if (a.p.head_dim <= 128) return launch_tc_as<128, CT, 1>(a, grid, st);
  return launch_tc_as<256, CT, 1>(a, grid, st);
}

}  // namespace

int launch_paged_attention_tc(const AttendArgs& a, int cache_type, long long grid, cudaStream_t st) {
  switch (cache_type) {
    case MIMIR_B200_T_F16: return launch_tc_dim<MIMIR_B200_T_F16>(a, grid, st);
    case MIMIR_B200_T_BF16: return launch_tc_dim<MIMIR_B200_T_BF16>(a, grid, st);
    case MIMIR_B200_T_I8: return launch_tc_dim<MIMIR_B200_T_I8>(a, grid, st);
    default: return launch_tc_dim<MIMIR_B200_T_E4M3>(a, grid, st);
  }
}

}  // namespace mb
