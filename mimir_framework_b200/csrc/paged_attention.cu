// paged_attention.cu — attention of new tokens over a paged key / value cache: softmax(scale q k^T + mask) v per head, the heads of a
// group sharing their key head, each sequence with its own lengths.
//
// One token a sequence reads every cached key and value once and computes little: the cache's bytes at the memory rate are the
// floor.  So K and V go from global memory straight into the registers that feed the tensor instruction (mma.sync m16n8k16), with no
// shared memory between: the contraction index of Q K^T may be permuted (Q's fragments are laid out the same way), and so may the
// columns of P V, so that a lane reads eight consecutive elements of a row each time and a warp whole sectors.
//   rows     16 (token, head of the group) pairs of one key head are a tile: heads that share keys share the read
//   keys     a warp takes blocks of KB keys with a running maximum and sum per row; warps, and the CTAs of a cluster, split the blocks and
//            meet in (distributed) shared memory in a fixed order
//   K        lane (g, t) holds elements 8 t .. 8 t + 7 of each 32 of key g:  two contraction steps
//   V        lane (g, t) holds elements 8 g .. 8 g + 7 of each 64 of keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9: eight column tiles
// fp32 caches, and what meets them, are two terms of 11 bits with fp32's exponents (hi + lo, m16n8k8): an element keeps 22 bits by itself, whatever
// is beside it.  Halves would take half the tensor instructions (64 sequences of up to 4 K keys 368 us, 445 so; heads of 64 199 and 218) but cannot
// hold what is far from one.  Over other caches fp32 queries and probabilities are two IEEE-half terms (22 bits): queries after a power of two per row has brought
// their largest to [1, 2).  Probabilities are two terms for bfloat16 caches too (16 bits), one half (11 bits) where only the result is bfloat16.
// Codes of eight bits are exact in half; their scales multiply scores and probabilities.  For fp32 results each block's P V starts from
// zero and is added in fp32, because the tensor core's accumulation truncates (1.5e-8 of the value an instruction, up to 2^-23).
// 64 sequences of up to 4 K bfloat16 keys, 8 key heads of 128: 165 us, 0.75 of the copy rate (bytes in flight: eight warps an SM, whose registers
// hold them; CTAs of unequal length).  4 of up to 128 K e4m3 keys: 210 us, 0.69 of it (the loads' latency again, and codes that become halves).
#include <cmath>

#include "common.h"
#include "launch.cuh"
#include "paged.cuh"
#include "paged_attention.cuh"

namespace mb {
namespace {

constexpr int PA_WARPS = 4, PA_THREADS = 32 * PA_WARPS, PA_ROWS = 16;

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// m16n8k8 of fp32 numbers with 11 bits: lane (g, t) has rows g and g + 8 of A in columns t (x, y) and t + 4 (z, w), rows t and t + 4 of column g of B
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// a number of fp32 as two of 11 bits each, off by 2^-22 of it whatever its size (the first is cut off, not rounded: an instruction less, and
// the largest numbers stay finite)
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = __float_as_uint(x) & 0xffffe000u;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(x - __uint_as_float(hi)));
}
template <bool BF>
__device__ __forceinline__ void mma16(float (&c)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  if constexpr (BF) mma_bf16(c, a, b0, b1);
  else mma_f16(c, a, b0, b1);
}
// shared memory of cluster rank `rank`
__device__ __forceinline__ uint32_t cluster_address(const float* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))), "r"(rank));
  return a;
}
__device__ __forceinline__ float ld_cluster(const float* p, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_address(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster4(const float* p, uint32_t rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_address(p, rank)) : "memory");
  return v;
}

template <int CT, int NQ, int NP, int DP>  // terms of a query and of a probability
struct PagedShape {
  static constexpr bool BF = CT == MIMIR_B200_T_BF16, WIDE = CT == MIMIR_B200_T_F32;
  // halves: probabilities of up to 2^14 (times a code's scale 2^15) are exact to 2^-39 of the largest where 2^-25 would be
  static constexpr float ROOM = BF || WIDE ? 0.0f : 14.0f;
  static constexpr bool FRESH = NQ == 2;                                // P V of a block apart from O
  static constexpr int KB = type_bytes(CT) == 1 || (type_bytes(CT) == 2 && DP <= 128) ? 32 : 16;  // keys of a block
  static constexpr int UD = CT == MIMIR_B200_T_F32 ? 64 : DP < 128 ? DP : 128;  // head elements loaded at a time
  static constexpr int Q_STEPS = DP / (WIDE ? 8 : 16), Q_BYTES = NQ * Q_STEPS * 32 * 16;  // of the contraction
  static constexpr int O_STRIDE = DP + 4;
  static constexpr int SMEM = Q_BYTES + PA_WARPS * PA_ROWS * (O_STRIDE + 2) * 4 + 2 * PA_ROWS * 4;
};

// (three CTAs to an SM where that spills little; fp32 caches, heads of 64, 64 sequences of up to 4 K keys: 285 us in three, 218 in two)
template <int CT, int NQ, int NP, int DP>
__global__ void __launch_bounds__(PA_THREADS, DP > 64 || CT == MIMIR_B200_T_F32 ? 2 : 3)
paged_attention_kernel(const __grid_constant__ AttendArgs a) {
  using S = PagedShape<CT, NQ, NP, DP>;
  constexpr bool BF = S::BF, CODED = CT == MIMIR_B200_T_I8 || CT == MIMIR_B200_T_E4M3, WIDE = S::WIDE;
  constexpr int KB = S::KB, NG = KB / 8, UD = S::UD, NU = DP / UD;
  constexpr float LOG2E = 1.4426950408889634f;
  extern __shared__ __align__(16) uint8_t smem[];
  uint4* sq = reinterpret_cast<uint4*>(smem);                        // [NQ][Q_STEPS][32 lanes]
  float* so = reinterpret_cast<float*>(smem + S::Q_BYTES);           // [warp][16][O_STRIDE]
  float* sm = so + PA_WARPS * PA_ROWS * S::O_STRIDE;                 // [warp][16] maxima, then [warp][16] sums
  float* sl = sm + PA_WARPS * PA_ROWS;
  float* sscale = sl + PA_WARPS * PA_ROWS;                           // [16]
  const PagedView& p = a.p;
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);  // (known to be the same in all lanes: uniform branches)
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = static_cast<int>(blockIdx.x) % a.cluster;
  const int part = static_cast<int>(blockIdx.x) / a.cluster;
  const int split = part % a.splits, unit = part / a.splits;
  const int tile = unit % a.tiles, sh = unit / a.tiles, head = sh % p.kv_heads, s = sh / p.kv_heads;
  const PagedSeq q = paged_seq(p, s);
  const int r0 = tile * PA_ROWS, n_rows = q.rows * a.group;
  // Launched behind chunks it runs beside their last blocks, of which it reads nothing; one block of it ends after them, and so does the launch.
  const bool last = blockIdx.x + 1 == gridDim.x;
  if (r0 >= n_rows || n_rows > a.few) {  // (the whole cluster)
    if (last) pdl_wait();
    return;
  }
  const int r_end = min(r0 + PA_ROWS, n_rows);
  const int pos0 = q.kv - q.rows;  // of the sequence's first new token
  const int pos_first = pos0 + r0 / a.group, pos_last = pos0 + (r_end - 1) / a.group;
  const int k_end = a.causal ? min(q.kv, pos_last + 1) : q.kv;
  const int k_begin = a.window > 0 ? max(0, pos_first - a.window + 1) : 0;
  const int b_first = k_begin / KB, blocks = k_end > k_begin ? (k_end + KB - 1) / KB - b_first : 0;
  const int workers = a.splits * a.cluster * PA_WARPS, me = (split * a.cluster + rank) * PA_WARPS + warp;
  const int b0 = b_first + static_cast<int>(static_cast<long long>(blocks) * me / workers);
  const int b1 = b_first + static_cast<int>(static_cast<long long>(blocks) * (me + 1) / workers);

  // ---- the queries of the tile as fragments, hi (+ lo): a warp takes four rows -------------------------------------------------
#pragma unroll
  for (int i = 0; i < PA_ROWS / PA_WARPS; ++i) {
    const int row = i * PA_WARPS + warp, r = r0 + row;
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = 0.0f;
    const int d = lane * 8;
    if (r < r_end && d < p.head_dim) {
      const int tok = r / a.group, h = head * a.group + r - tok * a.group;
      const char* src = static_cast<const char*>(a.q) + ((q.row0 + tok) * a.q_row + h * a.q_head + d) * static_cast<long long>(type_bytes(a.type));
      if (a.type == MIMIR_B200_T_F32) unpack8<MIMIR_B200_T_F32>(load8<MIMIR_B200_T_F32>(src), f);
      else if (a.type == MIMIR_B200_T_F16) unpack8<MIMIR_B200_T_F16>(load8<MIMIR_B200_T_F16>(src), f);
      else unpack8<MIMIR_B200_T_BF16>(load8<MIMIR_B200_T_BF16>(src), f);
    }
    float scale = 1.0f;
    if (!BF && !WIDE && a.type != MIMIR_B200_T_F16) {
      float top = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(f[e]));
#pragma unroll
      for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      // two to the exponent of the largest, in [2^-126, 2^126] (an infinity stays one)
      const int e2 = min(252, max(1, static_cast<int>(__float_as_uint(top) >> 23)));
      scale = __uint_as_float(static_cast<uint32_t>(e2) << 23);
      const float inv = __uint_as_float(static_cast<uint32_t>(254 - e2) << 23);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] *= inv;
    }
    if (lane == 0) sscale[row] = scale;
    if (WIDE && d < DP) {
      // elements 8 c + 2 i and + 1 belong to lane (row % 8, c % 4) of step 4 (c / 4) + i: registers row / 8 and row / 8 + 2
      const int c = lane, to = (row & 7) * 4 + (c & 3), reg = row >> 3;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        uint32_t hi, lo;
        split_tf32(f[e], hi, lo);
        uint32_t* w = reinterpret_cast<uint32_t*>(sq + (4 * (c / 4) + e / 2) * 32 + to) + reg + 2 * (e & 1);
        w[0] = hi, w[S::Q_STEPS * 32 * 4] = lo;
      }
    } else if (d < DP) {
      // elements 8 c .. 8 c + 7 belong to lane (row % 8, c % 4) of steps 2 (c / 4) and 2 (c / 4) + 1: registers row / 8 and row / 8 + 2
      const int c = lane;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t hi0, lo0, hi1, lo1;
        split2<BF>(f[4 * half], f[4 * half + 1], hi0, lo0);
        split2<BF>(f[4 * half + 2], f[4 * half + 3], hi1, lo1);
        const int step = 2 * (c / 4) + half, to = (row & 7) * 4 + (c & 3), reg = row >> 3;
        uint32_t* w = reinterpret_cast<uint32_t*>(sq + step * 32 + to);
        w[reg] = hi0, w[reg + 2] = hi1;
        if constexpr (NQ == 2) {
          w = reinterpret_cast<uint32_t*>(sq + (S::Q_STEPS + step) * 32 + to);
          w[reg] = lo0, w[reg + 2] = lo1;
        }
      }
    }
  }
  __syncthreads();

  // scores in the exponent's base two, and the positions of this lane's two rows
  float c2[2];
  int lim_hi[2], lim_lo[2];  // keys lim_lo .. lim_hi - 1 are seen
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    c2[i] = a.scale * LOG2E * sscale[g + 8 * i];
    const int pos = pos0 + min(r0 + g + 8 * i, r_end - 1) / a.group;
    lim_hi[i] = a.causal ? min(q.kv, pos + 1) : q.kv;
    lim_lo[i] = a.window > 0 ? max(0, pos - a.window + 1) : 0;
  }
  const int all_lo = a.window > 0 ? max(0, pos_last - a.window + 1) : 0, all_hi = a.causal ? min(q.kv, pos_first + 1) : q.kv;

  float o[DP / 8][4];
#pragma unroll
  for (int j = 0; j < DP / 8; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[j][i] = 0.0f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

  // ---- pages of groups of eight keys (a page holds a multiple of eight): a lane looks one up, 32 of them ahead of their blocks -----------
  int ahead_page, ahead_slot;  // of this lane's group of the next 32
  int window = b0 * NG;        // first group of the present 32
  auto look_up = [&](int first_group) {
    const int key = (first_group + lane) * 8;
    ahead_page = -2;  // no key of it is wanted
    if (first_group + lane < b1 * NG && key < k_end && key + 7 >= k_begin) {
      const int pi = p.by_page.div(key);
      ahead_slot = key - pi * p.page_size;
      ahead_page = __ldg(p.table + s * p.table_stride + pi);
    }
  };
  long long g_off, g_soff;  // where this lane's group begins in the pages and in the scales, -1: nowhere
  unsigned g_there;         // lanes whose group is somewhere
  auto take_window = [&]() {
    g_off = -1;
    if (static_cast<unsigned>(ahead_page) < static_cast<unsigned>(p.n_pages)) {
      g_off = ahead_page * p.page_stride + ahead_slot * p.slot_stride + head * p.head_stride;
      g_soff = (static_cast<long long>(ahead_page) * p.kv_heads + head) * p.page_size + ahead_slot;
    } else if (ahead_page != -2) {
      atomicOr(p.flags, PAGED_BAD_PAGE);
    }
    g_there = __ballot_sync(0xffffffffu, g_off >= 0);
    look_up(window + 32);
  };
  long long off[NG], soff[NG];
  unsigned there = 0;   // groups of the block that are somewhere
  bool whole = false;   // every key of the block is there
  auto place_pages = [&](int b) {
    int at = b * NG - window;
    if (at >= 32) {
      window += 32, at -= 32;
      take_window();
    }
    there = (g_there >> at) & ((1u << NG) - 1);
    whole = there == (1u << NG) - 1 && b * KB >= k_begin && b * KB + KB <= k_end;
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      off[j] = __shfl_sync(0xffffffffu, g_off, at + j);
      if constexpr (CODED) soff[j] = __shfl_sync(0xffffffffu, g_soff, at + j) + 2 * t;
    }
    if (at + 2 * NG <= 32) {  // the next block's rows, a line a lane
      constexpr int LINES = DP * type_bytes(CT) > 128 ? DP * type_bytes(CT) / 128 : 1;  // of a row
#pragma unroll
      for (int n = 0; n < 2 * KB * LINES / 32; ++n) {
        const int i = n * 32 + lane, line = i % LINES, key = (i / LINES) % KB, is_v = i / (LINES * KB);
        const long long row = __shfl_sync(0xffffffffu, g_off, at + NG + key / 8);
        const char* src = static_cast<const char*>(is_v ? p.v : p.k) + (row + (key & 7) * p.slot_stride) * type_bytes(CT) + 128 * line;
        asm volatile("prefetch.global.L2 [%0];" ::"l"(row >= 0 && 128 * line < p.head_dim * type_bytes(CT) ? src : static_cast<const char*>(p.k)));
      }
    }
  };
  Raw8<CT> kr[NG][UD / 32], vr[KB / 16][4][(UD + 63) / 64];
  float2 ks[NG], vs[NG];
  const long long k_lane = (g * p.slot_stride + 8 * t) * type_bytes(CT), v_lane = (2 * t * p.slot_stride + 8 * g) * type_bytes(CT), row_bytes = p.slot_stride * type_bytes(CT);
  const bool full_dim = p.head_dim == DP;
  auto load_k = [&](int b, int u) {
    if (whole && full_dim) {  // (most blocks: nothing to test)
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        const char* base = static_cast<const char*>(p.k) + off[j] * type_bytes(CT) + k_lane;
#pragma unroll
        for (int c = 0; c < UD / 32; ++c) kr[j][c] = load8<CT>(base + (u * UD + 32 * c) * type_bytes(CT));
        if (CODED && u == 0) ks[j] = __ldg(reinterpret_cast<const float2*>(p.k_scale + soff[j]));
      }
      return;
    }
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      const bool go = ((there >> j) & 1) && b * KB + 8 * j + g < k_end;
      const char* base = static_cast<const char*>(p.k) + off[j] * type_bytes(CT) + k_lane;
#pragma unroll
      for (int c = 0; c < UD / 32; ++c) {
        if (go && u * UD + 32 * c + 8 * t < p.head_dim) kr[j][c] = load8<CT>(base + (u * UD + 32 * c) * type_bytes(CT));
        else
#pragma unroll
          for (uint32_t& w : kr[j][c].w) w = 0;
      }
      if (CODED && u == 0) {
        ks[j] = make_float2(0.0f, 0.0f);
        if ((there >> j) & 1) ks[j] = __ldg(reinterpret_cast<const float2*>(p.k_scale + soff[j]));
      }
    }
  };
  auto load_v = [&](int b, int u) {
    if (whole && full_dim) {
#pragma unroll
      for (int j = 0; j < NG; ++j) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {  // keys 2 t, 2 t + 1 of the group
          const char* base = static_cast<const char*>(p.v) + off[j] * type_bytes(CT) + v_lane + (i ? row_bytes : 0);
#pragma unroll
          for (int c = 0; c < (UD + 63) / 64; ++c) vr[j / 2][2 * (j & 1) + i][c] = load8<CT>(base + (u * UD + 64 * c) * type_bytes(CT));
        }
        if (CODED && u == 0) vs[j] = __ldg(reinterpret_cast<const float2*>(p.v_scale + soff[j]));
      }
      return;
    }
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      const int key = b * KB + 8 * j + 2 * t;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bool go = ((there >> j) & 1) && key + i < k_end && key + i >= k_begin;  // (a key that no row sees is zero whatever its slot holds)
        const char* base = static_cast<const char*>(p.v) + off[j] * type_bytes(CT) + v_lane + (i ? row_bytes : 0);
#pragma unroll
        for (int c = 0; c < (UD + 63) / 64; ++c) {
          Raw8<CT>& to = vr[j / 2][2 * (j & 1) + i][c];
          if (go && u * UD + 64 * c + 8 * g < p.head_dim) to = load8<CT>(base + (u * UD + 64 * c) * type_bytes(CT));
          else
#pragma unroll
            for (uint32_t& w : to.w) w = 0;
        }
      }
      if (CODED && u == 0) {
        vs[j] = make_float2(0.0f, 0.0f);
        if ((there >> j) & 1) vs[j] = __ldg(reinterpret_cast<const float2*>(p.v_scale + soff[j]));
        if (key >= k_end || key < k_begin) vs[j].x = 0.0f;
        if (key + 1 >= k_end || key + 1 < k_begin) vs[j].y = 0.0f;
      }
    }
  };

  float v_unit = 0.0f;  // codes: the power of two that O's values are in
  if (b0 < b1) {
    look_up(window);
    take_window();
    place_pages(b0);
    load_k(b0, 0);
    load_v(b0, 0);
  }
  for (int b = b0; b < b1; ++b) {
    // ---- scores ----------------------------------------------------------------------------------------------------------------
    float sc[NG][4], sc_q[WIDE ? NG : 1][4], sc_k[WIDE ? NG : 1][4];  // (fp32: sums of the smaller products apart, for shorter chains of instructions)
    const unsigned here = there;
    const bool full = whole && b * KB >= all_lo && b * KB + KB <= all_hi;
    float2 ks_now[NG];
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      if constexpr (CODED) ks_now[j] = ks[j];
#pragma unroll
      for (int i = 0; i < 4; ++i) sc[j][i] = 0.0f;
      if constexpr (WIDE) {
#pragma unroll
        for (int i = 0; i < 4; ++i) sc_q[j][i] = sc_k[j][i] = 0.0f;
      }
    }
#pragma unroll
    for (int u = 0; u < NU; ++u) {
#pragma unroll
      for (int c = 0; c < UD / 32; ++c) {
        if constexpr (WIDE) {
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            const int step = (u * UD + 32 * c) / 8 + h;
            const uint4 qa = sq[step * 32 + lane], ql = sq[(S::Q_STEPS + step) * 32 + lane];
#pragma unroll
            for (int j = 0; j < NG; ++j) {
              uint32_t hi[2], lo[2];
#pragma unroll
              for (int i = 0; i < 2; ++i) split_tf32(__uint_as_float(kr[j][c].w[2 * h + i]), hi[i], lo[i]);
              mma_tf32(sc[j], qa, hi[0], hi[1]);
              mma_tf32(sc_q[j], ql, hi[0], hi[1]);
              mma_tf32(sc_k[j], qa, lo[0], lo[1]);
            }
          }
          continue;
        }
        uint4 qa[2], ql[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int step = (u * UD + 32 * c) / 16 + h;
          qa[h] = sq[step * 32 + lane];
          if constexpr (NQ == 2) ql[h] = sq[(S::Q_STEPS + step) * 32 + lane];
        }
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          uint32_t hi[4];
          to_pairs<CT>(kr[j][c], hi);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            mma16<BF>(sc[j], qa[h], hi[2 * h], hi[2 * h + 1]);
            if constexpr (NQ == 2) mma16<BF>(sc[j], ql[h], hi[2 * h], hi[2 * h + 1]);
          }
        }
      }
      if (u + 1 < NU) load_k(b, u + 1);
    }
    // the next block's keys are on their way while this one's values are used
    if constexpr (NU == 1) {
      if (b + 1 < b1) {
        place_pages(b + 1);
        load_k(b + 1, 0);
      }
    }
    // ---- running maximum and sum -----------------------------------------------------------------------------------------------------
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int j = 0; j < NG; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float v = (WIDE ? sc[j][i] + (sc_q[j][i] + sc_k[j][i]) : sc[j][i]) * c2[i >> 1];
        if constexpr (CODED) v *= (i & 1) ? ks_now[j].y : ks_now[j].x;
        if (!full) {
          const int key = b * KB + 8 * j + 2 * t + (i & 1);
          if (!(((here >> j) & 1) && key < lim_hi[i >> 1] && key >= lim_lo[i >> 1])) v = -INFINITY;
        }
        sc[j][i] = v;
        mx[i >> 1] = fmaxf(mx[i >> 1], v);
      }
    float alpha[2], base[2];
    bool raise = false;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
      const float mn = fmaxf(m[i], mx[i] - S::ROOM);
      raise = raise || mn > m[i];
      base[i] = mn == -INFINITY ? 0.0f : mn;  // (a row that has seen nothing yet)
      alpha[i] = ex2f(m[i] - base[i]);
      m[i] = mn;
      l[i] *= alpha[i];
    }
    // codes' scales move into the probabilities, which a power of two keeps near one: halves have little range
    float2 vf[NG];
    if constexpr (CODED) {
      float top = 0.0f;
#pragma unroll
      for (int j = 0; j < NG; ++j) top = fmaxf(top, fmaxf(fabsf(vs[j].x), fabsf(vs[j].y)));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e2 = min(240, max(14, static_cast<int>(__float_as_uint(top) >> 23)));
      const float unit = fmaxf(v_unit, __uint_as_float(static_cast<uint32_t>(e2) << 23));
      const float inv = __uint_as_float(0x7f000000u - __float_as_uint(unit));  // (a power of two's reciprocal)
      if (unit > v_unit) {
        raise = true;
        const float f = v_unit * inv;
        alpha[0] *= f, alpha[1] *= f;
        v_unit = unit;
      }
#pragma unroll
      for (int j = 0; j < NG; ++j) vf[j] = make_float2(vs[j].x * inv, vs[j].y * inv);
    }
    if (!S::FRESH && __any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int j = 0; j < DP / 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[j][i] *= alpha[i >> 1];
    }
    uint4 ph[KB / (WIDE ? 8 : 16)], pl[KB / (WIDE ? 8 : 16)];
#pragma unroll
    for (int k16 = 0; k16 < KB / 16; ++k16) {
      uint32_t hi[2][2], lo[2][2];  // [group of eight keys][row]
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int j = 2 * k16 + x;
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[i] = ex2f(sc[j][i] - base[i >> 1]);
          l[i >> 1] += e[i];
          if constexpr (CODED) e[i] *= (i & 1) ? vf[j].y : vf[j].x;
        }
        if constexpr (WIDE) {  // (keys 2 t and 2 t + 1 of the group are columns t and t + 4)
          split_tf32(e[0], ph[j].x, pl[j].x), split_tf32(e[2], ph[j].y, pl[j].y), split_tf32(e[1], ph[j].z, pl[j].z), split_tf32(e[3], ph[j].w, pl[j].w);
        } else if constexpr (NP == 2) {
          split2<BF>(e[0], e[1], hi[x][0], lo[x][0]);
          split2<BF>(e[2], e[3], hi[x][1], lo[x][1]);
        } else {
          hi[x][0] = pack2<BF>(e[0], e[1]);
          hi[x][1] = pack2<BF>(e[2], e[3]);
        }
      }
      if constexpr (!WIDE) ph[k16] = make_uint4(hi[0][0], hi[0][1], hi[1][0], hi[1][1]);
      if constexpr (!WIDE && NP == 2) pl[k16] = make_uint4(lo[0][0], lo[0][1], lo[1][0], lo[1][1]);
    }
    // ---- values ------------------------------------------------------------------------------------------------------------------------
#pragma unroll
    for (int u = 0; u < NU; ++u) {
#pragma unroll
      for (int c = 0; c < (UD + 63) / 64; ++c) {
        float acc[8][4];
        if constexpr (S::FRESH) {
#pragma unroll
          for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[n][i] = 0.0f;
        }
#pragma unroll
        for (int k16 = 0; k16 < KB / 16; ++k16) {
          if constexpr (WIDE) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {  // groups of eight keys
#pragma unroll
              for (int n = 0; n < 8; ++n) {
                uint32_t hi[2], lo[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) split_tf32(__uint_as_float(vr[k16][2 * x + i][c].w[n]), hi[i], lo[i]);
                mma_tf32(acc[n], ph[2 * k16 + x], hi[0], hi[1]);
                mma_tf32(acc[n], pl[2 * k16 + x], hi[0], hi[1]);
                mma_tf32(acc[n], ph[2 * k16 + x], lo[0], lo[1]);
              }
            }
            continue;
          }
          uint32_t h4[4][4];  // [this lane's four keys][pair of columns]
#pragma unroll
          for (int i = 0; i < 4; ++i) to_pairs<CT>(vr[k16][i][c], h4[i]);
#pragma unroll
          for (int n = 0; n < 8; ++n) {  // column tiles
            float(&to)[4] = S::FRESH ? acc[n] : o[(u * UD + 64 * c) / 8 + n];
            const uint32_t sel = (n & 1) ? 0x7632 : 0x5410;
            const uint32_t w0 = __byte_perm(h4[0][n / 2], h4[1][n / 2], sel), w1 = __byte_perm(h4[2][n / 2], h4[3][n / 2], sel);
            mma16<BF>(to, ph[k16], w0, w1);
            if constexpr (NP == 2) mma16<BF>(to, pl[k16], w0, w1);
          }
        }
        if constexpr (S::FRESH) {
#pragma unroll
          for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float& oo = o[(u * UD + 64 * c) / 8 + n][i];
              oo = fmaf(oo, alpha[i >> 1], acc[n][i]);
            }
        }
      }
      if constexpr (NU > 1) {
        if (u + 1 < NU) load_v(b, u + 1);
      }
    }
    if constexpr (NU > 1) {
      if (b + 1 < b1) {
        place_pages(b + 1);
        load_k(b + 1, 0);
      }
    }
    if (b + 1 < b1) load_v(b + 1, 0);
  }
  if constexpr (CODED) {
    const float f = v_unit;
#pragma unroll
    for (int j = 0; j < DP / 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[j][i] *= f;
  }

  // ---- warps, then the cluster's CTAs, meet: only the tile's rows --------------------------------------------------------------------
  const int rows = r_end - r0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    const int row = g + 8 * i;
    if (row < rows) {
      if (t == 0) sm[warp * PA_ROWS + row] = m[i], sl[warp * PA_ROWS + row] = l[i];
      float* w = so + (warp * PA_ROWS + row) * S::O_STRIDE;
#pragma unroll
      for (int j = 0; j < DP / 8; j += 4) {  // tile (c, j % 8) has columns 64 c + 16 t + j % 8 and 8 more
        const int d = (j / 8) * 64 + 16 * t + (j & 7);
        *reinterpret_cast<float4*>(w + d) = make_float4(o[j][2 * i], o[j + 1][2 * i], o[j + 2][2 * i], o[j + 3][2 * i]);
        *reinterpret_cast<float4*>(w + d + 8) = make_float4(o[j][2 * i + 1], o[j + 1][2 * i + 1], o[j + 2][2 * i + 1], o[j + 3][2 * i + 1]);
      }
    }
  }
  if (a.cluster > 1) {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  } else {
    __syncthreads();
  }
  // four columns of a row a thread, over all of the cluster's threads
  const int quads = p.head_dim / 4;
  for (int i = rank * PA_THREADS + threadIdx.x; i < rows * quads; i += a.cluster * PA_THREADS) {
    const int row = i / quads, d = 4 * (i - row * quads);
    float top = -INFINITY;
    for (int c = 0; c < a.cluster; ++c)
#pragma unroll
      for (int w = 0; w < PA_WARPS; ++w) top = fmaxf(top, ld_cluster(sm + w * PA_ROWS + row, c));
    const float base = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int c = 0; c < a.cluster; ++c) {
      float4 part[PA_WARPS];
      float f[PA_WARPS], s4[PA_WARPS];
#pragma unroll
      for (int w = 0; w < PA_WARPS; ++w) {
        f[w] = ld_cluster(sm + w * PA_ROWS + row, c);
        s4[w] = ld_cluster(sl + w * PA_ROWS + row, c);
        part[w] = ld_cluster4(so + (w * PA_ROWS + row) * S::O_STRIDE + d, c);
      }
#pragma unroll
      for (int w = 0; w < PA_WARPS; ++w) {
        const float e = ex2f(f[w] - base);
        sum = fmaf(s4[w], e, sum);
        v[0] = fmaf(part[w].x, e, v[0]), v[1] = fmaf(part[w].y, e, v[1]), v[2] = fmaf(part[w].z, e, v[2]), v[3] = fmaf(part[w].w, e, v[3]);
      }
    }
    if (a.splits > 1) {
      *reinterpret_cast<float4*>(a.part_o + (static_cast<long long>(part) * PA_ROWS + row) * p.head_dim + d) = make_float4(v[0], v[1], v[2], v[3]);
      if (d == 0) a.part_ml[static_cast<long long>(part) * PA_ROWS + row] = make_float2(top, sum);
    } else {
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      store_out4(a, q.row0, r0 + row, head, d, v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
      if (d == 0) store_lse(a, q.row0, r0 + row, head, top, sum);
    }
  }
  if (a.cluster > 1) {  // no CTA leaves while others read its shared memory
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  if (last) pdl_wait();
}

// The parts of a tile that several CTAs or clusters computed, in order; a warp a row (a block a row: 16 us more for 16 K rows of two parts).
__global__ void __launch_bounds__(128) paged_merge_kernel(const __grid_constant__ AttendArgs a) {
  const PagedView& p = a.p;
  const int at = static_cast<int>(blockIdx.x) * 4 + static_cast<int>(threadIdx.x >> 5), unit = at / a.part_rows, row = at % a.part_rows, lane = threadIdx.x & 31;
  int tile, head;
  PagedSeq q;
  if (a.chunks) {
    const ChunkUnit u = chunk_unit(a, unit);
    q = u.seq, tile = u.tile, head = u.head;
  } else {
    const int sh = unit / a.tiles;
    tile = unit % a.tiles, head = sh % p.kv_heads;
    q = paged_seq(p, sh / p.kv_heads);
  }
  const int r = tile * a.part_rows + row, n_rows = q.rows * a.group;
  if (r >= n_rows || (!a.chunks && n_rows > a.few)) return;
  const float2* ml = a.part_ml + static_cast<long long>(unit) * a.splits * a.part_rows + row;
  const float* po = a.part_o + (static_cast<long long>(unit) * a.splits * a.part_rows + row) * p.head_dim;
  float top = -INFINITY, sum = 0.0f;
  for (int c = 0; c < a.splits; ++c) top = fmaxf(top, ml[c * a.part_rows].x);
  const float base = top == -INFINITY ? 0.0f : top;
  for (int c = 0; c < a.splits; ++c) sum = fmaf(ml[c * a.part_rows].y, exp2f(ml[c * a.part_rows].x - base), sum);
  for (int d = lane; d < p.head_dim; d += 32) {
    float v = 0.0f;
    for (int c = 0; c < a.splits; ++c)
      v = fmaf(po[static_cast<long long>(c) * a.part_rows * p.head_dim + d], exp2f(ml[c * a.part_rows].x - base), v);
    store_out(a, q.row0, r, head, d, sum == 0.0f ? 0.0f : v / sum);
  }
  if (lane == 0) store_lse(a, q.row0, r, head, top, sum);
}

// How a call is shared out between the two kernels, and each one's tiles over CTAs.
struct Share {
  bool rows = true, chunks = false;  // which kernels run
  int few = 0x7fffffff;
  int tiles = 1, cluster = 1, splits = 1;   // row kernel
  int tc_splits = 1;
  long long units = 0, tc_units = 0;
  size_t bytes = 0, tc_bytes = 0;
};
// Up to how many rows of a head go to the row kernel.  Up to 4 x 8 K keys, 8 key heads of 128, here and by tcgen05: 32 rows 57 and 53 us in
// bfloat16, 47 and 78 over int8, 76 and 49 for fp32; 64 rows 111 and 54 us in bfloat16.  Codes cost tcgen05 a pass through registers and shared
// memory: 64 rows of 4 x up to 128 K e4m3 keys 686 and 1006 us, 64 x up to 4 K 348 and 416, 128 rows 620 and 443; not so heads over 128 (int8, 64
// rows 824 and 614) or fp32 queries (456 and 441), whose share here grows as well.
int few_rows(const AttendLaunch& a) {
  const bool codes = a.cache_type == MIMIR_B200_T_I8 || a.cache_type == MIMIR_B200_T_E4M3;
  return codes && a.type != MIMIR_B200_T_F32 && a.p.head_dim <= 128 ? 64 : 32;
}
Share share_out(const AttendLaunch& a) {
  Share r;
  const int group = a.heads / a.p.kv_heads;
  const long long most = static_cast<long long>(a.p.max_rows) * group;
  const int most_few = few_rows(a);
  const int keys = a.window > 0 && a.window < a.p.max_kv ? a.window : a.p.max_kv;  // (of a row; a chunk sees a little more)
  const size_t row_bytes = a.p.head_dim * sizeof(float) + sizeof(float2);
  if (tc_takes(a.cache_type, a.type, a.p.head_dim) && most > most_few) {
    r.chunks = true;
    // (one sequence: its rows are many, and so are those of one token of a large group; of several sequences some may have few)
    r.rows = a.p.n_seqs > 1 && group <= most_few;
    r.few = r.rows ? most_few : 0;
    const int per = tc_tile_rows(a.type, a.p.head_dim);
    // at most so many tiles: full ones, and one of each sequence of more than `few` rows that is not
    const long long all = static_cast<long long>(a.p.n_rows) * group, chunks = all / (r.few + 1) < a.p.n_seqs ? all / (r.few + 1) : a.p.n_seqs;
    const long long longest = a.p.n_seqs * ((most + per - 1) / per);
    r.tc_units = a.p.kv_heads * (all / per + chunks < longest ? all / per + chunks : longest);
    // Keys are split while SMs are idle and it pays: 1.25 us a key tile (of 128 elements), against a second launch and the parts written and read
    // at 3 TB/s.  512 tokens of 32 heads over 1 K keys 28 us whole, 44 in two; over 8 K 127 and 95; 64 tokens over 8 K 124 and, in eight, 34.
    auto time = [&](int splits) {
      const double tiles = static_cast<double>((keys + TC_KEYS - 1) / TC_KEYS) / splits;
      return 1.25 * tiles * a.p.head_dim / 128 + (splits > 1 ? 3.0 + 2e-6 / 3 * static_cast<double>(r.tc_units) * splits * per * row_bytes : 0.0);
    };
    while (r.tc_units * r.tc_splits * 2 <= ctx().sm_count && keys >= 2 * TC_KEYS * r.tc_splits && time(2 * r.tc_splits) < time(r.tc_splits)) r.tc_splits *= 2;
    if (r.tc_splits > 1) r.tc_bytes = static_cast<size_t>(r.tc_units) * r.tc_splits * per * row_bytes;
  }
  if (!r.rows) return r;
  // A cluster of up to eight CTAs meets through shared memory at no extra launch; beyond that (few tiles, long sequences) clusters
  // leave parts in the workspace for a second launch.  Clusters until there are as many CTAs as SMs: blocks cost a few us to start and meet.
  // 8 key heads of 128, 16 sequences of up to 4 K keys 61 us (up to three CTAs a slot: 78), of up to 1 K 18 (25), 32 of up to 4 K 90 (101), one of
  // 4 K 9.1 (single CTAs: 15).
  const long long few = r.chunks ? most_few : most;
  r.tiles = static_cast<int>((few + PA_ROWS - 1) / PA_ROWS);
  r.units = static_cast<long long>(a.p.n_seqs) * a.p.kv_heads * r.tiles;
  const long long slots = 2LL * ctx().sm_count;
  while (r.cluster < 8 && r.units * r.cluster < ctx().sm_count && keys >= 128 * 2 * r.cluster) r.cluster *= 2;
  // Parts: 512 keys a CTA or more while all CTAs find room at once, 2048 or more where that takes a second round (8 of 4 K keys 29 us in one, 41 in
  // two; 4 of 128 K e4m3 keys 243 and 206).
  while (r.units * r.cluster * r.splits < slots &&
         keys >= (r.units * r.cluster * r.splits * 2 <= slots ? 512 : 2048) * 2LL * r.cluster * r.splits)
    r.splits *= 2;
  if (r.splits > 1) r.bytes = static_cast<size_t>(r.units) * r.splits * PA_ROWS * row_bytes;
  return r;
}

template <int CT, int NQ, int NP, int DP>
int launch_rows_as(const AttendArgs& a, long long grid, cudaStream_t st) {
  using S = PagedShape<CT, NQ, NP, DP>;
  static PerDeviceOnce once;
  MB_TRY(once.run([]() -> int {
    MB_CUDA(cudaFuncSetAttribute(paged_attention_kernel<CT, NQ, NP, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
    return MIMIR_B200_OK;
  }));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(PA_THREADS);
  cfg.dynamicSmemBytes = S::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (a.cluster > 1) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(a.cluster);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
  }
  if (a.behind_chunks) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  MB_CUDA(cudaLaunchKernelEx(&cfg, paged_attention_kernel<CT, NQ, NP, DP>, a));
  count_launch();
  return MIMIR_B200_OK;
}
template <int CT, int NQ, int NP>
int launch_rows_dim(const AttendArgs& a, long long grid, cudaStream_t st) {
  if (a.p.head_dim <= 64) return launch_rows_as<CT, NQ, NP, 64>(a, grid, st);
  if (a.p.head_dim <= 128) return launch_rows_as<CT, NQ, NP, 128>(a, grid, st);
  return launch_rows_as<CT, NQ, NP, 256>(a, grid, st);
}
// Queries of fp32 are two terms; probabilities two for results of fp32 or half, one (11 bits) for bfloat16's 8.
template <int CT>
int launch_rows_type(const AttendArgs& a, long long grid, cudaStream_t st) {
  if (a.type == MIMIR_B200_T_F32) return launch_rows_dim<CT, 2, 2>(a, grid, st);
  if (a.type == MIMIR_B200_T_F16) return launch_rows_dim<CT, 1, 2>(a, grid, st);
  return launch_rows_dim<CT, 1, 1>(a, grid, st);
}

}  // namespace

size_t paged_attention_ws_bytes(const AttendLaunch& a) {
  const Share r = share_out(a);
  return r.bytes + r.tc_bytes;
}

namespace {
int launch_merge(const AttendArgs& a, long long units, cudaStream_t st) {
  paged_merge_kernel<<<static_cast<unsigned>(units * a.part_rows / 4), 128, 0, st>>>(a);
  MB_CUDA(cudaGetLastError());
  count_launch();
  return MIMIR_B200_OK;
}
}  // namespace

int launch_paged_attention(const AttendLaunch& l, cudaStream_t st) {
  const Share r = share_out(l);
  const size_t need = r.bytes + r.tc_bytes;
  if (need > 0 && (!l.ws || l.ws_bytes < need))
    return fail(MIMIR_B200_E_INVALID, "paged_attention: a workspace of %zu bytes is needed (paged_attention_workspace), got %zu", need, l.ws ? l.ws_bytes : 0);
  const long long grid = r.units * r.splits * r.cluster;
  if (grid > 0x7fffffffLL || r.units * PA_ROWS > 0x7fffffffLL || r.tc_units * r.tc_splits > 0x7fffffffLL)
    return fail(MIMIR_B200_E_INVALID, "paged_attention: too many rows and heads for one call");
  AttendArgs a = {};
  a.p = l.p;
  a.q = l.q, a.out = l.out, a.lse = l.lse;
  a.q_row = l.q_row, a.q_head = l.q_head, a.o_row = l.o_row, a.o_head = l.o_head;
  a.type = l.type, a.heads = l.heads, a.group = l.heads / l.p.kv_heads, a.causal = l.causal, a.window = l.window, a.scale = l.scale;
  a.few = r.few;
  a.err_word = ctx().dev_error_word;
  auto parts = [&](size_t offset, long long units, int splits, int rows) {
    a.splits = splits, a.part_rows = rows;
    a.part_o = reinterpret_cast<float*>(static_cast<char*>(l.ws) + offset);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + static_cast<size_t>(units) * splits * rows * l.p.head_dim);
  };
  AttendArgs chunks = a;
  if (r.chunks) {
    a.chunks = 1;
    parts(r.bytes, r.tc_units, r.tc_splits, tc_tile_rows(l.type, l.p.head_dim));
    chunks = a;
    MB_TRY(launch_paged_attention_tc(a, l.cache_type, r.tc_units * r.tc_splits, st));
  }
  if (!r.rows) return r.tc_splits > 1 ? launch_merge(chunks, r.tc_units, st) : MIMIR_B200_OK;
  a.tiles = r.tiles, a.cluster = r.cluster, a.chunks = 0, a.behind_chunks = r.chunks;
  parts(0, r.units, r.splits, PA_ROWS);
  switch (l.cache_type) {
    case MIMIR_B200_T_F32: MB_TRY((launch_rows_dim<MIMIR_B200_T_F32, 2, 2>(a, grid, st))); break;
    case MIMIR_B200_T_BF16: MB_TRY((launch_rows_dim<MIMIR_B200_T_BF16, 1, 2>(a, grid, st))); break;
    case MIMIR_B200_T_F16: MB_TRY(launch_rows_type<MIMIR_B200_T_F16>(a, grid, st)); break;
    case MIMIR_B200_T_I8: MB_TRY(launch_rows_type<MIMIR_B200_T_I8>(a, grid, st)); break;
    default: MB_TRY(launch_rows_type<MIMIR_B200_T_E4M3>(a, grid, st)); break;
  }
  if (r.tc_splits > 1) MB_TRY(launch_merge(chunks, r.tc_units, st));
  if (r.splits > 1) MB_TRY(launch_merge(a, r.units, st));
  return MIMIR_B200_OK;
}

}  // namespace mb
