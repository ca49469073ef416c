// paged_attention.cuh — arguments and result stores of the paged attention kernels.
#pragma once

#include "paged.cuh"

namespace mb {

struct AttendArgs {
  PagedView p;
  const void* q;
  void* out;
  float* lse;                              // natural logarithm of the row's sum of exponentials, or null
  long long q_row, q_head, o_row, o_head;  // elements
  int type, heads, group, causal, window;
  float scale;
  int few;                                 // (token, head) rows of a sequence and key head: up to so many are the row kernel's
  int tiles, cluster, splits;              // of the rows of a sequence; CTAs and clusters that share a tile's keys
  int part_rows;                           // rows of a tile
  int chunks;                              // tiles of the sequences with more than `few` rows only, numbered by chunk_unit()
  int behind_chunks;                       // the row kernel: launched behind the chunks' kernel, with which it shares nothing
  float* part_o;                           // [unit][split][part_rows][head_dim], [unit][split][part_rows] (max, sum): splits > 1
  float2* part_ml;
  int* err_word;
};
// paged_attention_tc.cu: chunks of many rows; not fp32 caches, nor fp32 queries of heads over 128
constexpr int TC_KEYS = 128, TC_ROWS = 128;
inline bool tc_takes(int cache_type, int type, int head_dim) { return cache_type != MIMIR_B200_T_F32 && (type != MIMIR_B200_T_F32 || head_dim <= 128); }
inline int tc_tile_rows(int type, int head_dim) { return head_dim <= 128 && type != MIMIR_B200_T_F32 ? 2 * TC_ROWS : TC_ROWS; }
int launch_paged_attention_tc(const AttendArgs& a, int cache_type, long long grid, cudaStream_t st);

namespace {
// The `unit`-th tile of the sequences that have more than `few` rows, by a whole warp: their tiles of the first key head, the last first (its
// rows see the most keys), then the next head's, then the next sequence's.  A grid over sequences x the longest one's tiles had mostly empty
// blocks in a batch of one chunk and many single tokens (2048 new tokens and 31 single ones: 8192 blocks, 306 us in all; so numbered 512, 248).
struct ChunkUnit {
  PagedSeq seq;
  int s = -1, head = 0, tile = 0;
};
__device__ __forceinline__ ChunkUnit chunk_unit(const AttendArgs& a, int unit) {
  ChunkUnit u;
  const int lane = threadIdx.x & 31;
  for (int first = 0; first < a.p.n_seqs; first += 32) {
    PagedSeq q;
    if (first + lane < a.p.n_seqs) q = paged_seq(a.p, first + lane);
    const int rows = q.rows * a.group, tiles = rows > a.few ? (rows + a.part_rows - 1) / a.part_rows : 0;
    int sum = tiles * a.p.kv_heads;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int v = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += v;
    }
    const uint32_t behind = __ballot_sync(0xffffffffu, unit < sum);
    if (behind) {
      const int at = __ffs(behind) - 1, n = __shfl_sync(0xffffffffu, tiles, at), rest = unit - __shfl_sync(0xffffffffu, sum, at) + n * a.p.kv_heads;
      u.seq.row0 = __shfl_sync(0xffffffffu, q.row0, at);
      u.seq.rows = __shfl_sync(0xffffffffu, q.rows, at);
      u.seq.kv = __shfl_sync(0xffffffffu, q.kv, at);
      u.s = first + at, u.head = rest / n, u.tile = n - 1 - rest % n;
      return u;
    }
    unit -= __shfl_sync(0xffffffffu, sum, 31);
  }
  return u;
}

__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
  if constexpr (BF) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <bool BF>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (BF) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <bool BF>
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = pack2<BF>(x, y);
  const float2 h = unpack2<BF>(hi);
  lo = pack2<BF>(x - h.x, y - h.y);
}

// eight elements of a cache of 16 or 8 bits as four pairs in the tensor type
template <int CT>
__device__ __forceinline__ void to_pairs(const Raw8<CT>& r, uint32_t (&hi)[4]) {
  if constexpr (CT == MIMIR_B200_T_I8) {
    // 0x6400 | (code + 128) is 1024 + 128 + code as a half
    const __half2 off = __floats2half2_rn(1152.0f, 1152.0f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t b = r.w[i / 2] ^ 0x80808080u;
      const uint32_t w = __byte_perm(b, 0x64646464u, (i & 1) ? 0x4342 : 0x4140);
      const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&w), off);
      hi[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  } else if constexpr (CT == MIMIR_B200_T_E4M3) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(hi[2 * i]), "=r"(hi[2 * i + 1]) : "r"(r.w[i]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) hi[i] = r.w[i];
  }
}

__device__ __forceinline__ void store_out(const AttendArgs& a, int row0, int r, int kv_head, int d, float v) {
  const int tok = r / a.group, h = kv_head * a.group + r - tok * a.group;
  const long long at = (row0 + tok) * a.o_row + h * a.o_head + d;
  if (a.type == MIMIR_B200_T_F32) static_cast<float*>(a.out)[at] = v;
  else if (a.type == MIMIR_B200_T_F16) static_cast<__half*>(a.out)[at] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v);
}
// columns d .. d + 3
__device__ __forceinline__ void store_out4(const AttendArgs& a, int row0, int r, int kv_head, int d, float v0, float v1, float v2, float v3) {
  const int tok = r / a.group, h = kv_head * a.group + r - tok * a.group;
  const long long at = (row0 + tok) * a.o_row + h * a.o_head + d;
  if (a.type == MIMIR_B200_T_F32) *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = make_float4(v0, v1, v2, v3);
  else if (a.type == MIMIR_B200_T_F16) *reinterpret_cast<uint2*>(static_cast<__half*>(a.out) + at) = make_uint2(pack2<false>(v0, v1), pack2<false>(v2, v3));
  else *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + at) = make_uint2(pack2<true>(v0, v1), pack2<true>(v2, v3));
}
// top is in base two; a row that saw no key has -infinity
__device__ __forceinline__ void store_lse(const AttendArgs& a, int row0, int r, int kv_head, float top, float sum) {
  if (!a.lse) return;
  const int tok = r / a.group, h = kv_head * a.group + r - tok * a.group;
  a.lse[static_cast<long long>(row0 + tok) * a.heads + h] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
}

}  // namespace
}  // namespace mb
