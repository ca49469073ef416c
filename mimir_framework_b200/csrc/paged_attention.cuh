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
  int part_rows, last_first;               // rows of a tile; tiles are numbered from the last
  int behind_chunks;                       // the row kernel: launched behind the chunks' kernel, with which it shares nothing
  float* part_o;                           // [unit][split][part_rows][head_dim], [unit][split][part_rows] (max, sum): splits > 1
  float2* part_ml;
  int* err_word;
};
// paged_attention_tc.cu: chunks of many rows; not fp32 caches, nor fp32 queries of heads over 128
constexpr int TC_KEYS = 128, TC_ROWS = 128;
inline bool tc_takes(int cache_type, int type, int head_dim) { return cache_type != MIMIR_B200_T_F32 && (type != MIMIR_B200_T_F32 || head_dim <= 128); }
inline int tc_tile_rows(int type, int head_dim) { return head_dim <= 128 && type != MIMIR_B200_T_F32 ? 2 * TC_ROWS : TC_ROWS; }
int launch_paged_attention_tc(const AttendArgs& a, int cache_type, cudaStream_t st);

namespace {

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

// eight elements of a cache type as four pairs in the tensor type (and, of fp32, what those leave in a second four)
template <int CT>
__device__ __forceinline__ void to_pairs(const Raw8<CT>& r, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
  if constexpr (CT == MIMIR_B200_T_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) split2<false>(__uint_as_float(r.w[2 * i]), __uint_as_float(r.w[2 * i + 1]), hi[i], lo[i]);
  } else if constexpr (CT == MIMIR_B200_T_I8) {
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
