// linear.cuh — what the two kernels of the serving group's products share: rows times a weight matrix on tcgen05 with both operands K-major,
// as they lie in memory.
//
//   z[m][n] = sum_k x[m][k] w[n][k]  (times x_scale[m] w_scale[n] for E4M3)  + bias[n],    out = act(z) + residual,  or  act(z) * z_up
//
// A K block is 128 bytes of every operand row (64 values of 16 bits, 128 of 8), the span of the shared-memory swizzle; four instructions of 32
// bytes each take it.  What differs between the operand types is the instruction's kind and format alone.
#pragma once

#include "common.h"
#include "epilogue.cuh"
#include "layer.cuh"
#include "paged.cuh"
#include "sm100_ptx.cuh"

namespace mb {

constexpr int LIN_BLOCK = 128;   // bytes of a row in a K block
constexpr int LIN_W_BOX = 64;    // weight rows of a TMA box
// How much is added up in the tensor core before the sum is taken out and added rounded, since an instruction truncates, by up to 2^-22 of the magnitudes:
// for results of F32 256 inputs (2^-18; E4M3 2^-19), of 16 bits 96 K blocks, 384 instructions (2^-13.4, a fifth of fp16's half step, at worst; a sum
// whose terms have either sign loses some 2^-17 of itself).
// F32, operands of bfloat16: 2.3e-7 of the result off from 256 inputs on (plain fp32 sums of 256 inputs 1.1e-7, of 4 096 6.1e-7).  With 128 inputs it would be
// 1.2e-7, and 2 048 x 4 096 x 4 096 take 70 us instead of 58, 4 096 x 4 096 x 4 096 of E4M3, which loses nothing (4e-8 either way), 103 instead of 75.
// 16 bits: with 16 blocks products of 2 048 rows took 3 to 5 % longer, in 8 bits 6 to 12 %; with 96 only those of more inputs do, 1 to 3 % (with 64 also
// rows off their boundary, where the results are the bound: 3 040 x 4 162 x 2 190 with residual 8 %).
constexpr int LIN_CHUNK_F32 = 256, LIN_CHUNK_BLOCKS = 96;
static_assert(LIN_CHUNK_F32 % LIN_BLOCK == 0, "a sum is one K block at least, whatever the type");

// (Scales and biases are read by load_float, behind pdl_wait: the norm that makes the scales may be the kernel before, still at work when this one starts,
// and a load that goes by memory which does not change while the kernel runs has no claim to see them.)
struct LinearParams {
  const float* x_scale;
  const float* w_scale;
  const float* up_scale;
  const float* bias;
  const float* up_bias;
  const char* residual;
  char* out;
  long long residual_row, out_row;  // bytes
  int rows, n_out, out_type, act;
  int kblocks, chunk;               // K blocks of a product, and at most of a sum in tensor memory
  uint32_t formats;                 // instruction descriptor: operand formats
  bool vec_out, vec_res;            // result, residual: all rows on 16 bytes
  int* err_word;
};

// K blocks of a product, and of a sum in tensor memory at most
inline int linear_kblocks(const MimirLinear& a) { return static_cast<int>((static_cast<long long>(a.n_in) * type_bytes(a.type) + LIN_BLOCK - 1) / LIN_BLOCK); }
inline int linear_chunk(const MimirLinear& a) { return a.out_type == MIMIR_B200_T_F32 ? LIN_CHUNK_F32 * type_bytes(a.type) / LIN_BLOCK : LIN_CHUNK_BLOCKS; }

// linear_tiles.cu (many rows): tiles of 256 rows x 256 features; linear_rows.cu (few): 128 features and up to 256 rows
double linear_tiles_us(const MimirLinear& a, bool gated);
int launch_linear_tiles(const MimirLinear& a, const LinearParams& p, bool gated, cudaStream_t st);
double linear_rows_us(const MimirLinear& a, bool gated);
int launch_linear_rows(const MimirLinear& a, const LinearParams& p, bool gated, cudaStream_t st);
// tensor map of an operand: boxes of 128 bytes x `box_rows` rows, 128-byte swizzle, zeros beyond its rows and inputs
int make_operand_map(CUtensorMap* map, const void* base, int type, long long rows, int n_in, long long stride, int box_rows);
// of a result whose rows are on 16 bytes: boxes of 64 bytes x 32 rows, 64-byte swizzle
int make_result_map(CUtensorMap* map, const void* base, int type, long long rows, int n_out, long long stride);

namespace {

__device__ __forceinline__ float load_float(const float* p) {
  float v;
  asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1)
               : "memory");
}
// into L2
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* map, int c0, int c1) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1) : "memory");
}
// into this CTA's shared memory, counted on a barrier of the pair's
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, uint32_t bar_cluster_addr, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_cluster_addr), "r"(c0), "r"(c1)
               : "memory");
}
// Arrives in a CTA of the cluster.  What it orders is tensor memory, by the fences on both sides; a release at the cluster's scope would wait for every
// store of the thread (0.6 us a tile).
__device__ __forceinline__ void mbar_arrive_remote(uint32_t bar_cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster_addr) : "memory");
}
// 8-bit floats: 32 values of K an instruction
__device__ __forceinline__ void umma_f8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_f8_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// An instruction descriptor without its operand formats (LinearParams::formats): fp32 sums, both operands K-major
__host__ __device__ constexpr uint32_t linear_idesc(int m, int n) {
  return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// not a number stays one
__device__ __forceinline__ float relu_nan(float x) {
  float y;
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(y) : "f"(x));
  return y;
}
// 1 / (1 + 2^t): an exponential of 2^-22, a reciprocal of 2^-23 and an addition; below 2^-126 zero.  With d: 2^t (1 + d) for a small d, t up to 126.9
__device__ __forceinline__ float exp2_fast(float t) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  return e;
}
__device__ __forceinline__ float reciprocal_fast(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float logistic(float t) { return reciprocal_fast(1.0f + exp2_fast(t)); }
__device__ __forceinline__ float logistic(float t, float d) {
  const float e = exp2_fast(t);
  return reciprocal_fast(1.0f + fmaf(e, d, e));
}
// 1 / (1 + exp(-x)).  Rounding t alone would cost |x| 2^-24 of the exponential, so what it loses goes back in, as in silu2 (epilogue.cuh).
__device__ __forceinline__ float sigmoid_fast(float x) {
  const float n = x > 64.0f ? -64.0f : -x, t = fminf(n * 1.44269504f, 126.9f);
  return logistic(t, fmaf(t, 1.904654e-9f, fmaf(t, -0.693147182f, n)));
}
// GELU of two values as gelu_ref has it, x / (1 + exp(-2u)), for results of F32: the exponent -2u log2 e = C x (1 + K x^2) is some 460 where the result
// is about to vanish, and each of its roundings would cost as many units of the exponential, so every product's rest is kept (by fused
// multiply-adds) and put back in.  (4 096 x 1 024 x 4 096 57 us; with gelu_ref, 1e-6 of the value off at x = -5, 49.)
__device__ __forceinline__ void gelu2_f32(float& x0, float& x1) {
  // (the exponential is 0 or beyond fp32 from 16 on; not a number comes back in with the last product)
  const float a0 = fminf(fmaxf(x0, -16.0f), 16.0f), a1 = fminf(fmaxf(x1, -16.0f), 16.0f);
  auto both = [](float v) { return pack2(v, v); };
  const unsigned long long a = pack2(a0, a1), ns = mul2(a, pack2(-a0, -a1)), s_rest = fma2(a, a, ns);  // ns: -x^2
  const unsigned long long nq = fma2(both(0.044715f), ns, both(-1.0f));                                // -(1 + K x^2)
  unsigned long long q_rest = fma2(both(-0.044715f), ns, add2(nq, both(1.0f)));
  q_rest = fma2(both(0.044715f), s_rest, fma2(both(-1.5461444e-9f), ns, q_rest));
  const unsigned long long h = mul2(a, both(-2.3022082f)), nh = mul2(a, both(2.3022082f));             // C x
  const unsigned long long nh_rest = fma2(a, both(1.2948402e-8f), fma2(a, both(2.3022082f), h));
  const unsigned long long nt = mul2(h, nq);                                                           // -C x (1 + K x^2)
  const unsigned long long d = mul2(fma2(nh_rest, nq, fma2(h, q_rest, fma2(nh, nq, nt))), both(0.693147182f));
  float t0, t1, r0, r1;
  unpack2(nt, t0, t1);
  const unsigned long long e = pack2(exp2_fast(fminf(-t0, 126.9f)), exp2_fast(fminf(-t1, 126.9f)));
  unpack2(add2(fma2(e, d, e), both(1.0f)), r0, r1);
  unpack2(mul2(pack2(x0, x1), pack2(reciprocal_fast(r0), reciprocal_fast(r1))), x0, x1);
}
// tanh |x| = 1 - 2 / (1 + exp(2 |x|)), from 1/2 on, where the difference loses a bit; below its series x - x^3 / 3 + 2 x^5 / 15 - ... (next term 1e-7 of the
// value at 1/2).  (tanhf, called for each element: 3 000 x 192 x 5 800 74 us, so 25.)
__device__ __forceinline__ float tanh_fast(float x) {
  const float a = fabsf(x), s = x * x;
  float p = 3.5921281e-3f;            // 21844 / 6081075
  p = fmaf(p, s, -8.8632355e-3f);     // 1382 / 155925
  p = fmaf(p, s, 2.1869488e-2f);      // 62 / 2835
  p = fmaf(p, s, -5.3968254e-2f);     // 17 / 315
  p = fmaf(p, s, 1.3333333e-1f);      // 2 / 15
  p = fmaf(p, s, -3.3333333e-1f);     // 1 / 3
  const float small = fmaf(x * s, p, x), large = fmaf(-2.0f, logistic(a * 2.885390082f), 1.0f);
  return a < 0.5f ? small : copysignf(large, x);
}
// Within 10 units of 2^-24 of its value for results of F32; GELU of 16 bits within its exponent's |2u| 2^-22 besides.
template <int N>
__device__ __forceinline__ void activate(float (&v)[N], int act, int out_type) {
  switch (act) {
    case -1: break;
    case MIMIR_B200_ELT_GELU:
      if (out_type == MIMIR_B200_T_F32) {
#pragma unroll
        for (int j = 0; j < N; j += 2) gelu2_f32(v[j], v[j + 1]);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = gelu_ref(v[j]);
      }
      break;
    case MIMIR_B200_ELT_SILU:
#pragma unroll
      for (int j = 0; j < N; j += 2) silu2(v[j], v[j + 1]);
      break;
    case MIMIR_B200_ELT_RELU:
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = relu_nan(v[j]);
      break;
    case MIMIR_B200_ELT_TANH:
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = tanh_fast(v[j]);
      break;
    default:
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = sigmoid_fast(v[j]);
  }
}

__device__ __forceinline__ float load_typed(const char* p, int type) {
  if (type == MIMIR_B200_T_F32) return *reinterpret_cast<const float*>(p);
  if (type == MIMIR_B200_T_F16) return __half2float(*reinterpret_cast<const __half*>(p));
  return __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(p));
}
__device__ __forceinline__ void store_typed(char* p, int type, float v) {
  if (type == MIMIR_B200_T_F32) *reinterpret_cast<float*>(p) = v;
  else if (type == MIMIR_B200_T_F16) *reinterpret_cast<__half*>(p) = __float2half_rn(v);
  else *reinterpret_cast<__nv_bfloat16*>(p) = __float2bfloat16_rn(v);
}
// Eight neighbouring values, `left` of them there; vec: all, on 16 bytes
__device__ __forceinline__ void store_eight(char* p, int type, bool vec, int left, const float (&v)[8]) {
  if (vec) {
    if (type == MIMIR_B200_T_F32) store8<MIMIR_B200_T_F32>(p, pack8<MIMIR_B200_T_F32>(v));
    else if (type == MIMIR_B200_T_F16) store8<MIMIR_B200_T_F16>(p, pack8<MIMIR_B200_T_F16>(v));
    else store8<MIMIR_B200_T_BF16>(p, pack8<MIMIR_B200_T_BF16>(v));
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < left) store_typed(p + j * type_bytes(type), type, v[j]);
}

}  // namespace
}  // namespace mb
