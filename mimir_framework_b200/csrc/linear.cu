// linear.cu — rows times a weight matrix, with bias, activation and residual, and the gated pair of products: one tile of fp32 products a CTA.
#include "common.h"
#include "epilogue.cuh"
#include "layer.cuh"
#include "paged.cuh"

namespace mb {
namespace {

constexpr int LT = 32;  // rows, features and inputs of a tile

template <int T>
__device__ __forceinline__ float load1(const void* p, long long i) {
  if constexpr (T == MIMIR_B200_T_F16) return __half2float(static_cast<const __half*>(p)[i]);
  else if constexpr (T == MIMIR_B200_T_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  else if constexpr (T == MIMIR_B200_T_F32) return static_cast<const float*>(p)[i];
  else return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<const __nv_fp8_storage_t*>(p)[i], __NV_E4M3)));
}
__device__ __forceinline__ float load_as(const void* p, long long i, int type) {
  return type == MIMIR_B200_T_F32 ? load1<MIMIR_B200_T_F32>(p, i) : type == MIMIR_B200_T_F16 ? load1<MIMIR_B200_T_F16>(p, i) : load1<MIMIR_B200_T_BF16>(p, i);
}
__device__ __forceinline__ void store_as(void* p, long long i, int type, float v) {
  if (type == MIMIR_B200_T_F32) static_cast<float*>(p)[i] = v;
  else if (type == MIMIR_B200_T_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

template <int T, bool GATED>
__global__ void __launch_bounds__(LT* LT) linear_plain_kernel(const __grid_constant__ MimirLinear a) {
  __shared__ float xs[LT][LT + 1], ws[LT][LT + 1], us[GATED ? LT : 1][LT + 1];
  const int tx = threadIdx.x % LT, ty = threadIdx.x / LT;
  const long long row = static_cast<long long>(blockIdx.y) * LT + ty;
  const int col = blockIdx.x * LT + tx, wrow = blockIdx.x * LT + ty;
  float z = 0.0f, u = 0.0f;
  for (int k0 = 0; k0 < a.n_in; k0 += LT) {
    const int k = k0 + tx;
    xs[ty][tx] = row < a.rows && k < a.n_in ? load1<T>(a.x, row * a.x_stride + k) : 0.0f;
    ws[ty][tx] = wrow < a.n_out && k < a.n_in ? load1<T>(a.w, wrow * a.w_stride + k) : 0.0f;
    if (GATED) us[ty][tx] = wrow < a.n_out && k < a.n_in ? load1<T>(a.up, wrow * a.up_stride + k) : 0.0f;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < LT; ++i) {
      z = fmaf(xs[ty][i], ws[tx][i], z);
      if (GATED) u = fmaf(xs[ty][i], us[tx][i], u);
    }
    __syncthreads();
  }
  if (row >= a.rows || col >= a.n_out) return;
  if (T == MIMIR_B200_T_E4M3) {
    z = z * a.x_scale[row] * a.w_scale[col];
    if (GATED) u = u * a.x_scale[row] * a.up_scale[col];
  }
  if (a.bias) z += a.bias[col];
  z = apply_act(z, a.activation);
  if (GATED) z *= a.up_bias ? u + a.up_bias[col] : u;
  else if (a.residual) z += load_as(a.residual, row * a.residual_stride + col, a.out_type);
  store_as(a.out, row * a.out_stride + col, a.out_type, z);
}

}  // namespace

int launch_linear(const MimirLinear& a, bool gated, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>((a.n_out + LT - 1) / LT), static_cast<unsigned>((a.rows + LT - 1) / LT));
  auto run = [&](auto kern) { kern<<<grid, LT * LT, 0, st>>>(a); };
  if (a.type == MIMIR_B200_T_F16) gated ? run(linear_plain_kernel<MIMIR_B200_T_F16, true>) : run(linear_plain_kernel<MIMIR_B200_T_F16, false>);
  else if (a.type == MIMIR_B200_T_BF16) gated ? run(linear_plain_kernel<MIMIR_B200_T_BF16, true>) : run(linear_plain_kernel<MIMIR_B200_T_BF16, false>);
  else gated ? run(linear_plain_kernel<MIMIR_B200_T_E4M3, true>) : run(linear_plain_kernel<MIMIR_B200_T_E4M3, false>);
  MB_CUDA(cudaGetLastError());
  count_launch();
  return MIMIR_B200_OK;
}

}  // namespace mb
