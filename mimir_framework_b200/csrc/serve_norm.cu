// serve_norm.cu — rows between a layer's products: residual addition, root-mean-square norm, a narrower type.
//
//   s = x + residual,  v = s / sqrt(mean(s^2) + eps) * gamma,  y = v, or codes of 8 bits and their scale
//
// One pass: a row lies in the registers of the threads that share it (eight elements at a time, so that loads and stores are 16 bytes), its
// sum of squares and, for codes, its largest magnitude are each one meeting of these threads.  Statistics are fp32.  Codes are those
// of an IEEE division by the scale, as in the cache.
#include "common.h"
#include "launch.cuh"
#include "layer.cuh"
#include "paged.cuh"

namespace mb {
namespace {

constexpr int NR_WARP_THREADS = 128;  // of a CTA whose warps have a row each

struct NormParams {
  const char* x;
  const char* residual;
  char* sum;
  const float* gamma;
  char* y;
  float* y_scale;
  long long x_row, residual_row, sum_row, y_row;  // bytes
  int rows, n, norm, early;
  bool x_vec, residual_vec, sum_vec, gamma_vec, y_vec;  // rows start on 16 bytes
  float eps;
};

// Eight elements from column `col` on, those from n on zero.
template <int T>
__device__ __forceinline__ Raw8<T> row_load8(const char* row, int col, int n, bool vec) {
  const char* p = row + static_cast<long long>(col) * type_bytes(T);
  if (vec && col + 8 <= n) return load8<T>(p);
  Raw8<T> r;
#pragma unroll
  for (uint32_t& w : r.w) w = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (col + e >= n) break;
    if constexpr (type_bytes(T) == 4) r.w[e] = reinterpret_cast<const uint32_t*>(p)[e];
    else r.w[e / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[e]) << (16 * (e & 1));
  }
  return r;
}
template <int T>
__device__ __forceinline__ void row_store8(char* row, int col, int n, bool vec, const Raw8<T>& r) {
  char* p = row + static_cast<long long>(col) * type_bytes(T);
  if (vec && col + 8 <= n) {
    store8<T>(p, r);
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (col + e >= n) break;
    if constexpr (type_bytes(T) == 4) reinterpret_cast<uint32_t*>(p)[e] = r.w[e];
    else if constexpr (type_bytes(T) == 2) reinterpret_cast<uint16_t*>(p)[e] = static_cast<uint16_t>(r.w[e / 2] >> (16 * (e & 1)));
    else reinterpret_cast<uint8_t*>(p)[e] = static_cast<uint8_t>(r.w[e / 4] >> (8 * (e & 3)));
  }
}

// A number of each thread of a row, joined; every thread has the result (`buf`: 32 words of the CTA's, of one meeting).
template <bool WARP, bool MAX>
__device__ __forceinline__ float meet(float v, float* buf) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const float w = __shfl_xor_sync(0xffffffffu, v, o);
    v = MAX ? fmaxf(v, w) : v + w;
  }
  if constexpr (WARP) return v;
  const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
  if (warps == 1) return v;
  if (lane == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  v = lane < warps ? buf[lane] : 0.0f;  // (sums and magnitudes: zero changes neither)
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const float w = __shfl_xor_sync(0xffffffffu, v, o);
    v = MAX ? fmaxf(v, w) : v + w;
  }
  return v;
}

// V vectors of eight elements a thread; WARP: a row to a warp, else to the CTA.
template <int TX, int TY, int V, bool WARP>
__global__ void __launch_bounds__(WARP ? NR_WARP_THREADS : 1024) norm_rows_serve_kernel(const __grid_constant__ NormParams p) {
  __shared__ float buf[2][32];
  pdl_early_if(p.early);
  pdl_wait();
  const int row = WARP ? blockIdx.x * (NR_WARP_THREADS / 32) + (threadIdx.x >> 5) : blockIdx.x;
  if (WARP && row >= p.rows) return;
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x, step = (WARP ? 32 : blockDim.x) * 8;
  const char* x = p.x + row * p.x_row;
  Raw8<TX> raw[V], res[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int col = v * step + t * 8;
    raw[v] = row_load8<TX>(x, col, p.n, p.x_vec);
    if (p.residual) res[v] = row_load8<TX>(p.residual + row * p.residual_row, col, p.n, p.residual_vec);
  }
  float f[V][8];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    unpack8<TX>(raw[v], f[v]);
    if (p.residual) {
      float g[8];
      unpack8<TX>(res[v], g);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[v][e] += g[e];
    }
  }
  if (p.norm) {
    float q = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float a = 0.0f, b = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; e += 2) a = fmaf(f[v][e], f[v][e], a), b = fmaf(f[v][e + 1], f[v][e + 1], b);
      q += a + b;
    }
    q = meet<WARP, false>(q, buf[0]);
    if (p.sum) {
#pragma unroll
      for (int v = 0; v < V; ++v) row_store8<TX>(p.sum + row * p.sum_row, v * step + t * 8, p.n, p.sum_vec, pack8<TX>(f[v]));
    }
    const float mean = __fdiv_rn(q, static_cast<float>(p.n)) + p.eps;
    float r = __frsqrt_rn(mean);
    if (!(q < INFINITY) || mean < 0x1p-100f) {
      // squares beyond fp32's range (or below it, next to no eps): once more with the row's largest near one
      float top = 0.0f, rest = 0.0f;
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fabsf(f[v][e]) > top || f[v][e] != f[v][e] ? fabsf(f[v][e]) : top;
      if (!(top < INFINITY)) top = INFINITY;  // (not a number is as good as infinite here)
      top = meet<WARP, true>(top, buf[1]);
      if (top > 0.0f && top < INFINITY) {
        const int k = max(-100, min(126, ilogbf(top)));
        const float down = scalbnf(1.0f, -k);
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            f[v][e] *= down;
            rest = fmaf(f[v][e], f[v][e], rest);
          }
        r = __frsqrt_rn(__fdiv_rn(meet<WARP, false>(rest, buf[0]), static_cast<float>(p.n)) + p.eps * down * down);
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int col = v * step + t * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) f[v][e] *= r;
      if (p.gamma) {
        float g[8];
        unpack8<MIMIR_B200_T_F32>(row_load8<MIMIR_B200_T_F32>(reinterpret_cast<const char*>(p.gamma), col, p.n, p.gamma_vec), g);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[v][e] = col + e < p.n ? f[v][e] * g[e] : 0.0f;
      }
    }
  } else if (p.sum) {
#pragma unroll
    for (int v = 0; v < V; ++v) row_store8<TX>(p.sum + row * p.sum_row, v * step + t * 8, p.n, p.sum_vec, pack8<TX>(f[v]));
  }
  float scale = 0.0f;
  if constexpr (TY == MIMIR_B200_T_E4M3) {
    float top = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (fabsf(f[v][e]) < INFINITY) top = fmaxf(top, fabsf(f[v][e]));
    scale = __fmul_rn(meet<WARP, true>(top, buf[1]), 1.0f / 448.0f);
    if (t == 0) p.y_scale[row] = scale;
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int col = v * step + t * 8;
    if (col >= p.n) break;
    if constexpr (TY == MIMIR_B200_T_E4M3) {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[v][e] = scale > 0.0f ? __fdiv_rn(f[v][e], scale) : 0.0f;
    }
    row_store8<TY>(p.y + row * p.y_row, col, p.n, p.y_vec, pack8<TY>(f[v]));
  }
}

template <int TX, int TY, int V, bool WARP>
int launch_as(const NormParams& p, int threads, cudaStream_t st) {
  const unsigned grid = WARP ? (static_cast<unsigned>(p.rows) + NR_WARP_THREADS / 32 - 1) / (NR_WARP_THREADS / 32) : static_cast<unsigned>(p.rows);
  NormParams q = p;
  q.early = pdl_small_grid(grid);
  MB_TRY(launch_pdl(norm_rows_serve_kernel<TX, TY, V, WARP>, dim3(grid), dim3(static_cast<unsigned>(threads)), 0, st, 1, q));
  count_launch();
  return MIMIR_B200_OK;
}
template <int TX, int TY>
int launch_rows(const NormParams& p, cudaStream_t st) {
  const int vectors = (p.n + 7) / 8;
  if (vectors <= 32) return launch_as<TX, TY, 1, true>(p, NR_WARP_THREADS, st);
  if (vectors <= 64) return launch_as<TX, TY, 2, true>(p, NR_WARP_THREADS, st);
  if (vectors <= 128) return launch_as<TX, TY, 4, true>(p, NR_WARP_THREADS, st);
  const int v = vectors <= 1024 ? 2 : 4;
  const int threads = round_up((vectors + v - 1) / v, 32);
  return v == 2 ? launch_as<TX, TY, 2, false>(p, threads, st) : launch_as<TX, TY, 4, false>(p, threads, st);
}
template <int TX>
int launch_to(const NormParams& p, int y_type, cudaStream_t st) {
  switch (y_type) {
    case MIMIR_B200_T_F32: return launch_rows<TX, MIMIR_B200_T_F32>(p, st);
    case MIMIR_B200_T_F16: return launch_rows<TX, MIMIR_B200_T_F16>(p, st);
    case MIMIR_B200_T_BF16: return launch_rows<TX, MIMIR_B200_T_BF16>(p, st);
    default: return launch_rows<TX, MIMIR_B200_T_E4M3>(p, st);
  }
}

bool vectors_at(const void* p, long long row_bytes, int vector_bytes) {
  return reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(vector_bytes) == 0 && row_bytes % vector_bytes == 0;
}

}  // namespace

int launch_norm_rows(const MimirNormRows& a, cudaStream_t st) {
  NormParams p = {};
  const int xs = type_bytes(a.type), ys = type_bytes(a.y_type);
  p.x = static_cast<const char*>(a.x), p.residual = static_cast<const char*>(a.residual), p.sum = static_cast<char*>(a.sum);
  p.gamma = a.gamma, p.y = static_cast<char*>(a.y), p.y_scale = a.y_scale;
  p.x_row = a.x_stride * xs, p.residual_row = a.residual_stride * xs, p.sum_row = a.sum_stride * xs, p.y_row = a.y_stride * ys;
  p.rows = a.rows, p.n = a.n, p.norm = a.norm, p.eps = a.eps;
  p.x_vec = vectors_at(p.x, p.x_row, 16), p.residual_vec = vectors_at(p.residual, p.residual_row, 16), p.sum_vec = vectors_at(p.sum, p.sum_row, 16);
  p.gamma_vec = vectors_at(p.gamma, 0, 16), p.y_vec = vectors_at(p.y, p.y_row, ys == 1 ? 8 : 16);
  switch (a.type) {
    case MIMIR_B200_T_F32: return launch_to<MIMIR_B200_T_F32>(p, a.y_type, st);
    case MIMIR_B200_T_F16: return launch_to<MIMIR_B200_T_F16>(p, a.y_type, st);
    default: return launch_to<MIMIR_B200_T_BF16>(p, a.y_type, st);
  }
}

}  // namespace mb
