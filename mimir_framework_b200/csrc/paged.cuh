// paged.cuh — what the serving kernels share: a paged key / value cache and a ragged batch as they come from the host, the checks
// of the numbers in device memory that index them, and the element types.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "mimir_b200.h"

namespace mb {

// What a kernel found in device memory that does not fit the call (dev_error_word[1]); such a sequence or page is left out.
enum : int { PAGED_BAD_ROWS = 1, PAGED_BAD_LEN = 2, PAGED_BAD_PAGE = 4 };

__host__ __device__ constexpr int type_bytes(int t) { return t == MIMIR_B200_T_F32 ? 4 : (t == MIMIR_B200_T_F16 || t == MIMIR_B200_T_BF16) ? 2 : 1; }

// n / d for 0 <= n < 2^31 by a multiplication (d fixed for a launch): with l = ceil(log2 d), n / d = (umulhi(m, n) + n) >> l
struct FastDiv {
  uint32_t m = 0, l = 0, d = 1;
  FastDiv() = default;
  explicit FastDiv(uint32_t v) : d(v) {
    while ((1ull << l) < d) ++l;
    m = static_cast<uint32_t>((((1ull << l) - d) << 32) / d + 1);
  }
  __device__ __forceinline__ int div(int n) const { return static_cast<int>((__umulhi(m, static_cast<uint32_t>(n)) + static_cast<uint32_t>(n)) >> l); }
};

struct PagedView {
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  long long page_stride, slot_stride, head_stride;  // elements
  int n_pages, page_size, kv_heads, head_dim;
  FastDiv by_page;
  const int* row_start;
  const int* kv_len;
  const int* table;
  long long table_stride;
  int n_seqs, n_rows, max_rows, max_kv;
  int* flags;
};

namespace {

// One sequence: its rows and keys, none of either where the numbers do not fit.
struct PagedSeq {
  int row0 = 0, rows = 0, kv = 0;
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedView& p, int s) {
  PagedSeq q;
  const int a = __ldg(p.row_start + s), b = __ldg(p.row_start + s + 1), kv = __ldg(p.kv_len + s);
  if (a < 0 || b < a || b > p.n_rows || b - a > p.max_rows) {
    atomicOr(p.flags, PAGED_BAD_ROWS);
    return q;
  }
  q.row0 = a;
  q.rows = b - a;
  if (kv < 0 || kv > p.max_kv || kv > p.table_stride * p.page_size) {
    atomicOr(p.flags, PAGED_BAD_LEN);
    return q;
  }
  q.kv = kv;
  return q;
}
// the page of a key of a sequence, -1 where it is none of the cache's
__device__ __forceinline__ int paged_page(const PagedView& p, int s, int page_index) {
  const int page = __ldg(p.table + s * p.table_stride + page_index);
  if (static_cast<unsigned>(page) < static_cast<unsigned>(p.n_pages)) return page;
  atomicOr(p.flags, PAGED_BAD_PAGE);
  return -1;
}

// ---- eight consecutive elements of a type, as they lie in memory ----------------------------------------------------------------
template <int T>
struct Raw8 {
  uint32_t w[type_bytes(T) * 2];
};
template <int T>
__device__ __forceinline__ Raw8<T> load8(const void* p) {
  Raw8<T> r;
  if constexpr (type_bytes(T) == 1) {
    const uint2 v = *static_cast<const uint2*>(p);
    r.w[0] = v.x, r.w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < type_bytes(T) / 2; ++i) {
      const uint4 v = static_cast<const uint4*>(p)[i];
      r.w[4 * i] = v.x, r.w[4 * i + 1] = v.y, r.w[4 * i + 2] = v.z, r.w[4 * i + 3] = v.w;
    }
  }
  return r;
}
template <int T>
__device__ __forceinline__ void store8(void* p, const Raw8<T>& r) {
  if constexpr (type_bytes(T) == 1) {
    *static_cast<uint2*>(p) = make_uint2(r.w[0], r.w[1]);
  } else {
#pragma unroll
    for (int i = 0; i < type_bytes(T) / 2; ++i) static_cast<uint4*>(p)[i] = make_uint4(r.w[4 * i], r.w[4 * i + 1], r.w[4 * i + 2], r.w[4 * i + 3]);
  }
}
// to fp32 and back (to nearest, ties to even)
template <int T>
__device__ __forceinline__ void unpack8(const Raw8<T>& r, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (T == MIMIR_B200_T_F32) {
      f[i] = __uint_as_float(r.w[i]);
    } else if constexpr (T == MIMIR_B200_T_F16) {
      f[i] = __half2float(__ushort_as_half(static_cast<unsigned short>(r.w[i / 2] >> (16 * (i & 1)))));
    } else if constexpr (T == MIMIR_B200_T_BF16) {
      f[i] = __uint_as_float((i & 1) ? (r.w[i / 2] & 0xffff0000u) : (r.w[i / 2] << 16));
    } else if constexpr (T == MIMIR_B200_T_I8) {
      f[i] = static_cast<float>(static_cast<int8_t>(r.w[i / 4] >> (8 * (i & 3))));
    } else {
      const __half_raw h = __nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(r.w[i / 4] >> (8 * (i & 3))), __NV_E4M3);
      f[i] = __half2float(__half(h));
    }
  }
}
template <int T>
__device__ __forceinline__ Raw8<T> pack8(const float (&f)[8]) {
  Raw8<T> r;
  if constexpr (T == MIMIR_B200_T_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.w[i] = __float_as_uint(f[i]);
  } else if constexpr (T == MIMIR_B200_T_F16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      r.w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  } else if constexpr (T == MIMIR_B200_T_BF16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      r.w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  } else if constexpr (T == MIMIR_B200_T_I8) {  // (values within +-127: the caller has divided by the scale)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t w = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) w |= (static_cast<uint32_t>(max(-127, min(127, __float2int_rn(f[4 * i + j])))) & 0xffu) << (8 * j);
      r.w[i] = w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t a = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * i], f[4 * i + 1]), __NV_SATFINITE, __NV_E4M3);
      const uint32_t b = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * i + 2], f[4 * i + 3]), __NV_SATFINITE, __NV_E4M3);
      r.w[i] = a | (b << 16);
    }
  }
  return r;
}

}  // namespace

// the launches behind the C calls (serve.cu); arguments are checked there
struct RopeLaunch {
  MimirRopePlan plan;
  const int* positions;
  const void* x;
  void* y;
  long long rows, x_row, x_head, y_row, y_head;
  int heads, dim, type;
};
int launch_rope(const RopeLaunch& r, cudaStream_t st);
int launch_cache_write(const PagedView& p, int cache_type, const void* k, const void* v, int type, long long row_stride, long long head_stride,
                       cudaStream_t st);
int launch_cache_read(const PagedView& p, int cache_type, const int* out_start, int out_rows, void* k, void* v, int type, long long row_stride,
                      long long head_stride, cudaStream_t st);
struct AttendLaunch {
  PagedView p;
  const void* q;
  void* out;
  float* lse;
  long long q_row, q_head, o_row, o_head;
  int cache_type, type, heads, causal, window;
  float scale;
  void* ws;
  size_t ws_bytes;
};
size_t paged_attention_ws_bytes(const AttendLaunch& a);
int launch_paged_attention(const AttendLaunch& a, cudaStream_t st);
struct SampleLaunch {
  const void* x;
  long long rows, row_stride;
  int n, type;
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  const float* uniform;
  int* ids;
  float* logprob;
};
int launch_sample_rows(const SampleLaunch& s, cudaStream_t st);

}  // namespace mb
