// paged_cache.cu — new keys and values into the pages of a cache, and sequences back out of it.
//
// Pure data movement: rows in, codes (and a scale per row and head in 8 bits) out, each once.  A vector of head_dim elements belongs to a
// group of lanes with eight elements each, so that a group's largest magnitude is a few shuffles and loads are 16 bytes.  A CTA looks
// up where its rows go once, in shared memory, and then moves all their heads.
//   I8:   scale = amax * (1 / 127), code = x / scale to nearest (ties to even)      E4M3: scale = amax * (1 / 448), likewise
// amax is over the finite elements; 1 / 127 and 1 / 448 are fp32 constants and the division is the IEEE one, so that codes are what any
// fp32 program gets that computes them so.
// Writing codes is bound by instruction issue (160 instructions for a warp's 256 elements, some 50 of them the quotients): 27 K tokens, 8 key heads of
// 128, bfloat16 to int8 46 us, 1.9 times its bytes' time at the copy rate.  Reading is bound by its bytes: 16 sequences of up to 8 K int8 keys to bfloat16 95 us, the copy rate.
#include "common.h"
#include "paged.cuh"

namespace mb {
namespace {

constexpr int PC_THREADS = 256;
constexpr int PC_ROWS = 32;     // most rows a CTA looks up
constexpr int PC_STARTS = 1024;  // sequence starts kept in shared memory
constexpr int PC_HEADS = 32;     // heads of a CTA

// the last s of 0 .. n with start[s] <= row, -1 if none (starts ascend; entries that do not are found out by the caller)
__device__ __forceinline__ int last_start(const int* start, int n, int row) {
  int lo = -1, hi = n + 1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= row) lo = mid;
    else hi = mid;
  }
  return lo;
}

struct CacheMove {
  PagedView p;
  const int* start;  // [n_seqs + 1] row_start (write) or out_start (read)
  int rows;
  void* k;
  void* v;
  long long row_stride, head_stride;
  int per_cta, group;  // rows of a CTA; lanes of a vector, a power of two
  FastDiv by_full, by_rest;  // vectors of a row of PC_HEADS heads, and of the last ones'
};

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float min3_nan(float a, float b, float c) {
  float d;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Codes of f / s, correctly rounded quotients by one reciprocal for all of them: with r = 1 / s rounded to nearest, q = f r and
// q + (f - q s) r with fused multiply-adds is the IEEE quotient (Markstein, IBM J. Res. Dev. 34, 1990), where nothing under- or overflows:
// s above 2^-80, for smaller f the code is zero either way.  Quotients of 16-bit values are often just between two codes, so their last
// bits count.  27 K tokens of 8 key heads of 128 to int8: 90 us with an IEEE division an element, 55 so.
template <int CT>
__device__ __forceinline__ Raw8<CT> quotient_codes(const float (&f)[8], float s) {
  const float r = s > 0.0f ? __fdiv_rn(1.0f, s) : 0.0f;
  float q[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float n = __fmul_rn(f[e], r);
    q[e] = __fmaf_rn(__fmaf_rn(-n, s, f[e]), r, n);
    if constexpr (CT != MIMIR_B200_T_I8) q[e] = copysignf(q[e], f[e]);  // (zeros)
  }
  if constexpr (CT != MIMIR_B200_T_I8) return pack8<CT>(q);
  Raw8<CT> codes;
  uint32_t w[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = __float_as_uint(q[e] + 12582912.0f);  // 1.5 * 2^23: the nearest integer in the low bits, as two's complement
#pragma unroll
  for (int i = 0; i < 2; ++i)
    codes.w[i] = __byte_perm(__byte_perm(w[4 * i], w[4 * i + 1], 0x0040), __byte_perm(w[4 * i + 2], w[4 * i + 3], 0x0040), 0x5410);
  return codes;
}

template <int CT, int T, bool WRITE>
__global__ void __launch_bounds__(PC_THREADS) cache_move_kernel(const __grid_constant__ CacheMove a) {
  constexpr bool CODED = CT == MIMIR_B200_T_I8 || CT == MIMIR_B200_T_E4M3;
  constexpr float TOP = CT == MIMIR_B200_T_I8 ? 127.0f : 448.0f, PART = 1.0f / TOP;
  __shared__ int starts[PC_STARTS];
  // in bytes: a row's slot in the pages (-1: the row is none of a sequence) and in the scales, and where it begins in the tensors; then the
  // same of a head, keys before values, from the pointers on (64-bit products a vector took a third of the instructions)
  __shared__ long long at[PC_ROWS], scale_at[PC_ROWS], row_at[PC_ROWS];
  __shared__ char *pool_of[2 * PC_HEADS], *mem_of[2 * PC_HEADS];
  __shared__ float* scales_of[2 * PC_HEADS];
  const PagedView& p = a.p;
  const int row0 = blockIdx.x * a.per_cta, rows = min(a.per_cta, a.rows - row0);
  const int head0 = blockIdx.y * PC_HEADS, heads = min(PC_HEADS, p.kv_heads - head0), per_row = 2 * heads;
  const bool kept = p.n_seqs < PC_STARTS;
  if (kept) {
    for (int i = threadIdx.x; i <= p.n_seqs; i += PC_THREADS) starts[i] = __ldg(a.start + i);
    __syncthreads();
  }
  if (static_cast<int>(threadIdx.x) < rows) {
    const int row = row0 + threadIdx.x, s = last_start(kept ? starts : a.start, p.n_seqs, row);
    long long where = -1, sc = 0;
    if (s >= 0 && s < p.n_seqs) {
      const int first = a.start[s], end = a.start[s + 1], kv = __ldg(p.kv_len + s);
      // (out_start of a read: as many rows as keys, the last ones of a longer range stay as they are)
      const int pos = WRITE ? kv - (end - row) : row - first;
      if (first < 0 || row < first || row >= end || end > a.rows || (WRITE && end - first > p.max_rows)) {
        atomicOr(p.flags, PAGED_BAD_ROWS);
      } else if (kv < 0 || kv > p.max_kv || kv > p.table_stride * p.page_size) {
        atomicOr(p.flags, PAGED_BAD_LEN);
      } else if (pos >= 0 && pos < kv) {
        const int pi = p.by_page.div(pos), slot = pos - pi * p.page_size, page = paged_page(p, s, pi);
        if (page >= 0) {
          where = (page * p.page_stride + slot * p.slot_stride) * type_bytes(CT);
          sc = static_cast<long long>(page) * p.kv_heads * p.page_size + slot;
        }
      }
    }
    at[threadIdx.x] = where;
    scale_at[threadIdx.x] = sc;
    row_at[threadIdx.x] = row * a.row_stride * type_bytes(T);
  } else if (threadIdx.x >= 64 && static_cast<int>(threadIdx.x) - 64 < per_row) {
    const int j = threadIdx.x - 64;
    const bool is_v = j >= heads;
    const long long head = head0 + (is_v ? j - heads : j);
    pool_of[j] = static_cast<char*>(is_v ? p.v : p.k) + head * p.head_stride * type_bytes(CT);
    mem_of[j] = static_cast<char*>(is_v ? a.v : a.k) + head * a.head_stride * type_bytes(T);
    if constexpr (CODED) scales_of[j] = (is_v ? p.v_scale : p.k_scale) + head * p.page_size;
  }
  __syncthreads();
  const int lane = threadIdx.x & (a.group - 1), d = lane * 8;
  const bool mine = d < p.head_dim;
  const int groups = PC_THREADS / a.group, vectors = rows * per_row;
  const FastDiv by_row = heads == PC_HEADS ? a.by_full : a.by_rest;
  // (whole warps stay in the loop for the shuffles; U vectors of a group are on their way together)
  constexpr int U = 4;
  for (int i0 = 0; i0 < vectors; i0 += U * groups) {
    Raw8<WRITE ? T : CT> raw[U];
    char* to[U];
    float* scale_of[U];
    bool go[U];
    float scale[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * groups + threadIdx.x / a.group;
      const bool there = i < vectors;
      const int row = there ? by_row.div(i) : 0, j = there ? i - row * per_row : 0;
      const long long slot = at[row];
      go[u] = there && mine && slot >= 0;
      char* mem = mem_of[j] + row_at[row] + d * type_bytes(T);
      char* pool = pool_of[j] + slot + d * type_bytes(CT);
      if constexpr (CODED) scale_of[u] = scales_of[j] + scale_at[row];
      to[u] = WRITE ? pool : mem;
      if (go[u]) raw[u] = load8<WRITE ? T : CT>(WRITE ? mem : pool);
      else
#pragma unroll
        for (uint32_t& w : raw[u].w) w = 0;
      if constexpr (!WRITE && CODED) scale[u] = go[u] ? *scale_of[u] : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[8];
      unpack8<WRITE ? T : CT>(raw[u], f);
      if constexpr (WRITE) {
        if constexpr (CODED) {
          // (a maximum of not a number is one)
          float amax = fmaxf(max3_nan(max3_nan(f[0], f[1], f[2]), max3_nan(f[3], f[4], f[5]), max3_nan(f[6], f[7], f[7])),
                             -min3_nan(min3_nan(f[0], f[1], f[2]), min3_nan(f[3], f[4], f[5]), min3_nan(f[6], f[7], f[7])));
          const bool finite = !__any_sync(0xffffffffu, !(amax < INFINITY));
          if (!finite) {
            amax = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (fabsf(f[e]) < INFINITY) amax = fmaxf(amax, fabsf(f[e]));
          }
          for (int o = a.group >> 1; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
          const float s = __fmul_rn(amax, PART);
          if (go[u] && lane == 0) *scale_of[u] = s;
          Raw8<CT> codes;
          if (finite && (s == 0.0f || s > 0x1p-80f)) {
            codes = quotient_codes<CT>(f, s);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              // (a scale of zero: nothing but zeros, infinities and magnitudes whose scale is below fp32's smallest)
              const float v = s > 0.0f ? __fdiv_rn(f[e], s) : 0.0f;
              f[e] = CT != MIMIR_B200_T_I8 ? v : v == v ? fmaxf(-TOP, fminf(TOP, v)) : 0.0f;
            }
            codes = pack8<CT>(f);
          }
          if (go[u]) store8<CT>(to[u], codes);
          continue;
        }
        if (go[u]) store8<CT>(to[u], pack8<CT>(f));
      } else {
        if constexpr (CODED) {
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] *= scale[u];
        }
        if (go[u]) store8<T>(to[u], pack8<T>(f));
      }
    }
  }
}

template <bool WRITE, int CT>
int launch_move_as(const CacheMove& a, int type, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>((a.rows + a.per_cta - 1LL) / a.per_cta), static_cast<unsigned>((a.p.kv_heads + PC_HEADS - 1) / PC_HEADS));
  if (type == MIMIR_B200_T_F32) cache_move_kernel<CT, MIMIR_B200_T_F32, WRITE><<<grid, PC_THREADS, 0, st>>>(a);
  else if (type == MIMIR_B200_T_F16) cache_move_kernel<CT, MIMIR_B200_T_F16, WRITE><<<grid, PC_THREADS, 0, st>>>(a);
  else cache_move_kernel<CT, MIMIR_B200_T_BF16, WRITE><<<grid, PC_THREADS, 0, st>>>(a);
  MB_CUDA(cudaGetLastError());
  count_launch();
  return MIMIR_B200_OK;
}

template <bool WRITE>
int launch_move(CacheMove a, int cache_type, int type, cudaStream_t st) {
  a.group = 1;
  while (a.group * 8 < a.p.head_dim) a.group *= 2;
  a.by_full = FastDiv(2 * PC_HEADS);
  a.by_rest = FastDiv(static_cast<uint32_t>(2 * ((a.p.kv_heads - 1) % PC_HEADS + 1)));
  // rows of a CTA: enough for a pass of its threads, and no fewer CTAs than SMs for that
  a.per_cta = 1;
  while (a.per_cta < PC_ROWS && a.rows >= 8LL * ctx().sm_count * a.per_cta) a.per_cta *= 2;
  switch (cache_type) {
    case MIMIR_B200_T_F32: return launch_move_as<WRITE, MIMIR_B200_T_F32>(a, type, st);
    case MIMIR_B200_T_F16: return launch_move_as<WRITE, MIMIR_B200_T_F16>(a, type, st);
    case MIMIR_B200_T_BF16: return launch_move_as<WRITE, MIMIR_B200_T_BF16>(a, type, st);
    case MIMIR_B200_T_I8: return launch_move_as<WRITE, MIMIR_B200_T_I8>(a, type, st);
    default: return launch_move_as<WRITE, MIMIR_B200_T_E4M3>(a, type, st);
  }
}

}  // namespace

int launch_cache_write(const PagedView& p, int cache_type, const void* k, const void* v, int type, long long row_stride, long long head_stride,
                       cudaStream_t st) {
  CacheMove a = {};
  a.p = p, a.start = p.row_start, a.rows = p.n_rows, a.k = const_cast<void*>(k), a.v = const_cast<void*>(v);
  a.row_stride = row_stride, a.head_stride = head_stride;
  return launch_move<true>(a, cache_type, type, st);
}
int launch_cache_read(const PagedView& p, int cache_type, const int* out_start, int out_rows, void* k, void* v, int type, long long row_stride,
                      long long head_stride, cudaStream_t st) {
  CacheMove a = {};
  a.p = p, a.start = out_start, a.rows = out_rows, a.k = k, a.v = v;
  a.row_stride = row_stride, a.head_stride = head_stride;
  return launch_move<false>(a, cache_type, type, st);
}

}  // namespace mb
