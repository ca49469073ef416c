// sample.cu — a token from each row of logits by a given random number: temperature, top-k, top-p and min-p.
//
//   w_i = exp((x_i - max) / T).  Candidates in the order (w descending, index ascending): the first top_k of them; of those the shortest
//   beginning that holds top_p of their mass; of those w_i >= min_p.  The token is the first index (in index order) at which the running
//   sum of the candidates' w exceeds u times their whole sum.
//
// A sum is compared with a border, so every w is a 64-bit integer (w times a power of two that leaves room for n of them): sums of
// integers are the same in every order.  The borders of top_k and top_p are found digit by digit of the logits' order (their
// bits, as unsigned integers that ascend with the value): counts and masses of 256 digits at a time, four rounds.
#include "common.h"
#include "paged.cuh"

namespace mb {
namespace {

constexpr int SA_THREADS = 1024, SA_WARPS = SA_THREADS / 32;

// ascending in the value; 0: not a candidate (not a number, -infinity)
__device__ __forceinline__ uint32_t order_of(float x) {
  if (!(x > -INFINITY)) return 0;
  const uint32_t b = __float_as_uint(x == 0.0f ? 0.0f : x);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) { return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o); }

template <int T>
__device__ __forceinline__ float logit(const void* row, int i) {
  if constexpr (T == MIMIR_B200_T_F32) return __ldg(static_cast<const float*>(row) + i);
  else if constexpr (T == MIMIR_B200_T_F16) return __half2float(static_cast<const __half*>(row)[i]);
  else return __bfloat162float(static_cast<const __nv_bfloat16*>(row)[i]);
}

template <class V>
__device__ __forceinline__ V warp_scan(V v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}
// exclusive sum over the block's threads; *total: of all
template <class V>
__device__ __forceinline__ V block_scan(V v, V* scratch, V* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const V inc = warp_scan(v, lane);
  __syncthreads();
  if (lane == 31) scratch[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    const V w = scratch[lane];
    const V s = warp_scan(w, lane);
    scratch[lane] = s - w;
    if (lane == 31) scratch[32] = s;
  }
  __syncthreads();
  *total = scratch[32];
  return scratch[warp] + inc - v;
}

struct Weigh {
  double top, inv_t, one;  // one: what a weight of 1 is as an integer
  __device__ __forceinline__ unsigned long long operator()(float x) const {
    return static_cast<unsigned long long>(__double2ull_rn(exp((static_cast<double>(x) - top) * inv_t) * one));
  }
};

template <int T>
__global__ void __launch_bounds__(SA_THREADS) sample_rows_kernel(const __grid_constant__ SampleLaunch a) {
  static_assert(SA_WARPS == 32, "block_scan");
  __shared__ unsigned long long mass[256];
  __shared__ unsigned count[256];
  __shared__ unsigned long long s64[33];
  __shared__ int s32[33];
  __shared__ uint32_t s_order;
  __shared__ int s_index;
  const int tid = threadIdx.x, lane = tid & 31, n = a.n;
  const long long row = blockIdx.x;
  const char* x = static_cast<const char*>(a.x) + row * a.row_stride * type_bytes(T);
  const float t = a.temperature ? __ldg(a.temperature + row) : 1.0f;
  const int top_k = a.top_k ? __ldg(a.top_k + row) : 0;
  const float top_p = a.top_p ? __ldg(a.top_p + row) : 1.0f, min_p = a.min_p ? __ldg(a.min_p + row) : 0.0f;
  const float u = __ldg(a.uniform + row);

  // the largest logit, and the first index that has it
  uint32_t best = 0;
  int at = n;
  for (int i = tid; i < n; i += SA_THREADS) {
    const uint32_t o = order_of(logit<T>(x, i));
    if (o > best) best = o, at = i;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const uint32_t ob = __shfl_xor_sync(0xffffffffu, best, o);
    const int oi = __shfl_xor_sync(0xffffffffu, at, o);
    if (ob > best || (ob == best && oi < at)) best = ob, at = oi;
  }
  if (tid == 0) s_order = 0, s_index = n;
  __syncthreads();
  if (lane == 0) atomicMax(&s_order, best);
  __syncthreads();
  if (lane == 0 && best == s_order) atomicMin(&s_index, at);
  __syncthreads();
  best = s_order;
  at = s_index;
  const float top = value_of(best);
  if (best == 0 || top == INFINITY || !(t > 0.0f)) {
    if (tid == 0) {
      a.ids[row] = best == 0 ? -1 : at;
      if (a.logprob) a.logprob[row] = best == 0 ? -INFINITY : 0.0f;
    }
    return;
  }
  int room = 0;  // n <= 2^room
  while ((1ll << room) < n) ++room;
  Weigh weigh;
  weigh.top = top;
  weigh.inv_t = 1.0 / static_cast<double>(t);
  weigh.one = static_cast<double>(1ull << min(62 - room, 52));

  // candidates: order > border, and the first `ties` of order == border
  uint32_t border = 0;
  int ties = 0;
  unsigned long long whole = 0;  // their mass
  auto rounds = [&](bool by_count, long long want_count, unsigned long long want_mass) {
    // the largest border whose candidates with that order or more are at least want_count many, or have want_mass; among orders >= floor_order
    uint32_t prefix = 0;
    unsigned long long above = 0;
    long long above_n = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      if (tid < 256) mass[tid] = 0, count[tid] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += SA_THREADS) {
        const float v = logit<T>(x, i);
        const uint32_t o = order_of(v);
        if (o == 0 || o < border) continue;
        if (shift < 24 && (o >> (shift + 8)) != (prefix >> (shift + 8))) continue;
        atomicAdd(&count[(o >> shift) & 255], 1u);
        if (!by_count) atomicAdd(&mass[(o >> shift) & 255], weigh(v));
      }
      __syncthreads();
      // thread d: what orders of digits above d hold
      const int d = 255 - tid;
      unsigned long long all;
      int all_n;
      const unsigned long long m_here = tid < 256 ? mass[d] : 0;
      const int c_here = tid < 256 ? static_cast<int>(count[d]) : 0;
      const unsigned long long m_before = block_scan(m_here, s64, &all) + above;
      const long long c_before = block_scan(c_here, s32, &all_n) + above_n;
      if (tid == 0) s_index = -1;
      __syncthreads();
      if (tid < 256 && c_here > 0) {
        const bool crosses = by_count ? (c_before < want_count && c_before + c_here >= want_count)
                                      : (m_before < want_mass && m_before + m_here >= want_mass);
        if (crosses) {
          s_index = d;
          s64[0] = m_before;
          s32[0] = static_cast<int>(c_before);
        }
      }
      __syncthreads();
      if (s_index < 0) return false;  // fewer than that: all of them
      prefix |= static_cast<uint32_t>(s_index) << shift;
      above = s64[0];
      above_n = s32[0];
    }
    const unsigned long long w = weigh(value_of(prefix));
    int many = static_cast<int>(count[prefix & 255]);
    if (by_count) {
      many = static_cast<int>(want_count - above_n);
    } else {
      // tie j (from 0) is kept while what is ahead of it is less than want_mass
      const unsigned long long left = want_mass - above, need = w ? (left + w - 1) / w : 1;
      if (need < static_cast<unsigned long long>(many)) many = static_cast<int>(need);
      if (prefix == border && ties > 0 && ties < many) many = ties;
    }
    border = prefix;
    ties = many;
    __syncthreads();
    return true;
  };
  if (top_k > 0 && top_k < n) rounds(true, top_k, 0);
  if (top_p < 1.0f) {
    // the mass of the candidates so far
    unsigned long long part = 0;
    for (int i = tid; i < n; i += SA_THREADS) {
      const float v = logit<T>(x, i);
      const uint32_t o = order_of(v);
      if (o > border) part += weigh(v);
    }
    block_scan(part, s64, &whole);
    if (border) whole += static_cast<unsigned long long>(ties) * weigh(value_of(border));
    const double want = ceil(static_cast<double>(top_p) * static_cast<double>(whole));
    rounds(false, 0, want >= 1.0 ? static_cast<unsigned long long>(want) : 1ull);
  }

  // running sums in index order: a thread has a stretch of the row
  const unsigned long long least = min_p > 0.0f ? static_cast<unsigned long long>(ceil(fmin(static_cast<double>(min_p), 1.0) * weigh.one)) : 0;
  const int stretch = (n + SA_THREADS - 1) / SA_THREADS;
  const int i0 = min(n, tid * stretch), i1 = min(n, i0 + stretch);
  int my_ties = 0, all_ties;
  if (border)
    for (int i = i0; i < i1; ++i) my_ties += order_of(logit<T>(x, i)) == border;
  const int ties_before = block_scan(my_ties, s32, &all_ties);
  auto walk = [&](unsigned long long from, unsigned long long until, unsigned long long* w_at) {
    int seen = ties_before;
    for (int i = i0; i < i1; ++i) {
      const float v = logit<T>(x, i);
      const uint32_t o = order_of(v);
      if (o == 0 || o < border) continue;
      if (border && o == border && seen++ >= ties) continue;
      const unsigned long long w = weigh(v);
      if (w < least) continue;
      from += w;
      *w_at = w;
      if (from > until) return i;
    }
    *w_at = from;
    return -1;
  };
  unsigned long long mine, total;
  walk(0, ~0ull, &mine);
  const unsigned long long before = block_scan(mine, s64, &total);
  // u times the sum, rounded down; below the sum
  double goal = floor(fmin(fmax(static_cast<double>(u), 0.0), 1.0) * static_cast<double>(total));
  unsigned long long until = static_cast<unsigned long long>(goal);
  if (until >= total) until = total - 1;
  if (before <= until && until < before + mine) {
    unsigned long long w;
    const int id = walk(before, until, &w);
    a.ids[row] = id;
    if (a.logprob) a.logprob[row] = static_cast<float>(log(static_cast<double>(w) / static_cast<double>(total)));
  }
}

}  // namespace

int launch_sample_rows(const SampleLaunch& s, cudaStream_t st) {
  const unsigned grid = static_cast<unsigned>(s.rows);
  if (s.type == MIMIR_B200_T_F32) sample_rows_kernel<MIMIR_B200_T_F32><<<grid, SA_THREADS, 0, st>>>(s);
  else if (s.type == MIMIR_B200_T_F16) sample_rows_kernel<MIMIR_B200_T_F16><<<grid, SA_THREADS, 0, st>>>(s);
  else sample_rows_kernel<MIMIR_B200_T_BF16><<<grid, SA_THREADS, 0, st>>>(s);
  MB_CUDA(cudaGetLastError());
  count_launch();
  return MIMIR_B200_OK;
}

}  // namespace mb
