// sample.cu — a token from each row of logits by a given random number: temperature, top-k, top-p and min-p.
//
//   w_i = exp((x_i - max) / T).  Candidates in the order (w descending, index ascending): the first top_k of them; of those the shortest
//   beginning that holds top_p of their mass; of those w_i >= min_p.  The token is the first index (in index order) at which the running
//   sum of the candidates' w exceeds u times their whole sum.
//
// A row is read once: a cluster of CTAs keeps it in shared memory, a slice each, and meets through distributed shared memory.
//   1. the largest logit, and in fp32 about how much all weights are
//   2. top_k: counts of 1024 intervals of (max - x) / T and the interval in which the border lies.  Up to 1024 logits down to that
//      are gathered, sorted and finished in one CTA; else the border itself is found among the interval's
//      top_p: rough masses of the intervals (one 32-bit addition in shared memory a logit) say between which two the border lies, a
//      part in 2^10 of the mass to either side, and what n roundings to units of 2^-30 may add.  Where min_p ends before them, top_p
//      takes nothing away.  Else every weight is taken exactly, what lies between the two is listed, and the border found among it.
//      min_p and top_p: what min_p leaves is summed roughly first, and mostly that is enough
//      A border among logits: up to 1024 are sorted in one CTA; more are divided by their bits until they are fewer or all the same
//   3. masses of the warps' stretches of the row in index order; the stretch in which u falls is walked
// Sums are compared with borders, so every w is an integer (w times a power of two that leaves room for n of them): sums of integers are
// the same in every order and division of the work.  w comes from a table of 2^(k / 64) and four terms of the exponential series in
// fp64, relative error under 2^-44.  A large batch waits for instructions: about 8 a logit to load and sum it roughly, 12 for the
// intervals, 36 for an exact weight.
#include <cooperative_groups.h>

#include <cmath>

#include "common.h"
#include "paged.cuh"

namespace mb {
namespace {

namespace cg = cooperative_groups;

constexpr int SA_THREADS = 512, SA_WARPS = SA_THREADS / 32, SA_BINS = 1024, SA_LIST = 1024;
constexpr size_t SA_SLICE = size_t(88) << 10;   // bytes of a row in a CTA's shared memory: two CTAs to an SM
constexpr size_t SA_LARGE = size_t(180) << 10;  // the most: one

// ascending in the value; 0: not a candidate (not a number, -infinity)
__device__ __forceinline__ uint32_t order_of(float x) {
  if (!(x > -INFINITY)) return 0;
  const uint32_t b = __float_as_uint(x == 0.0f ? 0.0f : x);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) { return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o); }

// elements of 16 bytes
template <int T>
struct Vec {
  static constexpr int N = 16 / type_bytes(T);
  static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[N]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (T == MIMIR_B200_T_F32) {
        f[i] = __uint_as_float(w[i]);
      } else if constexpr (T == MIMIR_B200_T_F16) {
        const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        f[2 * i] = p.x, f[2 * i + 1] = p.y;
      } else {
        f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
};
template <int T>
__device__ __forceinline__ float logit(const void* row, long long i) {
  if constexpr (T == MIMIR_B200_T_F32) return __ldg(static_cast<const float*>(row) + i);
  else if constexpr (T == MIMIR_B200_T_F16) return __half2float(static_cast<const __half*>(row)[i]);
  else return __bfloat162float(static_cast<const __nv_bfloat16*>(row)[i]);
}

using u64 = unsigned long long;

__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct Powers {
  double v[64];  // 2^(k / 64)
};

struct Border {          // candidates: order > order, and the first `ties` (of `equals`) of order == order
  uint32_t order;
  uint32_t ties, equals;
};
struct Found {
  int bin;               // -1: the candidates do not reach the border
  uint32_t above_n, in_n;
  u64 above, in;
};

struct SampleShared {
  double table[64];
  uint32_t count[SA_BINS], mass_lo[SA_BINS], mass_hi[SA_BINS];  // of this CTA's slice
  u64 list[SA_LIST];  // order in the high half; below it the index's complement where indices matter
  u64 weight[256];
  uint32_t list_n;
  u64 scan64[33];
  uint32_t scan32[33];
  // read by the cluster's other CTAs
  int first, known;
  u64 total;
  Found found;
  Border border;
  int window[2];                                                // intervals between which top_p's border lies
  u64 above, inside;                                            // masses ahead of them and in them
  uint32_t inside_n;
  u64 warp_mass[SA_WARPS];
  uint32_t warp_ties[SA_WARPS];
  float warp_top[SA_WARPS], warp_sum[SA_WARPS];
  float stay_sum[SA_WARPS];
  uint32_t stay_n[SA_WARPS];
  double scale;
};

// w of a candidate (what is none gets some w of its own: callers leave it out)
struct Weigh {
  double top, scale;  // log2(e) / T
  double one;         // what a weight of 1 is as an integer
  float least_x;      // w is zero there and below
  const double* table;
  __device__ __forceinline__ double power(float x) const { return (static_cast<double>(x) - top) * scale; }  // of two, before w is rounded to an integer
  __device__ __forceinline__ u64 operator()(float x) const {
    const double y = (static_cast<double>(fmaxf(x, least_x)) - top) * scale;
    const double s = y + 105553116266496.0;  // 1.5 * 2^46: y rounded to 64ths in the low bits
    const int k = __double2loint(s);
    const double r = y - (s - 105553116266496.0);
    double p = fma(r, 9.618129107628477e-3, 5.5504108664821580e-2);  // ln(2)^i / i!
    p = fma(p, r, 2.4022650695910071e-1);
    p = fma(p, r, 6.9314718055994531e-1);
    p = fma(p, r, 1.0);
    const double t = table[k & 63];
    const double w = __hiloint2double(__double2hiint(t) + ((k >> 6) << 20), __double2loint(t)) * p;
    return static_cast<u64>(__double_as_longlong(fma(w, one, 4503599627370496.0)) & 0xfffffffffffffll);  // (2^52: the integer in the low bits)
  }
};

// the logarithm of x's share, w of total: near one from the integers, else from the logit, of which a small w keeps few bits
__device__ __forceinline__ float log_share(const Weigh& weigh, float x, u64 w, u64 total) {
  const u64 left = total - w;
  if (left < w) return log1pf(-(static_cast<float>(left) / static_cast<float>(total)));
  return static_cast<float>(weigh.power(x) * 0.69314718055994531) - logf(static_cast<float>(total) * (1.0f / static_cast<float>(weigh.one)));
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
    const V w = lane < SA_WARPS ? scratch[lane] : 0;
    const V s = warp_scan(w, lane);
    scratch[lane] = s - w;
    if (lane == 31) scratch[32] = s;
  }
  __syncthreads();
  *total = scratch[32];
  return scratch[warp] + inc - v;
}

template <int T, bool KEPT>
__global__ void __launch_bounds__(SA_THREADS, 2) sample_rows_kernel(const __grid_constant__ SampleLaunch a, int slice, const __grid_constant__ Powers powers) {
  constexpr int V = Vec<T>::N;
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ SampleShared sh;
  const cg::cluster_group cluster = cg::this_cluster();
  const int ranks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  auto meet = [&]() {  // all threads of the row
    if (ranks > 1) cluster.sync();
    else __syncthreads();
  };
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, n = a.n;
  const long long row = blockIdx.x / ranks;
  const char* x = static_cast<const char*>(a.x) + row * a.row_stride * type_bytes(T);
  const int first = min(n, rank * slice), mine = min(n, first + slice) - first;  // this CTA's stretch (slice: a multiple of 32 V)
  const float t = a.temperature ? __ldg(a.temperature + row) : 1.0f;
  const int top_k = a.top_k ? __ldg(a.top_k + row) : 0;
  const float top_p = a.top_p ? __ldg(a.top_p + row) : 1.0f, min_p = a.min_p ? __ldg(a.min_p + row) : 0.0f;
  const float u = __ldg(a.uniform + row);
  const int vecs = (mine + V - 1) / V;

  // ---- vector i of the stretch; absent elements are not numbers -------------------------------------------------------------------------
  auto from_global = [&](int i, float (&f)[V]) {
    const bool aligned = (reinterpret_cast<uintptr_t>(x) & 15) == 0;  // (stretches start on whole vectors)
    if (aligned && (i + 1) * V <= mine) {
      Vec<T>::unpack(__ldg(reinterpret_cast<const uint4*>(x) + first / V + i), f);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = i * V + e < mine ? logit<T>(x, first + i * V + e) : __uint_as_float(0x7fc00000u);
    }
  };
  auto read = [&](int i, float (&f)[V]) {
    if constexpr (KEPT) Vec<T>::unpack(reinterpret_cast<const uint4*>(dyn)[i], f);
    else from_global(i, f);
  };

  // ---- 1. the largest, and a rough sum of the weights (a thread's by its own largest, which it raises as it goes) ------------------------
  const float s2 = t > 0.0f ? 1.4426950408889634f / t : 0.0f;
  if (tid == SA_THREADS - 1) sh.scale = 1.4426950408889634074 / static_cast<double>(t);  // (one thread: a fp64 division of all took as long as a pass)
  float top = -INFINITY, rough = 0.0f;
  const bool by_count = top_k > 0 && top_k < n, by_mass = top_p < 1.0f, sum_now = by_mass && !by_count;
  auto take_in = [&](const float (&f)[V]) {
    float m = f[0];
#pragma unroll
    for (int e = 1; e < V; ++e) m = fmaxf(m, f[e]);
    if (!sum_now) {
      top = fmaxf(top, m);
      return;
    }
    if (m > top) {
      rough *= ex2f(fmaxf((top - m) * s2, -200.0f));
      top = m;
    }
#pragma unroll
    for (int e = 0; e < V; ++e) rough += ex2f(fmaxf((f[e] - top) * s2, -200.0f));
  };
  if constexpr (KEPT) {
    const bool aligned = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
    constexpr int U = 4;
    for (int i0 = tid; i0 < vecs; i0 += U * SA_THREADS) {
      uint4 v[U];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int i = i0 + j * SA_THREADS;
        if (i >= vecs) continue;
        if (aligned && (i + 1) * V <= mine) {
          v[j] = __ldg(reinterpret_cast<const uint4*>(x) + first / V + i);
        } else {
          float f[V];
          from_global(i, f);
          if constexpr (T == MIMIR_B200_T_F32) {
            v[j] = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
          } else {
            const Raw8<T> r = pack8<T>(f);
            v[j] = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int i = i0 + j * SA_THREADS;
        if (i >= vecs) continue;
        reinterpret_cast<uint4*>(dyn)[i] = v[j];
        float f[V];
        Vec<T>::unpack(v[j], f);
        take_in(f);
      }
    }
  } else {
    for (int i = tid; i < vecs; i += SA_THREADS) {
      float f[V];
      read(i, f);
      take_in(f);
    }
  }
  // sums of parts that have their own largest
  auto join = [&](float& m, float& s, float om, float os) {
    const float mm = fmaxf(m, om);
    if (mm > -INFINITY) s = s * ex2f(fmaxf((m - mm) * s2, -200.0f)) + os * ex2f(fmaxf((om - mm) * s2, -200.0f));
    m = mm;
  };
  auto join_warp = [&]() {
    if (sum_now) {
#pragma unroll
      for (int o = 16; o; o >>= 1) {
        const float om = __shfl_xor_sync(0xffffffffu, top, o), os = __shfl_xor_sync(0xffffffffu, rough, o);
        join(top, rough, om, os);
      }
    } else {
#pragma unroll
      for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
  };
  join_warp();
  if (tid < 64) sh.table[tid] = powers.v[tid];
  if (tid == 0) sh.list_n = 0;
  if (lane == 0) sh.warp_top[warp] = top, sh.warp_sum[warp] = rough;
  meet();
  {  // every warp joins the parts of all
    top = -INFINITY, rough = 0.0f;
    for (int i = lane; i < ranks * SA_WARPS; i += 32) {
      const SampleShared* s = cluster.map_shared_rank(&sh, i / SA_WARPS);
      if (sum_now) join(top, rough, s->warp_top[i % SA_WARPS], s->warp_sum[i % SA_WARPS]);
      else top = fmaxf(top, s->warp_top[i % SA_WARPS]);
    }
    join_warp();
    rough = __shfl_sync(0xffffffffu, rough, 0);  // (a decision of the whole row hangs on it: the lanes' may round apart)
  }

  if (top == -INFINITY || top == INFINITY || !(t > 0.0f)) {  // the largest's first index, or none
    int at = 0x7fffffff;
    if (top > -INFINITY)
      for (int i = tid; i < vecs && at == 0x7fffffff; i += SA_THREADS) {
        float f[V];
        read(i, f);
#pragma unroll
        for (int e = V - 1; e >= 0; --e)
          if (f[e] == top) at = first + i * V + e;
      }
    at = __reduce_min_sync(0xffffffffu, at);
    __syncthreads();
    if (tid == 0) sh.first = 0x7fffffff;
    __syncthreads();
    if (lane == 0) atomicMin(&sh.first, at);
    meet();
    if (rank == 0 && tid == 0) {
      for (int c = 0; c < ranks; ++c) at = min(at, *cluster.map_shared_rank(&sh.first, c));
      a.ids[row] = top == -INFINITY ? -1 : at;
      if (a.logprob) a.logprob[row] = top == -INFINITY ? -INFINITY : 0.0f;
    }
    meet();  // (no CTA leaves while others read its shared memory)
    return;
  }
  int room = 0;  // n <= 2^room
  while ((1ll << room) < n) ++room;
  Weigh weigh;
  weigh.top = top;
  weigh.scale = sh.scale;
  weigh.one = static_cast<double>(1ull << min(62 - room, 51));
  {
    // some 600 powers of two down; where no float is about there, every other logit is further down than that
    float low = fmaxf(top - 415.888f * t, -3.4028234e38f);
    const float down = (top - low) * s2;
    if (!(down < 900.0f) || low >= top) {
      low = fmaxf(value_of(order_of(top) - 1), -3.4028235e38f);
      weigh.scale = fmin(weigh.scale, 600.0 / (static_cast<double>(top) - low));
    }
    weigh.least_x = low;
  }
  weigh.table = sh.table;
  // logits surely below min_p are left out before they are weighed (2e-3 and a part in 10 000 of slack for the fp32 product)
  const float least_w = min_p > 0.0f ? fminf(min_p, 1.0f) : 0.0f;
  const u64 least = static_cast<u64>(ceil(static_cast<double>(least_w) * weigh.one));
  const float sure = min_p > 0.0f ? (log2f(least_w) - 2e-3f) * (t * 0.69321f) : -INFINITY;  // of x - max
  // ---- 2. the border ---------------------------------------------------------------------------------------------------------------------
  Border border = {0, 0, 0};
  if (by_count || by_mass) {
    const float width = static_cast<float>(32.0 * weigh.scale);  // of (max - x), in intervals
    // rounded in the low bits of 2^23 + it; what is not a number is in the last one
    auto interval = [&](float v) { return static_cast<int>(__float_as_uint(fminf((top - v) * width, SA_BINS - 1.0f) + 8388608.0f) & (2 * SA_BINS - 1)); };
    auto add_mass = [&](int bin, u64 w) {
      const uint32_t lo = static_cast<uint32_t>(w), old = atomicAdd(&sh.mass_lo[bin], lo);
      const uint32_t hi = static_cast<uint32_t>(w >> 32) + (old + lo < old ? 1u : 0u);
      if (hi) atomicAdd(&sh.mass_hi[bin], hi);
    };
    bool cleared = false;
    auto clear = [&]() {
      if (cleared) meet();  // (others have read what is cleared)
      else __syncthreads();
      cleared = true;
      for (int i = tid; i < SA_BINS; i += SA_THREADS) sh.count[i] = sh.mass_lo[i] = sh.mass_hi[i] = 0;
      if (tid == 0) sh.found.bin = -1, sh.window[0] = sh.window[1] = SA_BINS - 1;
      __syncthreads();
    };
    // the interval in which the candidates reach want_n in number, or `want` in mass, counted from (above_n, above)
    u64 want = 0;
    auto find = [&](bool number, uint32_t want_n, uint32_t above_n, u64 above) {
      meet();
      u64 m[2] = {0, 0};
      uint32_t c[2] = {0, 0};
      for (int q = 0; q < ranks; ++q) {
        const SampleShared* s = cluster.map_shared_rank(&sh, q);
        const uint2 n2 = *reinterpret_cast<const uint2*>(s->count + 2 * tid);
        c[0] += n2.x, c[1] += n2.y;
        if (!number) {
          const uint2 lo = *reinterpret_cast<const uint2*>(s->mass_lo + 2 * tid), hi = *reinterpret_cast<const uint2*>(s->mass_hi + 2 * tid);
          m[0] += (static_cast<u64>(hi.x) << 32) + lo.x, m[1] += (static_cast<u64>(hi.y) << 32) + lo.y;
        }
      }
      u64 all = 0, mb = 0;
      uint32_t all_n;
      if (!number) mb = block_scan(m[0] + m[1], sh.scan64, &all);
      uint32_t cb = block_scan(c[0] + c[1], sh.scan32, &all_n);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const u64 ahead = above + mb;
        const uint32_t ahead_n = above_n + cb;
        if (c[h] > 0 && (number ? ahead_n < want_n && ahead_n + c[h] >= want_n : ahead < want && ahead + m[h] >= want))
          sh.found = {2 * tid + h, ahead_n, c[h], ahead, m[h]};
        mb += m[h], cb += c[h];
      }
      __syncthreads();
      return sh.found;
    };
    auto sort = [&](int size) {  // sh.list, descending
      for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j; j >>= 1) {
          for (int i = tid; i < size / 2; i += SA_THREADS) {
            const int p = ((i & ~(j - 1)) << 1) | (i & (j - 1));
            const u64 a0 = sh.list[p], a1 = sh.list[p | j];
            if ((a0 < a1) == ((p & k) == 0)) sh.list[p] = a1, sh.list[p | j] = a0;
          }
          __syncthreads();
        }
    };
    // what `pick` says yes to, nothing below `bottom`, into the first CTA's list, filled up there with zeros to a power of two from 64 on; the
    // number, elsewhere -1
    int size = 64;
    auto collect = [&](float bottom, auto&& pick) {
      SampleShared* home = cluster.map_shared_rank(&sh, 0);
      for (int i = tid; i < vecs; i += SA_THREADS) {
        float v[V];
        read(i, v);
        float m = v[0];
#pragma unroll
        for (int e = 1; e < V; ++e) m = fmaxf(m, v[e]);
        if (!(m >= bottom)) continue;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          if (pick(v[e])) {
            const uint32_t at = atomicAdd(&home->list_n, 1u);
            if (at < SA_LIST) home->list[at] = (static_cast<u64>(order_of(v[e])) << 32) | ~static_cast<uint32_t>(first + i * V + e);
          }
        }
      }
      meet();
      if (rank != 0) return -1;
      const int have = static_cast<int>(min(sh.list_n, static_cast<uint32_t>(SA_LIST)));
      while (size < have) size *= 2;
      for (int i = tid; i < SA_LIST; i += SA_THREADS)
        if (i >= have) sh.list[i] = 0;
      __syncthreads();
      if (tid == 0) sh.list_n = 0;
      return have;
    };

    // The border among the logits of orders range_lo .. range_hi, and of the interval f.bin where `number` says so (f: what lies ahead of
    // them and in them): level by level, then sorted or a single order.
    auto settle = [&](bool number, uint32_t want_n, Found f, uint32_t range_lo, uint32_t range_hi) {
      const int value_bin = f.bin;
      int shift = -1;
      float x_lo = value_of(range_lo), x_hi = value_of(range_hi);
      auto member = [&](float v) { return v >= x_lo && v <= x_hi && (!number || interval(v) == value_bin); };
      while (f.in_n > SA_LIST && shift != 0) {
        // their range of orders, divided evenly, the largest first
        shift = 0;
        while (((range_hi - range_lo) >> shift) >= SA_BINS) ++shift;
        clear();
        for (int i = tid; i < vecs; i += SA_THREADS) {
          float v[V];
          read(i, v);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            if (!member(v[e])) continue;
            const int bin = static_cast<int>((range_hi - order_of(v[e])) >> shift);
            atomicAdd(&sh.count[bin], 1u);
            if (!number) add_mass(bin, weigh(v[e]));
          }
        }
        f = find(number, want_n, f.above_n, f.above);
        if (f.bin < 0) return;  // (never: the sums are exact)
        range_hi -= static_cast<uint32_t>(f.bin) << shift;
        const uint32_t span = (1u << shift) - 1;
        if (range_hi - range_lo > span) range_lo = range_hi - span;
        x_lo = value_of(range_lo), x_hi = value_of(range_hi);
      }
      if (f.in_n <= SA_LIST && shift != 0) {
        if (collect(x_lo, member) >= 0) {
          sort(size);
          // a thread has two neighbours of the sorted list
          const uint32_t o0 = static_cast<uint32_t>(sh.list[2 * tid] >> 32), o1 = static_cast<uint32_t>(sh.list[2 * tid + 1] >> 32);
          const u64 w0 = o0 ? weigh(value_of(o0)) : 0, w1 = o1 ? weigh(value_of(o1)) : 0;
          u64 all;
          const u64 b0 = f.above + block_scan(w0 + w1, sh.scan64, &all);
          const uint32_t n0 = f.above_n + 2 * tid;
          auto test = [&](int at, u64 b, uint32_t bn, u64 w) {
            const uint32_t o = static_cast<uint32_t>(sh.list[at] >> 32);
            if (!o || !(number ? bn + 1 == want_n : b < want && b + w >= want)) return;
            // its equals ahead of it are candidates too
            int from = at, to = at;
            while (from > 0 && static_cast<uint32_t>(sh.list[from - 1] >> 32) == o) --from;
            while (to + 1 < SA_LIST && static_cast<uint32_t>(sh.list[to + 1] >> 32) == o) ++to;
            sh.border.order = o;
            sh.border.ties = static_cast<uint32_t>(at - from + 1);
            sh.border.equals = static_cast<uint32_t>(to - from + 1);
          };
          test(2 * tid, b0, n0, w0);
          test(2 * tid + 1, b0 + w0, n0 + 1, w1);
        }
        meet();
        border = *cluster.map_shared_rank(&sh.border, 0);
      } else {
        // one order alone
        border.order = range_hi;
        border.equals = f.in_n;
        const u64 w = weigh(value_of(border.order));
        if (number) {
          border.ties = want_n - f.above_n;
        } else {
          const u64 left = want - f.above, need = w ? (left + w - 1) / w : 1;  // tie j (from 0) is kept while what is ahead is less
          border.ties = need < f.in_n ? static_cast<uint32_t>(need) : f.in_n;
        }
      }
    };
    // The `have` logits of the list, in the first CTA: top_k, top_p and min_p in their order, then u in index order.  top_p's part is of the first
    // `most` of them, or of `outside`, which is known to a part in 2^10: false where that leaves open which ones stay.
    auto finish = [&](int have, uint32_t most, double outside) {
      auto part_of = [&](double all) {
        const double part = ceil(fmax(static_cast<double>(top_p), 0.0) * all);
        return part >= 1.0 ? static_cast<u64>(part) : 1ull;
      };
      auto limit_of = [&](u64 all) { return !by_mass ? ~0ull : part_of(outside > 0.0 ? outside * (1.0 - 0x1p-10) : static_cast<double>(all)); };
      const u64 beyond = outside > 0.0 ? part_of(outside * (1.0 + 0x1p-10)) : 0;  // (the limit may be up to this)
      auto until_of = [&](u64 all) {
        const u64 until = static_cast<u64>(floor(fmin(fmax(static_cast<double>(u), 0.0), 1.0) * static_cast<double>(all)));
        return until >= all ? all - 1 : until;
      };
      if (size <= 256) {
        // each with each, several threads a logit: how many and how much are ahead of it, then how much is before it by index (a sort
        // by one warp took 5000 cycles for 64)
        const int parts = SA_THREADS / size, item = tid / parts, part = tid % parts, per = size / parts;
        if (tid < size) sh.weight[tid] = sh.list[tid] ? weigh(value_of(static_cast<uint32_t>(sh.list[tid] >> 32))) : 0;
        __syncthreads();
        const u64 mine_l = sh.list[item], w = sh.weight[item];
        u64 ahead = 0;
        uint32_t rank_l = 0;
        for (int j = 0; j < per; ++j) {
          const int i = j * parts + part;
          if (sh.list[i] > mine_l) ++rank_l, ahead += sh.weight[i];
        }
        for (int o = parts >> 1; o; o >>= 1) ahead += __shfl_xor_sync(0xffffffffu, ahead, o), rank_l += __shfl_xor_sync(0xffffffffu, rank_l, o);
        const uint32_t last_rank = min(most, static_cast<uint32_t>(have)) - 1;
        if (mine_l && rank_l == last_rank && part == 0) sh.above = ahead + w;
        __syncthreads();
        const u64 limit = limit_of(sh.above);
        const u64 kept = mine_l && rank_l <= last_rank && ahead < limit && w >= least ? w : 0;
        if (part == 0) sh.weight[item] = kept;
        if (__syncthreads_or(mine_l && w >= least && ahead >= limit && ahead < beyond)) return false;
        u64 before = 0, all = 0;
        for (int j = 0; j < per; ++j) {
          const int i = j * parts + part;
          const u64 o = sh.weight[i];
          all += o;
          if (static_cast<uint32_t>(sh.list[i]) > static_cast<uint32_t>(mine_l)) before += o;  // (the index's complement)
        }
        for (int o = parts >> 1; o; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o), before += __shfl_xor_sync(0xffffffffu, before, o);
        const u64 until = until_of(all);
        if (part == 0 && before <= until && until < before + kept) {
          a.ids[row] = static_cast<int>(~static_cast<uint32_t>(mine_l));
          if (a.logprob) a.logprob[row] = log_share(weigh, value_of(static_cast<uint32_t>(mine_l >> 32)), kept, all);
        }
        return true;
      }
      sort(size);
      const u64 e0 = sh.list[2 * tid], e1 = sh.list[2 * tid + 1];
      const uint32_t o0 = static_cast<uint32_t>(e0 >> 32), o1 = static_cast<uint32_t>(e1 >> 32);
      const u64 w0 = o0 && 2u * tid < most ? weigh(value_of(o0)) : 0, w1 = o1 && 2u * tid + 1 < most ? weigh(value_of(o1)) : 0;
      u64 all;
      const u64 b0 = block_scan(w0 + w1, sh.scan64, &all);
      const u64 limit = limit_of(all);
      const bool k0 = o0 && 2u * tid < most && b0 < limit && w0 >= least, k1 = o1 && 2u * tid + 1 < most && b0 + w0 < limit && w1 >= least;
      // index order: the kept ones by their index's complement, descending
      sh.list[2 * tid] = k0 ? (e0 << 32) | o0 : 0;
      sh.list[2 * tid + 1] = k1 ? (e1 << 32) | o1 : 0;
      if (__syncthreads_or((w0 >= least && o0 && b0 >= limit && b0 < beyond) || (w1 >= least && o1 && b0 + w0 >= limit && b0 + w0 < beyond))) return false;
      sort(size);
      const u64 i0 = sh.list[2 * tid], i1 = sh.list[2 * tid + 1];
      const u64 x0 = i0 ? weigh(value_of(static_cast<uint32_t>(i0))) : 0, x1 = i1 ? weigh(value_of(static_cast<uint32_t>(i1))) : 0;
      const u64 at = block_scan(x0 + x1, sh.scan64, &all);
      const u64 until = until_of(all);
      auto take = [&](u64 item, u64 from, u64 w) {
        if (!(from <= until && until < from + w)) return;
        a.ids[row] = static_cast<int>(~static_cast<uint32_t>(item >> 32));
        if (a.logprob) a.logprob[row] = log_share(weigh, value_of(static_cast<uint32_t>(item)), w, all);
      };
      take(i0, at, x0);
      take(i1, at + x0, x1);
      return true;
    };

    bool done = false;
    // What min_p leaves, roughly: where that is less than top_p's part of all, top_p takes nothing away; where it is no more than the list has
    // room for, the list and the rough mass of all mostly say what top_p takes.  256 rows of 128 K logits in bfloat16: 92 us by the
    // intervals below, 69 so (top_p 0.95, min_p 0.02, temperatures about one).
    bool untouched = false;
    if (sum_now && min_p > 0.0f && weigh.scale == sh.scale) {
      const float bottom = fmaxf(top + sure, -3.4028235e38f);
      float s = 0.0f;
      uint32_t c = 0;
      for (int i = tid; i < vecs; i += SA_THREADS) {
        float v[V];
        read(i, v);
        float m = v[0];
#pragma unroll
        for (int e = 1; e < V; ++e) m = fmaxf(m, v[e]);
        if (!(m >= bottom)) continue;
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (v[e] >= bottom) s += ex2f((v[e] - top) * s2), ++c;
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      c = __reduce_add_sync(0xffffffffu, c);
      if (lane == 0) sh.stay_sum[warp] = s, sh.stay_n[warp] = c;
      meet();
      s = 0.0f, c = 0;
      for (int i = lane; i < ranks * SA_WARPS; i += 32) {  // (every warp of the row adds up the same)
        const SampleShared* q = cluster.map_shared_rank(&sh, i / SA_WARPS);
        s += q->stay_sum[i % SA_WARPS], c += q->stay_n[i % SA_WARPS];
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      c = __reduce_add_sync(0xffffffffu, c);
      untouched = s * (1.0f + 0x1p-10f) < top_p * rough * (1.0f - 0x1p-10f);
      if (!untouched && c <= SA_LIST) {
        const int have = collect(bottom, [&](float v) { return v >= bottom; });
        if (rank == 0) {
          const bool known = finish(have, static_cast<uint32_t>(have), static_cast<double>(rough) * weigh.one);
          if (tid == 0) sh.known = known;
        }
        meet();
        done = *cluster.map_shared_rank(&sh.known, 0) != 0;
      }
    }
    if (by_count) {
      clear();
      for (int i = tid; i < vecs; i += SA_THREADS) {
        float v[V];
        read(i, v);
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (v[e] > -INFINITY) atomicAdd(&sh.count[interval(v[e])], 1u);
      }
      const Found f = find(true, static_cast<uint32_t>(top_k), 0, 0);
      if (f.bin >= 0) {
        if (f.above_n + f.in_n <= SA_LIST) {
          const int have = collect(f.bin == SA_BINS - 1 ? -INFINITY : top - (f.bin + 1.5f) / width, [&](float v) { return v > -INFINITY && interval(v) <= f.bin; });
          if (have >= 0) finish(have, static_cast<uint32_t>(top_k), 0.0);
          done = true;
        } else {
          settle(true, static_cast<uint32_t>(top_k), f, order_of(-3.4028235e38f), order_of(top));
        }
      }
    }
    if (by_mass && !done && !untouched) {
      const Border counted = border;
      const float from = counted.order ? value_of(counted.order) : -3.4028235e38f;
      auto sum_up = [&](float v) {  // over the cluster
#pragma unroll
        for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane == 0) sh.warp_sum[warp] = v;
        meet();
        v = 0.0f;
        for (int i = lane; i < ranks * SA_WARPS; i += 32) v += cluster.map_shared_rank(&sh, i / SA_WARPS)->warp_sum[i % SA_WARPS];
#pragma unroll
        for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
      };
      if (!sum_now) {
        rough = 0.0f;
        for (int i = tid; i < vecs; i += SA_THREADS) {
          float v[V];
          read(i, v);
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (v[e] >= from) rough += ex2f(fmaxf((v[e] - top) * s2, -200.0f));
        }
        rough = sum_up(rough);
      }
      // rough masses of the intervals, in units of 2^-30 of all.  Those whose whole mass is a small part of what top_p leaves out are
      // not looked at (n weights of 2^-bits are 2^-12 of that): behind the window's end, if not behind its start
      clear();
      const float unit = log2f(rough) - 30.0f;
      const float bits = log2f(static_cast<float>(n)) - log2f(fmaxf(1.0f - top_p, 0x1p-24f) * rough) + 12.0f;
      const int cut = bits < 31.0f ? max(1, static_cast<int>(bits * 32.0f) + 1) : SA_BINS - 1;
      for (int i = tid; i < vecs; i += SA_THREADS) {
        float v[V];
        read(i, v);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const int bin = interval(v[e]);
          const uint32_t w = __float2uint_rn(ex2f(fmaf(v[e] - top, s2, -unit)));
          if (bin < cut && v[e] >= from) atomicAdd(&sh.mass_lo[bin], w);
        }
      }
      meet();
      {
        u64 m[2] = {0, 0}, all;
        for (int q = 0; q < ranks; ++q) {
          const uint2 lo = *reinterpret_cast<const uint2*>(cluster.map_shared_rank(&sh, q)->mass_lo + 2 * tid);
          m[0] += lo.x, m[1] += lo.y;
        }
        u64 ahead = block_scan(m[0] + m[1], sh.scan64, &all);
        const double near = static_cast<double>(top_p) * 0x1p30;
        // (each of n logits is rounded to a unit: up to half of one off, all the same way where they are alike)
        const double slack = 0x1p20 + 0.5 * n, low = near - slack, high = near + slack;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int i = 2 * tid + h;
          const double b = static_cast<double>(ahead), e = static_cast<double>(ahead + m[h]);
          if (i == 0 ? e >= low : b < low && e >= low) sh.window[0] = i;
          if (b < high && e >= high) sh.window[1] = i;
          ahead += m[h];
        }
        __syncthreads();
      }
      const int bin0 = sh.window[0], bin1 = sh.window[1];
      // min_p ends before top_p does: top_p takes nothing away
      if (!(min_p > 0.0f && !counted.order && interval(top + sure) < bin0)) {
        // the window as logits (its edges as near as fp32 has them: the part of the mass to either side is for that as well)
        float x_hi = bin0 == 0 ? top : fminf(top, top - (bin0 - 0.5f) / width), x_lo = bin1 == SA_BINS - 1 ? from : fmaxf(from, top - (bin1 + 0.5f) / width);
        // every weight exactly: ahead of the window, in it, all of them; how many in it
        u64 ahead = 0, in = 0, all = 0;
        uint32_t in_n = 0;
        for (int i = tid; i < vecs; i += SA_THREADS) {
          float v[V];
          read(i, v);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const u64 w = v[e] >= from ? weigh(v[e]) : 0;
            all += w;
            if (v[e] > x_hi) ahead += w;
            else if (v[e] >= x_lo) in += w, ++in_n;
          }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
          ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
          in += __shfl_xor_sync(0xffffffffu, in, o);
          all += __shfl_xor_sync(0xffffffffu, all, o);
        }
        in_n = __reduce_add_sync(0xffffffffu, in_n);
        __syncthreads();
        if (tid == 0) sh.above = sh.inside = sh.total = 0, sh.inside_n = 0;
        __syncthreads();
        if (lane == 0) atomicAdd(&sh.above, ahead), atomicAdd(&sh.inside, in), atomicAdd(&sh.total, all), atomicAdd(&sh.inside_n, in_n);
        meet();
        Found f = {0, 0, 0, 0, 0};
        all = 0;
        for (int q = 0; q < ranks; ++q) {
          const SampleShared* s = cluster.map_shared_rank(&sh, q);
          f.above += s->above, f.in += s->inside, f.in_n += s->inside_n, all += s->total;
        }
        // (equals of the counted border that are no candidates)
        const u64 surplus = counted.order ? static_cast<u64>(counted.equals - counted.ties) * weigh(value_of(counted.order)) : 0;
        const double part = ceil(fmax(static_cast<double>(top_p), 0.0) * static_cast<double>(all - surplus));
        want = part >= 1.0 ? static_cast<u64>(part) : 1ull;
        if (!(f.above < want && want <= f.above + f.in)) {  // (the rough masses were further off than they can be)
          f.in_n = 0xffffffffu, f.above = 0;
          x_lo = from, x_hi = top;
        }
        settle(false, 0, f, order_of(x_lo), order_of(x_hi));
        // never past the counted ones
        if (border.order < counted.order || (border.order == counted.order && border.ties > counted.ties && counted.order)) border = counted;
      }
    }
    if (done) {
      meet();  // (no CTA leaves while others read its shared memory)
      return;
    }
  }

  // ---- 3. running sums in index order --------------------------------------------------------------------------------------------------------
  const float border_x = border.order ? value_of(border.order) : -3.4028235e38f;
  const float least_x = fmaxf(border_x, top + sure);  // (top + sure rounds to no more than the least logit that min_p may leave)
  // a thread's own stretch of vectors: an odd number, so that a warp's reads fall into different banks
  const int stretch = ((vecs + SA_THREADS - 1) / SA_THREADS) | 1, v0 = min(vecs, tid * stretch), v1 = min(vecs, v0 + stretch);
  auto any = [&](const float (&v)[V]) {
    float m = v[0];
#pragma unroll
    for (int e = 1; e < V; ++e) m = fmaxf(m, v[e]);
    return m >= least_x;
  };
  auto weight = [&](float v, bool* tie) -> u64 {
    *tie = v == border_x && border.order;
    if (!(v >= least_x) || *tie) return 0;
    const u64 w = weigh(v);
    return w < least ? 0 : w;
  };
  u64 mass = 0;
  uint32_t ties = 0;
  for (int i = v0; i < v1; ++i) {
    float v[V];
    read(i, v);
    if (!any(v)) continue;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      bool tie;
      mass += weight(v[e], &tie);
      ties += tie;
    }
  }
  const u64 mass_inc = warp_scan(mass, lane);
  const uint32_t ties_inc = warp_scan(ties, lane);
  if (lane == 31) sh.warp_mass[warp] = mass_inc, sh.warp_ties[warp] = ties_inc;
  meet();
  u64 tie_w = border.order ? weigh(value_of(border.order)) : 0;
  if (tie_w < least) tie_w = 0;
  const uint32_t allowed = border.ties;
  // sums ahead of this warp, and of all
  u64 ahead = 0, total = 0;
  uint32_t ahead_t = 0, total_t = 0;
  for (int i = lane; i < ranks * SA_WARPS; i += 32) {
    const SampleShared* s = cluster.map_shared_rank(&sh, i / SA_WARPS);
    const u64 m = s->warp_mass[i % SA_WARPS];
    const uint32_t tt = s->warp_ties[i % SA_WARPS];
    total += m, total_t += tt;
    if (i < rank * SA_WARPS + warp) ahead += m, ahead_t += tt;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o), ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
  total_t = __reduce_add_sync(0xffffffffu, total_t), ahead_t = __reduce_add_sync(0xffffffffu, ahead_t);
  total += static_cast<u64>(min(total_t, allowed)) * tie_w;
  ahead += static_cast<u64>(min(ahead_t, allowed)) * tie_w;
  // u times the sum, rounded down; below the sum
  u64 until = static_cast<u64>(floor(fmin(fmax(static_cast<double>(u), 0.0), 1.0) * static_cast<double>(total)));
  if (until >= total) until = total - 1;
  // this thread's stretch: masses and equals of the border ahead of it
  const uint32_t t_from = ahead_t + ties_inc - ties;
  const u64 above_ahead = ahead - static_cast<u64>(min(ahead_t, allowed)) * tie_w + mass_inc - mass;
  const u64 from = above_ahead + static_cast<u64>(min(t_from, allowed)) * tie_w;
  const u64 to = above_ahead + mass + static_cast<u64>(min(t_from + ties, allowed)) * tie_w;
  const unsigned who = __ballot_sync(0xffffffffu, from <= until && until < to);
  if (who) {  // (one thread of the cluster): its warp walks its stretch, an element a lane
    const int l = __ffs(who) - 1;
    u64 run = __shfl_sync(0xffffffffu, from, l);
    uint32_t seen = __shfl_sync(0xffffffffu, t_from, l);
    const int e0 = __shfl_sync(0xffffffffu, v0, l) * V, e1 = __shfl_sync(0xffffffffu, v1, l) * V;
    for (int e = e0; e < e1; e += 32) {
      float v = __uint_as_float(0x7fc00000u);
      if constexpr (KEPT) {
        if (e + lane < e1) {
          if constexpr (T == MIMIR_B200_T_F32) v = reinterpret_cast<const float*>(dyn)[e + lane];
          else if constexpr (T == MIMIR_B200_T_F16) v = __half2float(reinterpret_cast<const __half*>(dyn)[e + lane]);
          else v = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(dyn)[e + lane]);
        }
      } else {
        if (e + lane < min(e1, mine)) v = logit<T>(x, first + e + lane);
      }
      bool tie;
      u64 w = weight(v, &tie);
      const unsigned equal = __ballot_sync(0xffffffffu, tie);
      if (tie && seen + __popc(equal & ((1u << lane) - 1)) < allowed) w = tie_w;
      const u64 inc = warp_scan(w, lane);
      if (run + inc - w <= until && until < run + inc) {
        a.ids[row] = first + e + lane;
        if (a.logprob) a.logprob[row] = log_share(weigh, v, w, total);
      }
      run += __shfl_sync(0xffffffffu, inc, 31);
      seen += __popc(equal);
      if (run > until) break;
    }
  }
  meet();
}

template <int T, bool KEPT>
int launch_as(const SampleLaunch& s, int cluster, int slice, cudaStream_t st) {
  const size_t smem = KEPT ? static_cast<size_t>(slice) * type_bytes(T) : 0;
  static PerDeviceOnce once;
  MB_TRY(once.run([]() -> int {
    MB_CUDA(cudaFuncSetAttribute(sample_rows_kernel<T, KEPT>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(SA_LARGE)));
    return MIMIR_B200_OK;
  }));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(s.rows * cluster));
  cfg.blockDim = dim3(SA_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  static const Powers powers = [] {
    Powers p;
    for (int k = 0; k < 64; ++k) p.v[k] = std::exp2(k / 64.0);
    return p;
  }();
  MB_CUDA(cudaLaunchKernelEx(&cfg, sample_rows_kernel<T, KEPT>, s, slice, powers));
  count_launch();
  return MIMIR_B200_OK;
}
template <int T>
int launch_t(const SampleLaunch& s, cudaStream_t st) {
  constexpr int STEP = 32 * Vec<T>::N;  // a warp's vectors
  // As few CTAs as hold the row two to an SM, and one to an SM rather than eight (clusters of eight start late and leave SMs idle): 128 rows of
  // 128 K fp32 logits 57 us in four, 71 in eight.  More while half the SMs are idle and each keeps a few thousand logits: 64 rows of 32 K
  // 12 us in one, 26 in eight; one of 128 K 13 in eight.
  int cluster = 1;
  auto holds = [&](int n) { return static_cast<long long>(n) * static_cast<long long>((n < 4 ? SA_SLICE : SA_LARGE) / type_bytes(T)) >= s.n; };
  while (cluster < 8 && (!holds(cluster) || (2 * s.rows * cluster < ctx().sm_count && s.n / cluster >= 4096))) cluster *= 2;
  const long long each = (s.n + cluster - 1) / cluster;
  const int slice = static_cast<int>((each + STEP - 1) / STEP * STEP);
  if (s.rows * cluster > 0x7fffffffLL) return fail(MIMIR_B200_E_INVALID, "sample_rows: too many rows for one call");
  return static_cast<size_t>(slice) * type_bytes(T) <= SA_LARGE ? launch_as<T, true>(s, cluster, slice, st) : launch_as<T, false>(s, cluster, slice, st);
}

}  // namespace

int launch_sample_rows(const SampleLaunch& s, cudaStream_t st) {
  if (s.type == MIMIR_B200_T_F32) return launch_t<MIMIR_B200_T_F32>(s, st);
  if (s.type == MIMIR_B200_T_F16) return launch_t<MIMIR_B200_T_F16>(s, st);
  return launch_t<MIMIR_B200_T_BF16>(s, st);
}

}  // namespace mb
