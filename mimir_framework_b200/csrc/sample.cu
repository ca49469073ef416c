// sample.cu — a token from each row of logits by a given random number: temperature, top-k, top-p and min-p.
//
//   w_i = exp((x_i - max) / T).  Candidates in the order (w descending, index ascending): the first top_k of them; of those the shortest
//   beginning that holds top_p of their mass; of those w_i >= min_p.  The token is the first index (in index order) at which the running
//   sum of the candidates' w exceeds u times their whole sum.
//
// A row is read once: a cluster of CTAs keeps it in shared memory, a slice each, and meets through distributed shared memory.
//   1. the largest logit
//   2. with top_k or top_p: counts (and masses) of 1024 intervals of (max - x) / T, and the interval in which the border lies.  Where
//      what can still be taken is at most 1024 logits, they are gathered, sorted and finished in one CTA.  Else the border itself is found:
//      the interval's logits are sorted, or divided again by their bits while they are more than 1024
//   3. masses of the warps' stretches of the row in index order; the stretch in which u falls is walked
// Sums are compared with borders, so every w is an integer (w times a power of two that leaves room for n of them): sums of integers are
// the same in every order and division of the work.  w comes from a table of 2^(k / 64) and four terms of the exponential series in
// fp64, relative error under 2^-44.  A large batch waits for the arithmetic: the weights (eleven fp64 operations each), and the two
// to three additions in shared memory of each logit that an interval of its own is kept for; those whose mass cannot reach the border
// are added up in registers (an fp32 sum of the weights says which).
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
  uint32_t list_n;
  u64 scan64[33];
  uint32_t scan32[33];
  // read by the cluster's other CTAs
  float top;
  int first;
  uint32_t low, high;
  uint32_t total_n;
  u64 total;
  Found found;
  Border border;
  uint32_t least_n;                                             // candidates up to the last interval that min_p leaves
  float rough;
  u64 warp_mass[SA_WARPS];
  uint32_t warp_ties[SA_WARPS];
};

struct Weigh {
  double top, scale;  // log2(e) / T
  double one, magic;  // what a weight of 1 is as an integer, 2^52
  const double* table;
  // x <= top; 0 for what is not a candidate
  __device__ __forceinline__ u64 operator()(float x) const {
    const double y = fmax((static_cast<double>(x) - top) * scale, -600.0);  // (what is not a number becomes 2^-600, zero)
    const double s = y + 105553116266496.0;  // 1.5 * 2^46: y rounded to 64ths in the low bits
    const int k = __double2loint(s);
    const double r = (y - (s - 105553116266496.0)) * 0.69314718055994530942;
    double p = fma(r, 1.0 / 24, 1.0 / 6);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    const double t = table[k & 63];
    const double w = __hiloint2double(__double2hiint(t) + ((k >> 6) << 20), __double2loint(t)) * p;
    return static_cast<u64>(__double_as_longlong(fma(w, one, magic)) & 0xfffffffffffffll);
  }
};

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
__global__ void __launch_bounds__(SA_THREADS, 2) sample_rows_kernel(const __grid_constant__ SampleLaunch a, int slice) {
  constexpr int V = Vec<T>::N;
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ SampleShared sh;
  const cg::cluster_group cluster = cg::this_cluster();
  const int ranks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
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

  // ---- 1. the largest -------------------------------------------------------------------------------------------------------------------
  float top = -INFINITY;
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
#pragma unroll
        for (int e = 0; e < V; ++e) top = fmaxf(top, f[e]);
      }
    }
  } else {
    for (int i = tid; i < vecs; i += SA_THREADS) {
      float f[V];
      read(i, f);
#pragma unroll
      for (int e = 0; e < V; ++e) top = fmaxf(top, f[e]);
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (tid < 64) sh.table[tid] = exp2(tid * (1.0 / 64));
  if (tid == 0) sh.list_n = 0;
  if (lane == 0) reinterpret_cast<float*>(sh.scan32)[warp] = top;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < SA_WARPS; ++w) top = fmaxf(top, reinterpret_cast<float*>(sh.scan32)[w]);
    sh.top = top;
  }
  cluster.sync();
  top = -INFINITY;
  for (int c = 0; c < ranks; ++c) top = fmaxf(top, *cluster.map_shared_rank(&sh.top, c));

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
    cluster.sync();
    if (rank == 0 && tid == 0) {
      for (int c = 0; c < ranks; ++c) at = min(at, *cluster.map_shared_rank(&sh.first, c));
      a.ids[row] = top == -INFINITY ? -1 : at;
      if (a.logprob) a.logprob[row] = top == -INFINITY ? -INFINITY : 0.0f;
    }
    cluster.sync();  // (no CTA leaves while others read its shared memory)
    return;
  }
  int room = 0;  // n <= 2^room
  while ((1ll << room) < n) ++room;
  Weigh weigh;
  weigh.top = top;
  weigh.scale = 1.4426950408889634074 / static_cast<double>(t);
  weigh.one = static_cast<double>(1ull << min(62 - room, 51));
  weigh.magic = 4503599627370496.0;
  weigh.table = sh.table;
  // logits surely below min_p are left out before they are weighed (2^-10 of slack for the fp32 product)
  const double least_w = min_p > 0.0f ? fmin(static_cast<double>(min_p), 1.0) : 0.0;
  const u64 least = static_cast<u64>(ceil(least_w * weigh.one));
  const float sure = min_p > 0.0f ? static_cast<float>((log2(least_w) - 1e-3) / weigh.scale * 1.0001) : -INFINITY;  // of x - max

  // ---- 2. the border ---------------------------------------------------------------------------------------------------------------------
  const bool by_count = top_k > 0 && top_k < n, by_mass = top_p < 1.0f;
  Border border = {0, 0, 0};
  if (by_count || by_mass) {
    const float width = static_cast<float>(32.0 * weigh.scale);  // of (max - x), in intervals
    const int share = SA_BINS / ranks;                           // intervals that this CTA adds up
    int cut = SA_BINS - 1;                                       // from this one on they are one
    auto interval = [&](float v) {
      const int i = __float2int_rz((top - v) * width);
      return i < cut ? i : SA_BINS - 1;
    };
    auto add_mass = [&](int bin, u64 w) {
      const uint32_t lo = static_cast<uint32_t>(w), old = atomicAdd(&sh.mass_lo[bin], lo);
      const uint32_t hi = static_cast<uint32_t>(w >> 32) + (old + lo < old ? 1u : 0u);
      if (hi) atomicAdd(&sh.mass_hi[bin], hi);
    };
    auto clear = [&]() {
      __syncthreads();
      for (int i = tid; i < SA_BINS; i += SA_THREADS) sh.count[i] = sh.mass_lo[i] = sh.mass_hi[i] = 0;
      if (tid == 0) sh.found.bin = -1;
      __syncthreads();
    };
    // the interval in which the candidates reach want_n in number or a part of the mass, counted from (above_n, above)
    u64 whole = 0, want = 0;
    auto find = [&](bool number, uint32_t want_n, uint32_t above_n, u64 above, int last) {
      cluster.sync();
      u64 m[2] = {0, 0};
      uint32_t c[2] = {0, 0};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int i = 2 * tid + h;
        if (i >= share) continue;
        for (int q = 0; q < ranks; ++q) {
          const SampleShared* s = cluster.map_shared_rank(&sh, q);
          c[h] += s->count[rank * share + i];
          if (!number) m[h] += (static_cast<u64>(s->mass_hi[rank * share + i]) << 32) + s->mass_lo[rank * share + i];
        }
      }
      u64 all = 0, mb = 0;
      uint32_t all_n;
      if (!number) mb = block_scan(m[0] + m[1], sh.scan64, &all);
      uint32_t cb = block_scan(c[0] + c[1], sh.scan32, &all_n);
      if (tid == 0) sh.total = all, sh.total_n = all_n;
      cluster.sync();
      u64 sum = 0;
      for (int q = 0; q < ranks; ++q) {
        const SampleShared* s = cluster.map_shared_rank(&sh, q);
        const u64 mq = s->total;
        if (q < rank) mb += mq, cb += s->total_n;
        sum += mq;
      }
      if (!number && want == 0) {  // (the first of the mass's levels)
        const Border& k = border;  // equals of the counted border that are not candidates
        whole = sum - (k.order ? static_cast<u64>(k.equals - k.ties) * weigh(value_of(k.order)) : 0);
        const double part = ceil(fmax(static_cast<double>(top_p), 0.0) * static_cast<double>(whole));
        want = part >= 1.0 ? static_cast<u64>(part) : 1ull;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int i = 2 * tid + h;
        if (i < share && c[h] > 0) {
          const u64 ahead = above + mb;
          const uint32_t ahead_n = above_n + cb;
          if (number ? ahead_n < want_n && ahead_n + c[h] >= want_n : ahead < want && ahead + m[h] >= want) {
            Found f;
            f.bin = rank * share + i;
            f.above = ahead, f.above_n = ahead_n, f.in = m[h], f.in_n = c[h];
            for (int q = 0; q < ranks; ++q) cluster.map_shared_rank(&sh, q)->found = f;
          }
        }
        mb += m[h], cb += c[h];
        if (i < share && rank * share + i == last)
          for (int q = 0; q < ranks; ++q) cluster.map_shared_rank(&sh, q)->least_n = above_n + cb;
      }
      cluster.sync();
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
    // what `pick` says yes to into the first CTA's list; true there, whose list is filled up with zeros to a power of two
    int size = 32;
    auto collect = [&](auto&& pick) {
      SampleShared* home = cluster.map_shared_rank(&sh, 0);
      for (int i = tid; i < vecs; i += SA_THREADS) {
        float v[V];
        read(i, v);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const uint32_t o = order_of(v[e]);
          if (o && pick(o, v[e])) {
            const uint32_t at = atomicAdd(&home->list_n, 1u);
            if (at < SA_LIST) home->list[at] = (static_cast<u64>(o) << 32) | ~static_cast<uint32_t>(first + i * V + e);
          }
        }
      }
      cluster.sync();
      if (rank != 0) return false;
      const int have = static_cast<int>(min(sh.list_n, static_cast<uint32_t>(SA_LIST)));
      while (size < have) size *= 2;
      for (int i = tid; i < SA_LIST; i += SA_THREADS)
        if (i >= have) sh.list[i] = 0;
      __syncthreads();
      if (tid == 0) sh.list_n = 0;
      sort(size);
      return true;
    };

    // The border in an interval found: level by level, then sorted or a single order.
    auto settle = [&](bool number, uint32_t want_n, Found f) {
      const int value_bin = f.bin;
      uint32_t range_lo = max(1u, border.order), range_hi = 0xffffffffu;  // (what top_k left out is no member)
      int shift = -1;
      auto member = [&](uint32_t o, float v) { return o >= range_lo && o <= range_hi && interval(v) == value_bin; };
      while (f.in_n > SA_LIST && shift != 0) {
        // their range of orders, divided evenly, the largest first
        uint32_t lo = 0xffffffffu, hi = 0;
        for (int i = tid; i < vecs; i += SA_THREADS) {
          float v[V];
          read(i, v);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const uint32_t o = order_of(v[e]);
            if (o && member(o, v[e])) lo = min(lo, o), hi = max(hi, o);
          }
        }
        lo = __reduce_min_sync(0xffffffffu, lo), hi = __reduce_max_sync(0xffffffffu, hi);
        __syncthreads();
        if (tid == 0) sh.low = 0xffffffffu, sh.high = 0;
        clear();
        if (lane == 0) atomicMin(&sh.low, lo), atomicMax(&sh.high, hi);
        cluster.sync();
        lo = 0xffffffffu, hi = 0;
        for (int q = 0; q < ranks; ++q) lo = min(lo, *cluster.map_shared_rank(&sh.low, q)), hi = max(hi, *cluster.map_shared_rank(&sh.high, q));
        shift = 0;
        while (((hi - lo) >> shift) >= SA_BINS) ++shift;
        for (int i = tid; i < vecs; i += SA_THREADS) {
          float v[V];
          read(i, v);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const uint32_t o = order_of(v[e]);
            if (o && member(o, v[e])) {
              atomicAdd(&sh.count[(hi - o) >> shift], 1u);
              if (!number) add_mass(static_cast<int>((hi - o) >> shift), weigh(v[e]));
            }
          }
        }
        f = find(number, want_n, f.above_n, f.above, -1);
        if (f.bin < 0) return;  // (never: the sums are exact)
        range_hi = hi - (static_cast<uint32_t>(f.bin) << shift);
        const uint32_t span = (1u << shift) - 1;
        range_lo = range_hi - lo < span ? lo : range_hi - span;
      }
      if (f.in_n <= SA_LIST && shift != 0) {
        if (collect(member)) {
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
        cluster.sync();
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
    // The few that can still be taken, in the first CTA: top_k, top_p and min_p in the sorted list, then u in index order.
    auto finish = [&](int last) {
      if (!collect([&](uint32_t, float v) { return interval(v) <= last; })) return;
      const u64 e0 = sh.list[2 * tid], e1 = sh.list[2 * tid + 1];
      const uint32_t o0 = static_cast<uint32_t>(e0 >> 32), o1 = static_cast<uint32_t>(e1 >> 32);
      const uint32_t most = by_count ? static_cast<uint32_t>(top_k) : 0xffffffffu;
      const u64 w0 = o0 && 2u * tid < most ? weigh(value_of(o0)) : 0, w1 = o1 && 2u * tid + 1 < most ? weigh(value_of(o1)) : 0;
      u64 all, limit = ~0ull;
      const u64 b0 = block_scan(w0 + w1, sh.scan64, &all);
      if (by_mass) {
        const double part = ceil(fmax(static_cast<double>(top_p), 0.0) * static_cast<double>(by_count ? all : whole));
        limit = part >= 1.0 ? static_cast<u64>(part) : 1ull;
      }
      const bool k0 = o0 && 2u * tid < most && b0 < limit && w0 >= least, k1 = o1 && 2u * tid + 1 < most && b0 + w0 < limit && w1 >= least;
      // index order: the kept ones by their index's complement, descending
      sh.list[2 * tid] = k0 ? (e0 << 32) | o0 : 0;
      sh.list[2 * tid + 1] = k1 ? (e1 << 32) | o1 : 0;
      __syncthreads();
      sort(size);
      const u64 i0 = sh.list[2 * tid], i1 = sh.list[2 * tid + 1];
      const u64 x0 = i0 ? weigh(value_of(static_cast<uint32_t>(i0))) : 0, x1 = i1 ? weigh(value_of(static_cast<uint32_t>(i1))) : 0;
      const u64 at = block_scan(x0 + x1, sh.scan64, &all);
      u64 until = static_cast<u64>(floor(fmin(fmax(static_cast<double>(u), 0.0), 1.0) * static_cast<double>(all)));
      if (until >= all) until = all - 1;
      auto take = [&](u64 item, u64 from, u64 w) {
        if (!(from <= until && until < from + w)) return;
        a.ids[row] = static_cast<int>(~static_cast<uint32_t>(item >> 32));
        if (a.logprob) a.logprob[row] = static_cast<float>(log(static_cast<double>(w) / static_cast<double>(all)));
      };
      take(i0, at, x0);
      take(i1, at + x0, x1);
    };

    const int last_min = min_p > 0.0f ? interval(top + sure) : SA_BINS - 1;  // intervals behind it are below min_p
    bool done = false;
    if (by_count) {
      clear();
      for (int i = tid; i < vecs; i += SA_THREADS) {
        float v[V];
        read(i, v);
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (v[e] > -INFINITY) atomicAdd(&sh.count[interval(v[e])], 1u);
      }
      const Found f = find(true, static_cast<uint32_t>(top_k), 0, 0, last_min);
      if (f.bin >= 0) {
        if (f.above_n + f.in_n <= SA_LIST) {
          finish(f.bin);
          done = true;
        } else {
          settle(true, static_cast<uint32_t>(top_k), f);
        }
      }
    }
    if (by_mass && !done) {
      const Border counted = border;
      if (!counted.order && slice >= 4096) {
        // a rough sum first: intervals whose whole mass cannot reach what top_p leaves out need not be kept apart
        const float s = static_cast<float>(weigh.scale);
        float sum = 0.0f;
        for (int i = tid; i < vecs; i += SA_THREADS) {
          float v[V];
          read(i, v);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            float w;
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(fmaxf((v[e] - top) * s, -200.0f)));
            sum += w;
          }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        __syncthreads();
        if (lane == 0) reinterpret_cast<float*>(sh.scan32)[warp] = sum;
        __syncthreads();
        if (tid == 0) {
          for (int w = 1; w < SA_WARPS; ++w) sum += reinterpret_cast<float*>(sh.scan32)[w];
          sh.rough = sum;
        }
        cluster.sync();
        sum = 0.0f;
        for (int q = 0; q < ranks; ++q) sum += *cluster.map_shared_rank(&sh.rough, q);
        const float bits = log2f(static_cast<float>(n) / ((1.0f - top_p) * sum)) + 1.0f;  // n weights of 2^-bits are half of what is left out
        cut = bits < 31.0f ? max(1, static_cast<int>(bits * 32.0f) + 1) : SA_BINS - 1;
      }
      clear();
      const float from = counted.order ? value_of(counted.order) : -INFINITY;
      u64 rest = 0;
      uint32_t rest_n = 0;
      for (int i = tid; i < vecs; i += SA_THREADS) {
        float v[V];
        read(i, v);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          if (counted.order && !(v[e] >= from)) continue;
          const u64 w = weigh(v[e]);
          const int bin = interval(v[e]);
          if (bin < SA_BINS - 1 && v[e] > -INFINITY) {
            atomicAdd(&sh.count[bin], 1u);
            add_mass(bin, w);
          } else {
            rest += w;
            rest_n += v[e] > -INFINITY;
          }
        }
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) rest += __shfl_xor_sync(0xffffffffu, rest, o);
      rest_n = __reduce_add_sync(0xffffffffu, rest_n);
      if (lane == 0 && rest_n) {
        atomicAdd(&sh.count[SA_BINS - 1], rest_n);
        add_mass(SA_BINS - 1, rest);
      }
      const int last = min_p > 0.0f ? interval(top + sure) : SA_BINS - 1;
      const Found f = find(false, 0, 0, 0, last);
      if (f.bin >= 0) {
        const bool least_first = last < f.bin;  // min_p leaves nothing near top_p's border
        if (!counted.order && (least_first ? sh.least_n : f.above_n + f.in_n) <= SA_LIST) {
          finish(least_first ? last : f.bin);
          done = true;
        } else if (!least_first || counted.order) {
          settle(false, 0, f);
          // never past the counted ones
          if (border.order < counted.order || (border.order == counted.order && border.ties > counted.ties && counted.order)) border = counted;
        }
      }
    }
    if (done) {
      cluster.sync();  // (no CTA leaves while others read its shared memory)
      return;
    }
  }

  // ---- 3. running sums in index order --------------------------------------------------------------------------------------------------------
  const float border_x = border.order ? value_of(border.order) : -INFINITY;
  const int per_warp = (vecs + SA_WARPS - 1) / SA_WARPS, v0 = min(vecs, warp * per_warp), v1 = min(vecs, v0 + per_warp);
  auto weight = [&](float v, bool* tie) -> u64 {
    *tie = false;
    if (!(v - top >= sure) || !(v >= border_x)) return 0;
    if (v == border_x && border.order) {
      *tie = true;
      return 0;
    }
    const u64 w = weigh(v);
    return w < least ? 0 : w;
  };
  u64 mass = 0;
  uint32_t ties = 0;
  for (int i = v0 + lane; i < v1; i += 32) {
    float v[V];
    read(i, v);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      bool tie;
      mass += weight(v[e], &tie);
      ties += tie;
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) mass += __shfl_xor_sync(0xffffffffu, mass, o);
  ties = __reduce_add_sync(0xffffffffu, ties);
  if (lane == 0) sh.warp_mass[warp] = mass, sh.warp_ties[warp] = ties;
  cluster.sync();
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
  const u64 warp_all = mass + static_cast<u64>(min(ahead_t + ties, allowed) - min(ahead_t, allowed)) * tie_w;
  // u times the sum, rounded down; below the sum
  u64 until = static_cast<u64>(floor(fmin(fmax(static_cast<double>(u), 0.0), 1.0) * static_cast<double>(total)));
  if (until >= total) until = total - 1;
  if (ahead <= until && until < ahead + warp_all) {  // (one warp of the cluster)
    u64 run = ahead;
    uint32_t seen = ahead_t;
    for (int i0 = v0; i0 < v1; i0 += 32) {
      float v[V];
      u64 w[V], sum = 0;
      uint32_t mine_t = 0;
      bool tie[V];
      const bool there = i0 + lane < v1;
      if (there) read(i0 + lane, v);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        tie[e] = false;
        w[e] = there ? weight(v[e], &tie[e]) : 0;
        mine_t += tie[e];
      }
      uint32_t t_at = seen + warp_scan(mine_t, lane) - mine_t;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if (tie[e] && t_at++ < allowed) w[e] = tie_w;
        sum += w[e];
      }
      const u64 inc = warp_scan(sum, lane);
      u64 at = run + inc - sum;
      if (at <= until && until < run + inc) {
        bool done = false;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          at += w[e];
          if (!done && at > until) {
            done = true;
            a.ids[row] = first + (i0 + lane) * V + e;
            if (a.logprob) a.logprob[row] = static_cast<float>(log(static_cast<double>(w[e]) / static_cast<double>(total)));
          }
        }
      }
      run = __shfl_sync(0xffffffffu, run + inc, 31);
      seen += __reduce_add_sync(0xffffffffu, mine_t);
      if (run > until) break;
    }
  }
  cluster.sync();
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
  MB_CUDA(cudaLaunchKernelEx(&cfg, sample_rows_kernel<T, KEPT>, s, slice));
  count_launch();
  return MIMIR_B200_OK;
}
template <int T>
int launch_t(const SampleLaunch& s, cudaStream_t st) {
  constexpr int STEP = 32 * Vec<T>::N;  // a warp's vectors
  // as few CTAs as hold the row two to an SM, more while SMs would be idle and each keeps a few thousand logits
  const int fits = static_cast<int>(SA_SLICE) / type_bytes(T);
  int cluster = 1;
  while (cluster < 8 && (static_cast<long long>(cluster) * fits < s.n || (s.rows * cluster < 2LL * ctx().sm_count && s.n / cluster >= 4096))) cluster *= 2;
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
