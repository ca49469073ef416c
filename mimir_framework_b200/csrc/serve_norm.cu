// serve_norm.cu — rows between a layer's products: residual addition, root-mean-square norm, a narrower type.
//
//   s = x + residual,  v = s / sqrt(mean(s^2) + eps) * gamma,  y = v, or codes of 8 bits and their scale
//
// One pass: a row lies in the registers of the threads that share it (eight elements at a time, so that loads and stores are 16 bytes), its
// sum of squares and, for codes, its largest magnitude are each one meeting of these threads.  Statistics are fp32.  Codes of rows
// without the norm are those of an IEEE division by the scale, as in the cache; of a norm's values see finish_row.
#include <algorithm>

#include "common.h"
#include "epilogue.cuh"
#include "launch.cuh"
#include "layer.cuh"
#include "paged.cuh"
#include "sm100_ptx.cuh"

namespace mb {
namespace {

constexpr int NR_WARP_THREADS = 128;  // of a CTA whose warps have a row each
constexpr int MEETINGS = 3;           // of a row's threads, over words of their own (a CTA that meets has 96 threads at least)
constexpr int NR_MAX_STAGES = 8, NR_RING = 108 * 1024;  // rows ahead at most, bytes of them in a CTA

struct NormParams {
  const char* x;
  const char* residual;
  char* sum;
  const float* gamma;
  char* y;
  float* y_scale;
  long long x_row, residual_row, sum_row, y_row;  // bytes
  int rows, n, norm, early, stages;
  bool vec;  // all rows (and gamma) start on 16 bytes, codes on 8
  float eps, inv_n;
  int* err_word;
};

// 16 bytes from byte `at` (even, below 16, the same for a row) of two times 16
__device__ __forceinline__ uint4 bytes_from(const uint4& a, const uint4& b, int at) {
  uint32_t w[5];
  switch (at >> 2) {
    case 0: w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x; break;
    case 1: w[0] = a.y, w[1] = a.z, w[2] = a.w, w[3] = b.x, w[4] = b.y; break;
    case 2: w[0] = a.z, w[1] = a.w, w[2] = b.x, w[3] = b.y, w[4] = b.z; break;
    default: w[0] = a.w, w[1] = b.x, w[2] = b.y, w[3] = b.z, w[4] = b.w;
  }
  if (!(at & 2)) return make_uint4(w[0], w[1], w[2], w[3]);
  return make_uint4(__funnelshift_r(w[0], w[1], 16), __funnelshift_r(w[1], w[2], 16), __funnelshift_r(w[2], w[3], 16), __funnelshift_r(w[3], w[4], 16));
}

// A thread's eight elements of a vector, those from n on zero.  VEC: all rows start on 16 bytes.  Else neighbours from column `col` on, or (`apart` > 0,
// where x is F32) every `apart`-th, so that a warp's lanes have neighbours.  Rows of 16 bits off their boundary come in the two times 16 bytes that hold a vector (both
// hold some of it) and leave as whole 16 bytes that a lane makes up with its neighbour's: every lane of a warp has to call.  (5 638 rows of 5 871
// halves with residual 67 us; element by element 137, 122 with lanes side by side.)
template <int T, bool VEC>
__device__ __forceinline__ Raw8<T> row_load8(const char* row, int col, int n, int apart) {
  const char* const p = row + static_cast<long long>(col) * type_bytes(T);
  const int off = VEC ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15);
  if ((VEC || apart == 0) && col + 8 <= n && off == 0) return load8<T>(p);
  Raw8<T> r;
  if constexpr (type_bytes(T) == 2 && !VEC) {
    if (col + 8 <= n) {
      const uint4 v = bytes_from(*reinterpret_cast<const uint4*>(p - off), *reinterpret_cast<const uint4*>(p - off + 16), off);
      r.w[0] = v.x, r.w[1] = v.y, r.w[2] = v.z, r.w[3] = v.w;
      return r;
    }
  }
  const int step = !VEC && apart ? apart : 1;
#pragma unroll
  for (uint32_t& w : r.w) w = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int at = col + e * step;
    if (at >= n) break;
    if constexpr (type_bytes(T) == 4) r.w[e] = reinterpret_cast<const uint32_t*>(row)[at];
    else r.w[e / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(row)[at]) << (16 * (e & 1));
  }
  return r;
}
template <int T, bool VEC>
__device__ __forceinline__ void row_store8(char* row, int col, int n, int apart, const Raw8<T>& r) {
  char* const p = row + static_cast<long long>(col) * type_bytes(T);
  const bool whole = col + 8 <= n;
  int first = 0, last = 8;  // the elements that go one by one
  if constexpr (VEC) {
    if (whole) {
      store8<T>(p, r);
      return;
    }
  } else if constexpr (type_bytes(T) == 2) {
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15);  // (the same for all of a row)
    if (apart == 0 && off) {
      const int lane = threadIdx.x & 31;
      const uint4 mine = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
      uint4 before;
      before.x = __shfl_up_sync(0xffffffffu, mine.x, 1), before.y = __shfl_up_sync(0xffffffffu, mine.y, 1);
      before.z = __shfl_up_sync(0xffffffffu, mine.z, 1), before.w = __shfl_up_sync(0xffffffffu, mine.w, 1);
      const bool next_whole = __shfl_down_sync(0xffffffffu, static_cast<int>(whole), 1) && lane < 31;
      if (whole && lane > 0) {
        *reinterpret_cast<uint4*>(p - off) = bytes_from(before, mine, 16 - off);
        first = 8 - off / 2;
      }
      if (whole && next_whole) last = 8 - off / 2;  // (the next lane has the rest)
    } else if (apart == 0 && whole) {
      store8<T>(p, r);
      return;
    }
  } else if (apart == 0 && whole && (reinterpret_cast<uintptr_t>(p) & (type_bytes(T) == 1 ? 7 : 15)) == 0) {
    store8<T>(p, r);
    return;
  }
  const int step = !VEC && apart ? apart : 1;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int at = col + e * step;
    if (e < first || e >= last || at >= n) continue;
    if constexpr (type_bytes(T) == 4) reinterpret_cast<uint32_t*>(row)[at] = r.w[e];
    else if constexpr (type_bytes(T) == 2) reinterpret_cast<uint16_t*>(row)[at] = static_cast<uint16_t>(r.w[e / 2] >> (16 * (e & 1)));
    else reinterpret_cast<uint8_t*>(row)[at] = static_cast<uint8_t>(r.w[e / 4] >> (8 * (e & 3)));
  }
}

// Two values in a register pair, for the instructions that work on both (epilogue.cuh); eight elements are four pairs.
using Pair = unsigned long long;
template <int T>
__device__ __forceinline__ void to_pairs(const Raw8<T>& r, Pair (&f)[4]) {
  float v[8];
  unpack8<T>(r, v);
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = pack2(v[2 * i], v[2 * i + 1]);
}
__device__ __forceinline__ void from_pairs(const Pair (&f)[4], float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) unpack2(f[i], v[2 * i], v[2 * i + 1]);
}
// the larger of two magnitudes and a third number, not a number if one of them is none
__device__ __forceinline__ float max_abs3(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// A number of each thread of a row, joined; every thread has the result.  `buf`: 24 words of the CTA's.  Between two meetings over the same words
// lies another one over others, or a barrier: a thread may still read when the next has gone on.
template <bool WARP, bool MAX>
__device__ __forceinline__ float meet(float v, float* buf) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const float w = __shfl_xor_sync(0xffffffffu, v, o);
    v = MAX ? fmaxf(v, w) : v + w;
  }
  if constexpr (WARP) return v;
  const int warps = blockDim.x >> 5;
  if (warps == 1) return v;
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  // (words of no warp are zero: neither sums nor magnitudes mind)
  const float4* words = reinterpret_cast<const float4*>(buf);
  auto four = [](float4 s) { return MAX ? fmaxf(fmaxf(s.x, s.y), fmaxf(s.z, s.w)) : (s.x + s.y) + (s.z + s.w); };
  const float a = four(words[0]), b = four(words[1]);
  v = MAX ? fmaxf(a, b) : a + b;
  if (warps > 8) {
    const float c = four(words[2]), d = four(words[3]);
    v = MAX ? fmaxf(v, fmaxf(c, d)) : v + (c + d);
    if (warps > 16) {
      const float e = four(words[4]), g = four(words[5]);
      v = MAX ? fmaxf(v, fmaxf(e, g)) : v + (e + g);
    }
  }
  return v;
}
// 1 / sqrt(x), off by less than 1.5 units of 2^-24: the approximation (2^-22) and a Newton step
__device__ __forceinline__ float root_reciprocal(float x) {
  float r;
  asm("rsqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  const float e = fmaf(-x * r, r, 1.0f);
  return fabsf(e) < 1.0f ? fmaf(0.5f * r, e, r) : r;  // (zero and infinity: as the approximation has them)
}

// A row from the sums s that its threads hold on: V vectors of eight elements each; WARP: a row to a warp, else to the CTA.  Instructions bound it
// where memory does not, so two elements go through one wherever there is such a one (8 192 rows of 4 096 with residual to codes took 37 M
// instructions and 47 us element by element, 28 M and 40 us so).
// NORM: 0, 1, or -1, which is what the call says (the ring's registers do not hold both kinds of codes).
template <int TX, int TY, int V, bool WARP, bool VEC, int NORM = -1>
__device__ __forceinline__ void finish_row(const NormParams& p, int row, int t, int step, int apart, Pair (&f)[V][4], float (&buf)[MEETINGS][32]) {
  const int col0 = !VEC && apart ? t : t * 8;
  if (p.sum) {
    char* const sum = p.sum + row * p.sum_row;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float s[8];
      from_pairs(f[v], s);
      row_store8<TX, VEC>(sum, v * step + col0, p.n, apart, pack8<TX>(s));
    }
  }
  const bool norm = NORM < 0 ? p.norm != 0 : NORM == 1;
  float root = 1.0f;  // that the elements still lack
  if (norm) {
    Pair q2 = pack2(0.0f, 0.0f);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      Pair a = mul2(f[v][0], f[v][0]);
#pragma unroll
      for (int i = 1; i < 4; ++i) a = fma2(f[v][i], f[v][i], a);
      q2 = add2(q2, a);
    }
    float q0, q1;
    unpack2(q2, q0, q1);
    const float q = meet<WARP, false>(q0 + q1, buf[0]), mean = fmaf(q, p.inv_n, p.eps);
    float r = root_reciprocal(mean);
    if (!(q < INFINITY) || mean < 0x1p-100f) {
      // squares beyond fp32's range (or below it, next to no eps): once more with the row's largest near one
      float top = 0.0f, rest = 0.0f;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float s[8];
        from_pairs(f[v], s);
#pragma unroll
        for (int e = 0; e < 8; e += 2) top = max_abs3(s[e], s[e + 1], top);
      }
      if (!(top < INFINITY)) top = INFINITY;  // (not a number is as good as infinite here)
      top = meet<WARP, true>(top, buf[2]);
      if (top > 0.0f && top < INFINITY) {
        const int k = max(-100, min(126, ilogbf(top)));
        const float down = scalbnf(1.0f, -k);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float s[8];
          from_pairs(f[v], s);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            s[e] *= down;
            rest = fmaf(s[e], s[e], rest);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) f[v][i] = pack2(s[2 * i], s[2 * i + 1]);
        }
        r = root_reciprocal(fmaf(meet<WARP, false>(rest, buf[0]), p.inv_n, p.eps * down * down));
      }
    }
    // For codes only the root's power of two goes into the elements, which it leaves exact; the rest of it, from one to two, cancels in their
    // quotients by the largest: a rounding less, and s gamma has v's range.  (No root: one of a mean that is zero, infinite or not a number.)
    if (TY == MIMIR_B200_T_E4M3 && r > 0.0f && r < INFINITY) {
      root = __uint_as_float((__float_as_uint(r) & 0x007fffffu) | 0x3f800000u);
      r = __uint_as_float(__float_as_uint(r) & 0x7f800000u);
    }
    const Pair r2 = pack2(r, r);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int col = v * step + col0;
#pragma unroll
      for (int i = 0; i < 4; ++i) f[v][i] = mul2(f[v][i], r2);
      if (p.gamma) {
        Pair g[4];
        to_pairs<MIMIR_B200_T_F32>(row_load8<MIMIR_B200_T_F32, VEC>(reinterpret_cast<const char*>(p.gamma), col, p.n, apart), g);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[v][i] = mul2(f[v][i], g[i]);
      }
    }
  }
  char* const y = p.y + row * p.y_row;
  if constexpr (TY == MIMIR_B200_T_E4M3) {
    float top = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float s[8];
      from_pairs(f[v], s);
#pragma unroll
      for (int e = 0; e < 8; e += 2) top = max_abs3(s[e], s[e + 1], top);
    }
    top = meet<WARP, true>(top < INFINITY ? top : INFINITY, buf[1]);  // (infinite, too, for what is not a number)
    const bool finite = top < INFINITY;
    if (!finite) {  // over the finite ones
      top = 0.0f;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float s[8];
        from_pairs(f[v], s);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (fabsf(s[e]) < INFINITY) top = fmaxf(top, fabsf(s[e]));
      }
      top = meet<WARP, true>(top, buf[0]);
    }
    const float part = __fmul_rn(top, 1.0f / 448.0f);
    if (t == 0) p.y_scale[row] = __fmul_rn(part, root);
    // Without the norm codes of the IEEE quotients by one reciprocal, as the cache's (a zero's sign aside): those of 16-bit values are often
    // just between two codes.  Of a norm's values products with 448 / largest (`again` is zero), which is nearer to the quotients by the
    // largest itself: of 33 M codes 20 % fewer fall on the other side of a border than by the rounded scale.
    const bool quick = finite && (part == 0.0f || part > 0x1p-80f);
    const float inverse = part > 0.0f ? (norm ? __fdiv_rn(448.0f, top) : __frcp_rn(part)) : 0.0f, again = norm ? 0.0f : inverse;
    const Pair r2 = pack2(inverse, inverse), s2 = pack2(-part, -part), again2 = pack2(again, again);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int col = v * step + col0;
      if (col >= p.n) break;
      float s[8];
      if (quick) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const Pair n = mul2(f[v][i], r2);
          unpack2(NORM == 1 ? n : fma2(fma2(n, s2, f[v][i]), again2, n), s[2 * i], s[2 * i + 1]);
        }
      } else {
        from_pairs(f[v], s);
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] = part > 0.0f ? __fdiv_rn(s[e], part) : fabsf(s[e]) < INFINITY ? 0.0f : s[e];  // (none: a row with none finite but zeros)
      }
      row_store8<TY, VEC>(y, col, p.n, apart, pack8<TY>(s));
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float s[8];
      from_pairs(f[v], s);
      row_store8<TY, VEC>(y, v * step + col0, p.n, apart, pack8<TY>(s));
    }
  }
}

// Threads of a CTA at most and CTAs to an SM at least, for the registers: rows of F32 have two vectors a thread up to 12 288 elements (2 048 rows of
// them to bfloat16 with residual 59 us, with four 74), of 16 bits up to 8 192 (4 096 rows of 10 240 to codes 64 us, with four 54).
template <int TX, bool WARP, int V>
constexpr int norm_threads() { return WARP ? NR_WARP_THREADS : V == 2 && TX == MIMIR_B200_T_F32 ? 768 : 512; }
template <int TX, bool WARP, int V>
constexpr int norm_ctas() { return WARP ? (V == 4 ? 4 : 8) : V == 2 ? (TX == MIMIR_B200_T_F32 ? 2 : 3) : V == 4 ? 2 : 1; }

template <int TX, int TY, int V, bool WARP, bool VEC>
__global__ void __launch_bounds__(norm_threads<TX, WARP, V>(), norm_ctas<TX, WARP, V>()) norm_rows_serve_kernel(const __grid_constant__ NormParams p) {
  __shared__ __align__(16) float buf[MEETINGS][32];
  pdl_early_if(p.early);
  if (!WARP && threadIdx.x < MEETINGS * 32) buf[threadIdx.x >> 5][threadIdx.x & 31] = 0.0f;
  pdl_wait();
  const int row = WARP ? blockIdx.x * (NR_WARP_THREADS / 32) + (threadIdx.x >> 5) : blockIdx.x;
  if (WARP && row >= p.rows) return;
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x, step = (WARP ? 32 : blockDim.x) * 8;
  const int apart = VEC || TX != MIMIR_B200_T_F32 ? 0 : step / 8, col0 = apart ? t : t * 8;
  const char* const x = p.x + row * p.x_row;
  Pair f[V][4];
  Raw8<TX> raw[V], res[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    raw[v] = row_load8<TX, VEC>(x, v * step + col0, p.n, apart);
    if (p.residual) res[v] = row_load8<TX, VEC>(p.residual + row * p.residual_row, v * step + col0, p.n, apart);
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    to_pairs<TX>(raw[v], f[v]);
    if (p.residual) {
      Pair g[4];
      to_pairs<TX>(res[v], g);
#pragma unroll
      for (int i = 0; i < 4; ++i) f[v][i] = add2(f[v][i], g[i]);
    }
  }
  if (!WARP) __syncthreads();  // (the words of no warp)
  finish_row<TX, TY, V, WARP, VEC>(p, row, t, step, apart, f, buf);
}

// The same for many long rows of 16 bits without a residual: few CTAs fit into the registers, so the rows come through a ring in shared memory by
// bulk copies asked for several rows ahead, and what is on its way does not stand still while a row's threads meet.  5 003 rows of 12 288 halves
// to codes 38 us, without it 46 (with a residual 65 against 54, and for rows that more CTAs hold 63 against 40: not there).
template <int TX, int TY, int NORM>
__global__ void __launch_bounds__(512, 2) norm_rows_ring_kernel(const __grid_constant__ NormParams p) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ __align__(8) uint64_t bars[NR_MAX_STAGES];
  __shared__ __align__(16) float buf[MEETINGS][32];
  __shared__ volatile int abort_word;
  const int t = threadIdx.x, step = blockDim.x * 8, apart = gridDim.x;
  const uint32_t bytes = static_cast<uint32_t>(p.n) * type_bytes(TX);
  if (t < MEETINGS * 32) buf[t >> 5][t & 31] = 0.0f;
  if (t == 0) {
    for (int s = 0; s < p.stages; ++s) mbar_init(&bars[s], 1);
    abort_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async_smem();
  }
  __syncthreads();
  pdl_wait();
  auto ask = [&](int row, int s) {
    mbar_expect_tx(&bars[s], bytes);
    bulk_load_1d(ring + s * bytes, p.x + row * p.x_row, bytes, &bars[s]);
  };
  long long next = blockIdx.x;  // the row that is asked for next
  if (t == 0)
    for (int s = 0; s < p.stages && next < p.rows; ++s, next += apart) ask(static_cast<int>(next), s);
  int stage = 0;
  uint32_t phase = 0;
#pragma unroll 1
  for (long long row = blockIdx.x; row < p.rows; row += apart) {
    const bool ok = mbar_wait(&bars[stage], phase, &abort_word, p.err_word, 121);
    const char* x = reinterpret_cast<const char*>(ring + stage * bytes);
    Pair f[4][4];
#pragma unroll
    for (int v = 0; v < 4; ++v) to_pairs<TX>(row_load8<TX, true>(x, v * step + t * 8, p.n, 0), f[v]);
    if (!__syncthreads_and(ok)) {  // a wait gave up: nothing may still be on its way into shared memory when the CTA ends
      if (t == 0) {
        int still = 0;
        for (; row < next; row += apart) {
          mbar_wait(&bars[stage], phase, &still, p.err_word, 122);
          if (++stage == p.stages) { stage = 0; phase ^= 1; }
        }
      }
      break;
    }
    if (t == 0 && next < p.rows) {
      ask(static_cast<int>(next), stage);
      next += apart;
    }
    finish_row<TX, TY, 4, false, true, NORM>(p, static_cast<int>(row), t, step, 0, f, buf);
    if (++stage == p.stages) { stage = 0; phase ^= 1; }
  }
}

template <int TX, int TY, int V, bool WARP>
int launch_as(const NormParams& p, int threads, cudaStream_t st) {
  constexpr int PER = WARP ? NR_WARP_THREADS / 32 : 1;
  const unsigned grid = (static_cast<unsigned>(p.rows) + PER - 1) / PER;
  NormParams q = p;
  if constexpr (!WARP && V == 4 && TX != MIMIR_B200_T_F32) {
    const size_t row_bytes = static_cast<size_t>(p.n) * type_bytes(TX);
    const unsigned at_once = static_cast<unsigned>(ctx().sm_count * 2);
    if (p.vec && !p.residual && row_bytes % 16 == 0 && grid > 2 * at_once) {
      q.stages = static_cast<int>(std::min<size_t>(NR_RING / row_bytes, NR_MAX_STAGES));  // (rows of up to 32 KB: three at least)
      auto run = [&](auto kern, PerDeviceOnce& once) -> int {
        MB_TRY(once.run([&]() -> int {
          MB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, NR_RING));
          return MIMIR_B200_OK;
        }));
        return launch_pdl(kern, dim3(at_once), dim3(static_cast<unsigned>(threads)), q.stages * row_bytes, st, 1, q);
      };
      static PerDeviceOnce plain, normed;
      if (p.norm) MB_TRY((run(norm_rows_ring_kernel<TX, TY, 1>, normed)));
      else MB_TRY((run(norm_rows_ring_kernel<TX, TY, 0>, plain)));
      count_launch();
      return MIMIR_B200_OK;
    }
  }
  q.early = pdl_small_grid(grid);
  MB_TRY(launch_pdl(p.vec ? norm_rows_serve_kernel<TX, TY, V, WARP, true> : norm_rows_serve_kernel<TX, TY, V, WARP, false>, dim3(grid),
                    dim3(static_cast<unsigned>(threads)), 0, st, 1, q));
  count_launch();
  return MIMIR_B200_OK;
}
template <int TX, int TY>
int launch_rows(const NormParams& p, cudaStream_t st) {
  const int vectors = (p.n + 7) / 8;
  auto threads = [&](int v) { return round_up((vectors + v - 1) / v, 32); };
  if (vectors <= 32) return launch_as<TX, TY, 1, true>(p, NR_WARP_THREADS, st);
  if (vectors <= 64) return launch_as<TX, TY, 2, true>(p, NR_WARP_THREADS, st);
  if (vectors <= 128) return launch_as<TX, TY, 4, true>(p, NR_WARP_THREADS, st);
  if (vectors <= norm_threads<TX, false, 2>() * 2) return launch_as<TX, TY, 2, false>(p, threads(2), st);
  if (vectors <= 2048) return launch_as<TX, TY, 4, false>(p, threads(4), st);
  return launch_as<TX, TY, 8, false>(p, threads(8), st);
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
  p.rows = a.rows, p.n = a.n, p.norm = a.norm, p.eps = a.eps, p.inv_n = 1.0f / static_cast<float>(a.n), p.err_word = ctx().dev_error_word;
  p.vec = vectors_at(p.x, p.x_row, 16) && vectors_at(p.residual, p.residual_row, 16) && vectors_at(p.sum, p.sum_row, 16) && vectors_at(p.gamma, 0, 16) &&
          vectors_at(p.y, p.y_row, ys == 1 ? 8 : 16);
  switch (a.type) {
    case MIMIR_B200_T_F32: return launch_to<MIMIR_B200_T_F32>(p, a.y_type, st);
    case MIMIR_B200_T_F16: return launch_to<MIMIR_B200_T_F16>(p, a.y_type, st);
    default: return launch_to<MIMIR_B200_T_BF16>(p, a.y_type, st);
  }
}

}  // namespace mb
