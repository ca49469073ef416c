// rope.cu — rotary positions: pairs of a head's elements turned by an angle that grows with the token's position,
//   (a, b) -> m (a cos t - b sin t, a sin t + b cos t),   t = position * f_i,   f_i = base^(-2 i / rot) (stretched for long contexts).
//
// The angle is kept as a fraction of a turn in 64-bit fixed point: step_i = f_i / (2 pi) * 2^64, so position * step_i modulo 2^64 is the
// fraction itself, exact in the integer product; what is off is step_i's rounding alone, position * 2^-65 turns.  (In fp32 the
// angle of position 100 000 would be off by up to 0.004.)  The quadrant comes off in integers, and the rest, at most an eighth of
// a turn, becomes fp32 with its full 24 bits.
// Bound by its bytes: 8192 rows of 40 heads of 128 in fp32, 64 of them turned, 54 us, 0.95 of the rate of a plain copy.
#include <cmath>

#include "common.h"
#include "paged.cuh"

namespace mb {
namespace {

constexpr int RO_THREADS = 256;

__device__ __forceinline__ float2 turn_cos_sin(uint64_t phase) {
  const uint64_t quad = (phase + (1ull << 61)) >> 62;
  const long long rest = static_cast<long long>(phase - (quad << 62));  // [-2^61, 2^61)
  float s, c;
  sincospif(__ll2float_rn(rest) * 0x1p-63f, &s, &c);  // (in half turns)
  const bool swap = quad & 1;
  const float a = swap ? s : c, b = swap ? c : s;
  return make_float2((quad == 1 || quad == 2) ? -a : a, (quad & 2) ? -b : b);
}

template <int T>
struct RopeElem { using type = float; };
template <>
struct RopeElem<MIMIR_B200_T_F16> { using type = __half; };
template <>
struct RopeElem<MIMIR_B200_T_BF16> { using type = __nv_bfloat16; };
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f(float v, float* p) { *p = v; }
__device__ __forceinline__ void from_f(float v, __half* p) { *p = __float2half_rn(v); }
__device__ __forceinline__ void from_f(float v, __nv_bfloat16* p) { *p = __float2bfloat16_rn(v); }

// cosines and sines of `rows` rows from row0 on (one pair serves every head)
__device__ __forceinline__ void angles(const RopeLaunch& r, long long row0, int rows, float2* cs) {
  const int pairs = r.plan.rot_dim / 2;
  for (int i = threadIdx.x; i < rows * pairs; i += RO_THREADS) {
    const int row = i / pairs, pr = i - row * pairs;
    const float2 v = turn_cos_sin(r.plan.step[pr] * static_cast<uint64_t>(static_cast<long long>(__ldg(r.positions + row0 + row))));
    cs[i] = make_float2(v.x * r.plan.magnitude, v.y * r.plan.magnitude);
  }
  __syncthreads();
}

// Any sizes, strides and alignment: an element pair, or an element that passes, a thread.
template <int T>
__global__ void __launch_bounds__(RO_THREADS) rope_kernel(const __grid_constant__ RopeLaunch r, int per_cta) {
  using E = typename RopeElem<T>::type;
  extern __shared__ float2 cs[];  // [per_cta][pairs]
  const int pairs = r.plan.rot_dim / 2;
  const long long row0 = static_cast<long long>(blockIdx.x) * per_cta;
  const int rows = static_cast<int>(min(static_cast<long long>(per_cta), r.rows - row0));
  angles(r, row0, rows, cs);
  const int rest = r.x == r.y ? 0 : r.dim - r.plan.rot_dim;  // elements that pass as they are
  const int per_head = pairs + rest, per_row = per_head * r.heads;
  for (int i = threadIdx.x; i < rows * per_row; i += RO_THREADS) {
    const int row = i / per_row, j = i - row * per_row, head = j / per_head, e = j - head * per_head;
    const E* x = static_cast<const E*>(r.x) + (row0 + row) * r.x_row + head * r.x_head;
    E* y = static_cast<E*>(r.y) + (row0 + row) * r.y_row + head * r.y_head;
    if (e < pairs) {
      const int ia = r.plan.interleaved ? 2 * e : e, ib = r.plan.interleaved ? 2 * e + 1 : e + pairs;
      const float2 t = cs[row * pairs + e];
      const float a = to_f(x[ia]), b = to_f(x[ib]);
      from_f(a * t.x - b * t.y, y + ia);
      from_f(a * t.y + b * t.x, y + ib);
    } else {
      const int at = r.plan.rot_dim + e - pairs;
      y[at] = x[at];
    }
  }
}

// Eight elements at a time (two loads of fp32): heads, strides and the turned part whole multiples of them, pointers 16-byte aligned.  An
// item is eight elements: of both halves (INTER false), or eight neighbours (INTER true); or eight that pass.  The bytes bound it, each
// read and written once; RO_ITEMS items a thread are on their way together, which one at a time did not cover.
constexpr int RO_ITEMS = 2;
template <int T, bool INTER>
__global__ void __launch_bounds__(RO_THREADS) rope_vector_kernel(const __grid_constant__ RopeLaunch r, int per_cta, FastDiv by_row, FastDiv by_head) {
  extern __shared__ float2 cs[];
  const int pairs = r.plan.rot_dim / 2;
  const long long row0 = static_cast<long long>(blockIdx.x) * per_cta;
  const int rows = static_cast<int>(min(static_cast<long long>(per_cta), r.rows - row0));
  angles(r, row0, rows, cs);
  const int turned = INTER ? r.plan.rot_dim / 8 : pairs / 8, per_head = static_cast<int>(by_head.d), per_row = static_cast<int>(by_row.d);
  constexpr int SIZE = type_bytes(T);
  for (int i0 = threadIdx.x; i0 < rows * per_row; i0 += RO_ITEMS * RO_THREADS) {
    Raw8<T> a[RO_ITEMS], b[RO_ITEMS];
    long long at[RO_ITEMS];
    int angle[RO_ITEMS];
#pragma unroll
    for (int u = 0; u < RO_ITEMS; ++u) {
      const int i = i0 + u * RO_THREADS;
      angle[u] = -2;
      if (i >= rows * per_row) continue;
      const int row = by_row.div(i), j = i - row * per_row, head = by_head.div(j), e = j - head * per_head;
      const bool pass = e >= turned;
      const int d = pass ? r.plan.rot_dim + 8 * (e - turned) : 8 * e;
      const char* x = static_cast<const char*>(r.x) + ((row0 + row) * r.x_row + head * r.x_head + d) * SIZE;
      at[u] = ((row0 + row) * r.y_row + head * r.y_head + d) * SIZE;
      angle[u] = pass ? -1 : row * pairs + (INTER ? 4 * e : 8 * e);
      a[u] = load8<T>(x);
      if (!INTER && !pass) b[u] = load8<T>(x + pairs * SIZE);
    }
#pragma unroll
    for (int u = 0; u < RO_ITEMS; ++u) {
      if (angle[u] == -2) continue;
      char* y = static_cast<char*>(r.y) + at[u];
      if (angle[u] >= 0) {
        float f[8], g[8];
        unpack8<T>(a[u], f);
        if constexpr (INTER) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 t = cs[angle[u] + e];
            g[2 * e] = f[2 * e] * t.x - f[2 * e + 1] * t.y;
            g[2 * e + 1] = f[2 * e] * t.y + f[2 * e + 1] * t.x;
          }
          a[u] = pack8<T>(g);
        } else {
          unpack8<T>(b[u], g);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 t = cs[angle[u] + e];
            const float p = f[e] * t.x - g[e] * t.y;
            g[e] = f[e] * t.y + g[e] * t.x;
            f[e] = p;
          }
          a[u] = pack8<T>(f);
          store8<T>(y + pairs * SIZE, pack8<T>(g));
        }
      }
      store8<T>(y, a[u]);
    }
  }
}

template <int T>
int launch_rope_as(const RopeLaunch& r, cudaStream_t st) {
  const int pairs = r.plan.rot_dim / 2, rest = r.x == r.y ? 0 : r.dim - r.plan.rot_dim;
  const bool inter = r.plan.interleaved != 0;
  auto whole = [](long long v) { return v % 8 == 0; };
  const bool vector = whole(inter ? r.plan.rot_dim : pairs) && whole(rest) && whole(r.plan.rot_dim) && whole(r.x_row) && whole(r.x_head) && whole(r.y_row) &&
                      whole(r.y_head) && reinterpret_cast<uintptr_t>(r.x) % 16 == 0 && reinterpret_cast<uintptr_t>(r.y) % 16 == 0;
  const int per_row = r.heads * (vector ? (inter ? r.plan.rot_dim : pairs) / 8 + rest / 8 : pairs + rest);
  // rows of a CTA: for a few items a thread, and no fewer CTAs than fill the SMs
  int per_cta = 1;
  while (per_cta < 8 && r.rows >= 8LL * ctx().sm_count * per_cta && per_cta * per_row < 4 * RO_THREADS) per_cta *= 2;
  const unsigned grid = static_cast<unsigned>((r.rows + per_cta - 1) / per_cta);
  const size_t smem = static_cast<size_t>(per_cta) * pairs * sizeof(float2);
  if (!vector) rope_kernel<T><<<grid, RO_THREADS, smem, st>>>(r, per_cta);
  else if (inter) rope_vector_kernel<T, true><<<grid, RO_THREADS, smem, st>>>(r, per_cta, FastDiv(per_row), FastDiv(per_row / r.heads));
  else rope_vector_kernel<T, false><<<grid, RO_THREADS, smem, st>>>(r, per_cta, FastDiv(per_row), FastDiv(per_row / r.heads));
  MB_CUDA(cudaGetLastError());
  count_launch();
  return MIMIR_B200_OK;
}

}  // namespace

int launch_rope(const RopeLaunch& r, cudaStream_t st) {
  if (r.type == MIMIR_B200_T_F32) return launch_rope_as<MIMIR_B200_T_F32>(r, st);
  if (r.type == MIMIR_B200_T_F16) return launch_rope_as<MIMIR_B200_T_F16>(r, st);
  return launch_rope_as<MIMIR_B200_T_BF16>(r, st);
}

}  // namespace mb

extern "C" int mimir_b200_rope_plan(const MimirRopeSpec* spec, MimirRopePlan* plan) {
  using mb::fail;
  if (!spec || !plan) return fail(MIMIR_B200_E_INVALID, "rope_plan: null argument");
  const int rot = spec->rot_dim;
  if (rot <= 0 || (rot & 1) || rot > 2 * MIMIR_B200_MAX_ROPE_PAIRS)
    return fail(MIMIR_B200_E_INVALID, "rope_plan: rot_dim %d is not an even number of 2 to %d", rot, 2 * MIMIR_B200_MAX_ROPE_PAIRS);
  if (!(spec->base > 1.0) || !std::isfinite(spec->base)) return fail(MIMIR_B200_E_INVALID, "rope_plan: base must be finite and above 1");
  if (spec->scaling < MIMIR_B200_ROPE_NONE || spec->scaling > MIMIR_B200_ROPE_RAMP) return fail(MIMIR_B200_E_INVALID, "rope_plan: unknown scaling %d", spec->scaling);
  if (spec->scaling != MIMIR_B200_ROPE_NONE && (!(spec->factor > 0.0) || !std::isfinite(spec->factor)))
    return fail(MIMIR_B200_E_INVALID, "rope_plan: factor must be finite and positive");
  const bool ranged = spec->scaling == MIMIR_B200_ROPE_BANDS || spec->scaling == MIMIR_B200_ROPE_RAMP;
  if (ranged && !(spec->low > 0.0 && spec->high > spec->low && std::isfinite(spec->high) && spec->original_len > 0.0 && std::isfinite(spec->original_len)))
    return fail(MIMIR_B200_E_INVALID, "rope_plan: 0 < low < high and original_len > 0 are needed");
  if (!std::isfinite(static_cast<float>(spec->magnitude)) || spec->magnitude < 0.0) return fail(MIMIR_B200_E_INVALID, "rope_plan: magnitude must be finite in fp32 and not negative");
  const long double two_pi = 6.283185307179586476925286766559L, base = spec->base, factor = spec->factor;
  int first = 0, last = 0;
  if (spec->scaling == MIMIR_B200_ROPE_RAMP) {
    auto place = [&](long double turns) { return rot * std::log(spec->original_len / (two_pi * turns)) / (2 * std::log(base)); };
    const long double a = std::floor(place(spec->high)), b = std::ceil(place(spec->low));
    first = static_cast<int>(a < 0 ? 0 : a > rot ? rot : a);
    last = static_cast<int>(b > rot - 1 ? rot - 1 : b < 0 ? 0 : b);
  }
  MimirRopePlan out = {};
  out.rot_dim = rot;
  out.interleaved = spec->interleaved ? 1 : 0;
  out.magnitude = spec->magnitude > 0.0 ? static_cast<float>(spec->magnitude) : 1.0f;
  for (int i = 0; i < rot / 2; ++i) {
    long double f = std::pow(base, -2.0L * i / rot);
    if (spec->scaling == MIMIR_B200_ROPE_LINEAR) {
      f /= factor;
    } else if (spec->scaling == MIMIR_B200_ROPE_BANDS) {
      long double part = (spec->original_len * f / two_pi - spec->low) / (static_cast<long double>(spec->high) - spec->low);
      part = part < 0 ? 0 : part > 1 ? 1 : part;
      f *= part + (1 - part) / factor;
    } else if (spec->scaling == MIMIR_B200_ROPE_RAMP) {
      long double ramp = (i - first) / (last > first ? static_cast<long double>(last - first) : 0.001L);
      ramp = ramp < 0 ? 0 : ramp > 1 ? 1 : ramp;
      f *= (1 - ramp) + ramp / factor;
    }
    const long double turns = f / two_pi;  // of a position; whole turns do not count
    const long double step = (turns - std::floor(turns)) * 18446744073709551616.0L + 0.5L;
    out.step[i] = step >= 18446744073709551616.0L ? 0 : static_cast<uint64_t>(step);
    if (spec->inverse) out.step[i] = 0 - out.step[i];
  }
  *plan = out;
  return MIMIR_B200_OK;
}
