// paged_attention.cuh — arguments and result stores of the paged attention kernels.
#pragma once

#include "paged.cuh"

namespace mb {

struct AttendArgs {
  PagedView p;
  const void* q;
  void* out;
  float* lse;                              // natural logarithm of the row's sum of exponentials, or null
  long long q_row, q_head, o_row, o_head;  // elements
  int type, heads, group, causal, window;
  float scale;
  int tiles, cluster, splits;              // of the rows of a sequence; CTAs and clusters that share a tile's keys
  float* part_o;                           // [unit][split][16][head_dim], [unit][split][16] (max, sum): splits > 1
  float2* part_ml;
};

namespace {

__device__ __forceinline__ void store_out(const AttendArgs& a, int row0, int r, int kv_head, int d, float v) {
  const int tok = r / a.group, h = kv_head * a.group + r - tok * a.group;
  const long long at = (row0 + tok) * a.o_row + h * a.o_head + d;
  if (a.type == MIMIR_B200_T_F32) static_cast<float*>(a.out)[at] = v;
  else if (a.type == MIMIR_B200_T_F16) static_cast<__half*>(a.out)[at] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v);
}
// top is in base two; a row that saw no key has -infinity
__device__ __forceinline__ void store_lse(const AttendArgs& a, int row0, int r, int kv_head, float top, float sum) {
  if (!a.lse) return;
  const int tok = r / a.group, h = kv_head * a.group + r - tok * a.group;
  a.lse[static_cast<long long>(row0 + tok) * a.heads + h] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
}

}  // namespace
}  // namespace mb
