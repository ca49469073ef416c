// linear_rows.cu — products of few rows: the weights' bytes are the bound, or there are not tiles enough for the SMs.
//
// The weights are the M side (128 features, the lanes of tensor memory), up to 256 rows of x (of a gated pair 128) the N side: an instruction costs the same whatever its
// N, and a narrow N takes little shared memory from the ring that the weights stream through.  Where features and rows make fewer tiles
// than there are SMs, the CTAs of a cluster (up to eight) share n_in; their sums go into one another's shared memory by rows of x, and each adds up its
// rows in the order of the shares, so that a result has the same bits every time.  A gated pair has two accumulators in the same lanes.
//   warp 0 TMA, warp 1 instructions, warps 2-9 results: two for each 32 features, 16 rows of x at a time in turn.
#include "launch.cuh"
#include "linear.cuh"

namespace mb {
namespace {

constexpr int RM = 128;                 // features of a CTA
constexpr int MAX_STAGES = 16, THREADS = 320, EPI = 256, W_BYTES = RM * LIN_BLOCK;
constexpr int BARS = 512;

struct RowParams {
  LinearParams l;
  int rows_tile, row_tiles;  // rows of x of a CTA (a multiple of 16), tiles of them
  int splits, part_rows;     // CTAs that share n_in, and rows of x that each of them finishes
  int stages, stage_bytes;
  int tmem_cols, early;
};

__device__ __forceinline__ void st_cluster(uint32_t addr, float v) { asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory"); }
__device__ __forceinline__ float act_one(float z, int act) {
  float v[2] = {z, 0.0f};
  activate(v, act);
  return v[0];
}

// U: of results of F32 how many times 16 rows that a warp holds while it adds up; 0: other results.
template <bool F8, bool GATED, int U>
__global__ void __launch_bounds__(THREADS, U > 2 ? 1 : 2)
linear_rows_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_up,
                   const __grid_constant__ RowParams rp) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t bars[2 * MAX_STAGES + 4];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_word;
  uint64_t *full_bar = bars, *empty_bar = bars + MAX_STAGES, *acc_full = bars + 2 * MAX_STAGES, *acc_empty = acc_full + 2;
  volatile int* abort_flag = &abort_word;

  const LinearParams& p = rp.l;
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int splits = rp.splits, rank = splits > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int tile = blockIdx.x / splits, ft = tile / rp.row_tiles, rt = tile - ft * rp.row_tiles;
  const int n = rp.rows_tile;
  const int kb0 = static_cast<int>(static_cast<long long>(p.kblocks) * rank / splits), kb1 = static_cast<int>(static_cast<long long>(p.kblocks) * (rank + 1) / splits);

  if (threadIdx.x == 0) {
    for (int s = 0; s < rp.stages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], EPI / 32);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async_smem();
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, rp.tmem_cols);
    tmem_relinquish();
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = tmem_slot;
  pdl_early_if(rp.early);
  pdl_wait();

  const uint32_t acc_cols = static_cast<uint32_t>(GATED ? 2 * n : n);
  float* const parts = reinterpret_cast<float*>(smem);  // [splits][GATED ? 2 : 1][part_rows][RM], once the ring is done with
  const int quad = warp & 3, half = (warp - 2) >> 2;

  if (warp == 0) {
    const bool one = elect_one();
    constexpr int per_block = F8 ? LIN_BLOCK : LIN_BLOCK / 2;
    const uint32_t bytes = static_cast<uint32_t>((GATED ? 2 : 1) * W_BYTES + n * LIN_BLOCK);
    int stage = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait_warp(&empty_bar[stage], phase ^ 1, abort_flag, p.err_word, 111)) break;
      if (one) {
        uint8_t* base = smem + stage * rp.stage_bytes;
        uint64_t* bar = &full_bar[stage];
        mbar_expect_tx(bar, bytes);
        tma_load_2d(base, &map_w, bar, kb * per_block, ft * RM);
        if constexpr (GATED) tma_load_2d(base + W_BYTES, &map_up, bar, kb * per_block, ft * RM);
        tma_load_2d(base + (GATED ? 2 : 1) * W_BYTES, &map_x, bar, kb * per_block, rt * n);
      }
      __syncwarp();
      if (++stage == rp.stages) { stage = 0; phase ^= 1; }
    }
    // what was asked for has landed and been used (or the abort flag is up) before the ring becomes something else
    for (int s = 0; s < rp.stages; ++s) {
      if (!mbar_wait_warp(&empty_bar[stage], phase ^ 1, abort_flag, p.err_word, 112)) break;
      if (++stage == rp.stages) { stage = 0; phase ^= 1; }
    }
  } else if (warp == 1) {
    const bool one = elect_one();
    const uint32_t idesc = linear_idesc(RM, n) | p.formats;
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 0;
    bool ready = false, ok = true;
    for (int kb = kb0; kb < kb1 && ok;) {
      if (!mbar_wait_warp(&acc_empty[acc], acc_phase ^ 1, abort_flag, p.err_word, 113)) break;
      tcgen05_fence_after();
      const uint32_t d = tmem + acc * acc_cols;
      const int from = kb, to = min(kb1, kb + p.chunk);
      for (; kb < to; ++kb) {
        if (!__all_sync(0xffffffffu, ready) && !mbar_wait_warp(&full_bar[stage], phase, abort_flag, p.err_word, 114)) { ok = false; break; }
        tcgen05_fence_after();
        const uint32_t sa = smem_u32(smem + stage * rp.stage_bytes);
        const uint64_t dw = make_smem_desc(sa, LIN_BLOCK), du = dw + (W_BYTES >> 4), dx = dw + ((GATED ? 2 : 1) * W_BYTES >> 4);
        uint64_t* done = &empty_bar[stage];
        if (++stage == rp.stages) { stage = 0; phase ^= 1; }
        ready = mbar_test(&full_bar[stage], phase);
        if (one) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t add = (kb != from || k != 0) ? 1u : 0u;
            if constexpr (F8) {
              umma_f8(d, dw + 2 * k, dx + 2 * k, idesc, add);
              if constexpr (GATED) umma_f8(d + n, du + 2 * k, dx + 2 * k, idesc, add);
            } else {
              umma_bf16(d, dw + 2 * k, dx + 2 * k, idesc, add);
              if constexpr (GATED) umma_bf16(d + n, du + 2 * k, dx + 2 * k, idesc, add);
            }
          }
          umma_commit(done);
        }
        __syncwarp();
      }
      if (!ok) break;
      if (one) umma_commit(&acc_full[acc]);
      __syncwarp();
      if (++acc == 2) { acc = 0; acc_phase ^= 1; }
    }
  }

  // ---- results: a lane has a feature, a register a row of x ----
  const bool results = warp >= 2;
  const int feature = ft * RM + quad * 32 + lane, units = n / 16;
  const uint32_t lanes = tmem + (static_cast<uint32_t>(quad * 32) << 16);
  const int size = p.out_type == MIMIR_B200_T_F32 ? 4 : 2;
  // 16 rows of x from row `col` of the tile on, all of n_in: to the result
  float w_scale = 1.0f, up_scale = 1.0f, bias = 0.0f, up_bias = 0.0f;
  if (results && feature < p.n_out && splits == 1) {
    if constexpr (F8) w_scale = __ldg(p.w_scale + feature);
    if constexpr (F8 && GATED) up_scale = __ldg(p.up_scale + feature);
    if (p.bias) bias = __ldg(p.bias + feature);
    if (GATED && p.up_bias) up_bias = __ldg(p.up_bias + feature);
  }
  auto finish16 = [&](float (&z)[16], float (&u)[16], int col) {
    const int row0 = rt * n + col;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      if constexpr (F8) {
        const float sx = row0 + j < p.rows ? __ldg(p.x_scale + row0 + j) : 0.0f;
        z[j] = fmaf(z[j] * sx, w_scale, bias);
        if constexpr (GATED) u[j] = fmaf(u[j] * sx, up_scale, up_bias);
      } else {
        z[j] += bias;
        if constexpr (GATED) u[j] += up_bias;
      }
    }
    activate(z, p.act);
    if (feature < p.n_out) {
      if constexpr (GATED) {
#pragma unroll
        for (int j = 0; j < 16; ++j) z[j] *= u[j];
      } else if (p.residual) {
        float q[16];
#pragma unroll
        for (int j = 0; j < 16; ++j)
          q[j] = row0 + j < p.rows ? load_typed(p.residual + (row0 + j) * p.residual_row + static_cast<long long>(feature) * size, p.out_type) : 0.0f;
#pragma unroll
        for (int j = 0; j < 16; ++j) z[j] += q[j];
      }
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (row0 + j < p.rows) store_typed(p.out + (row0 + j) * p.out_row + static_cast<long long>(feature) * size, p.out_type, z[j]);
    }
    __syncwarp();
  };
  // ... or this CTA's share of n_in: to the CTA that finishes the row
  auto send16 = [&](const float (&z)[16], int which, int col) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int owner = (col + j) / rp.part_rows, at = ((rank * (GATED ? 2 : 1) + which) * rp.part_rows + (col + j - owner * rp.part_rows)) * RM + quad * 32 + lane;
      st_cluster(mapa_shared(smem_u32(parts + at), static_cast<uint32_t>(owner)), z[j]);
    }
  };
  constexpr int HELD = U > 0 ? U : 1;
  float v[HELD][16];
  bool ok = true;
  if (results) {
    if constexpr (U > 0) {
      // (of a gated pair: the first half of the registers for the one, the second for the other)
      constexpr int EACH = GATED ? U / 2 : U;
#pragma unroll
      for (int i = 0; i < U; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) v[i][j] = 0.0f;
      int acc = 0;
      uint32_t acc_phase = 0;
      for (int kb = kb0; kb < kb1; kb += p.chunk) {
        ok = mbar_wait_warp(&acc_full[acc], acc_phase, abort_flag, p.err_word, 115);
        if (!ok) break;
        tcgen05_fence_after();
#pragma unroll
        for (int i = 0; i < U; ++i) {
          const int unit = 2 * (i % EACH) + half;
          if (unit >= units) continue;
          float w[16];
          tmem_ld_32x16(lanes + acc * acc_cols + static_cast<uint32_t>(unit * 16 + (i >= EACH ? n : 0)), w);
#pragma unroll
          for (int j = 0; j < 16; ++j) v[i][j] += w[j];
        }
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[acc]);
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
      }
      if (ok && splits == 1) {
#pragma unroll
        for (int i = 0; i < EACH; ++i)
          if (2 * i + half < units) finish16(v[i], v[GATED ? i + EACH : i], (2 * i + half) * 16);
      }
    } else {
      ok = mbar_wait_warp(&acc_full[0], 0, abort_flag, p.err_word, 115);
      tcgen05_fence_after();
      if (ok && splits == 1) {
#pragma unroll 1
        for (int unit = half; unit < units; unit += 2) {
          float z[16], u[16];
          tmem_ld_32x16(lanes + static_cast<uint32_t>(unit * 16), z);
          if constexpr (GATED) tmem_ld_32x16(lanes + static_cast<uint32_t>(n + unit * 16), u);
          finish16(z, u, unit * 16);
        }
      }
    }
  }
  if (splits > 1) {
    __syncthreads();
    cluster_sync_all();  // every ring of the cluster is done with
    if (results && ok) {
      if constexpr (U > 0) {
        constexpr int EACH = GATED ? U / 2 : U;
#pragma unroll
        for (int i = 0; i < U; ++i)
          if (2 * (i % EACH) + half < units) send16(v[i], i / EACH, (2 * (i % EACH) + half) * 16);
      } else {
#pragma unroll 1
        for (int unit = half; unit < units; unit += 2) {
          float z[16];
          tmem_ld_32x16(lanes + static_cast<uint32_t>(unit * 16), z);
          send16(z, 0, unit * 16);
          if constexpr (GATED) {
            tmem_ld_32x16(lanes + static_cast<uint32_t>(n + unit * 16), z);
            send16(z, 1, unit * 16);
          }
        }
      }
    }
    __syncwarp();
    cluster_sync_all();  // every share has arrived
    const int f = static_cast<int>(threadIdx.x) - 64, fl = f & (RM - 1), feat = ft * RM + fl;
    if (f >= 0 && feat < p.n_out && !*abort_flag) {
      float ws = 1.0f, us = 1.0f, b = 0.0f, ub = 0.0f;
      if constexpr (F8) ws = __ldg(p.w_scale + feat);
      if constexpr (F8 && GATED) us = __ldg(p.up_scale + feat);
      if (p.bias) b = __ldg(p.bias + feat);
      if (GATED && p.up_bias) ub = __ldg(p.up_bias + feat);
      for (int t = f / RM; t < rp.part_rows; t += EPI / RM) {
        const int col = rank * rp.part_rows + t, row = rt * n + col;
        if (col >= n || row >= p.rows) break;
        float z = 0.0f, u = 0.0f;
        for (int s = 0; s < splits; ++s) {
          const float* from = parts + static_cast<size_t>((s * (GATED ? 2 : 1)) * rp.part_rows + t) * RM + fl;
          z += from[0];
          if constexpr (GATED) u += from[rp.part_rows * RM];
        }
        if constexpr (F8) {
          const float sx = __ldg(p.x_scale + row);
          z = fmaf(z * sx, ws, b);
          if constexpr (GATED) u = fmaf(u * sx, us, ub);
        } else {
          z += b;
          if constexpr (GATED) u += ub;
        }
        z = act_one(z, p.act);
        if constexpr (GATED) z *= u;
        else if (p.residual) z += load_typed(p.residual + row * p.residual_row + static_cast<long long>(feat) * size, p.out_type);
        store_typed(p.out + row * p.out_row + static_cast<long long>(feat) * size, p.out_type, z);
      }
    }
  }

  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    tcgen05_fence_after();
    tmem_dealloc(tmem, rp.tmem_cols);
  }
}

struct RowShape {
  int rows_tile, row_tiles, feature_tiles, splits, stages, stage_bytes, part_rows, per_sm;
  size_t smem;
  long long ctas;
};
RowShape row_shape(const MimirLinear& a, bool gated) {
  RowShape s;
  const int most = gated ? 128 : 256;  // (two accumulators, and their shares in shared memory)
  s.row_tiles = (a.rows + most - 1) / most;
  s.rows_tile = round_up((a.rows + s.row_tiles - 1) / s.row_tiles, 16);
  s.feature_tiles = (a.n_out + RM - 1) / RM;
  const int blocks = static_cast<int>((static_cast<long long>(a.n_in) * type_bytes(a.type) + LIN_BLOCK - 1) / LIN_BLOCK);
  const long long tiles = static_cast<long long>(s.row_tiles) * s.feature_tiles;
  s.stage_bytes = (gated ? 2 : 1) * W_BYTES + s.rows_tile * LIN_BLOCK;
  s.per_sm = s.rows_tile <= 64 ? 2 : 1;
  const long long places = static_cast<long long>(ctx().sm_count) * s.per_sm;
  s.splits = 1;
  while (s.splits < 8 && tiles * (s.splits + 1) <= places && blocks / (s.splits + 1) >= 4) ++s.splits;
  s.part_rows = (s.rows_tile + s.splits - 1) / s.splits;
  const int ring = (s.per_sm == 2 ? 113 : 226) * 1024 - 1024 - BARS;
  s.stages = ring / s.stage_bytes;
  if (s.stages > MAX_STAGES) s.stages = MAX_STAGES;
  const size_t parts = s.splits > 1 ? static_cast<size_t>(s.splits) * (gated ? 2 : 1) * s.part_rows * RM * 4 : 0;
  s.smem = static_cast<size_t>(s.stages) * s.stage_bytes;
  if (parts > s.smem) s.smem = parts;
  s.smem += 1024;
  s.ctas = tiles * s.splits;
  return s;
}

template <bool F8, bool GATED, int U>
int launch_as(const CUtensorMap (&maps)[3], const RowParams& p, const RowShape& s, cudaStream_t st) {
  auto kern = linear_rows_kernel<F8, GATED, U>;
  static PerDeviceOnce once;
  MB_TRY(once.run([&]() -> int {
    MB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024));
    return MIMIR_B200_OK;
  }));
  MB_TRY(launch_pdl(kern, dim3(static_cast<unsigned>(s.ctas)), dim3(THREADS), s.smem, st, s.splits, maps[0], maps[1], maps[2], p));
  count_launch();
  return MIMIR_B200_OK;
}
template <bool F8, bool GATED>
int launch_for(const CUtensorMap (&maps)[3], const RowParams& p, const RowShape& s, cudaStream_t st) {
  if (p.l.out_type != MIMIR_B200_T_F32) return launch_as<F8, GATED, 0>(maps, p, s, st);
  return s.rows_tile <= (GATED ? 32 : 64) ? launch_as<F8, GATED, 2>(maps, p, s, st) : launch_as<F8, GATED, 8>(maps, p, s, st);
}

}  // namespace

double linear_rows_cycles(const MimirLinear& a, bool gated) {
  if (a.rows > 4096) return 1e30;
  const RowShape s = row_shape(a, gated);
  if (s.ctas > 0x7fffffffLL / 4) return 1e30;
  const double blocks = (static_cast<double>(a.n_in) * type_bytes(a.type) + LIN_BLOCK - 1) / LIN_BLOCK / s.splits;
  const double each = blocks * 4 * (gated ? 2 : 1) * (s.rows_tile > 64 ? s.rows_tile / 2.0 : 32.0) + 5000.0;
  return static_cast<double>((s.ctas + ctx().sm_count - 1) / ctx().sm_count) * each;
}

int launch_linear_rows(const MimirLinear& a, const LinearParams& l, bool gated, cudaStream_t st) {
  const RowShape s = row_shape(a, gated);
  CUtensorMap maps[3];
  MB_TRY(make_operand_map(&maps[0], a.x, a.type, a.rows, a.n_in, a.x_stride, s.rows_tile));
  MB_TRY(make_operand_map(&maps[1], a.w, a.type, a.n_out, a.n_in, a.w_stride, RM));
  maps[2] = maps[1];
  if (gated) MB_TRY(make_operand_map(&maps[2], a.up, a.type, a.n_out, a.n_in, a.up_stride, RM));
  RowParams p = {};
  p.l = l, p.rows_tile = s.rows_tile, p.row_tiles = s.row_tiles, p.splits = s.splits, p.part_rows = s.part_rows, p.stages = s.stages;
  p.stage_bytes = s.stage_bytes;
  const int cols = (l.out_type == MIMIR_B200_T_F32 ? 2 : 1) * (gated ? 2 : 1) * s.rows_tile;
  p.tmem_cols = 32;
  while (p.tmem_cols < cols) p.tmem_cols *= 2;
  p.early = pdl_small_grid(static_cast<unsigned>(s.ctas));
  if (a.type == MIMIR_B200_T_E4M3) return gated ? launch_for<true, true>(maps, p, s, st) : launch_for<true, false>(maps, p, s, st);
  return gated ? launch_for<false, true>(maps, p, s, st) : launch_for<false, false>(maps, p, s, st);
}

}  // namespace mb
