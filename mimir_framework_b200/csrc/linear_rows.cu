// linear_rows.cu — products of few rows: the weights' bytes are the bound, or there are not tiles enough for the SMs.
//
// The weights are the M side (features, the lanes of tensor memory), up to 256 rows of x (of a gated pair 128) the N side: an instruction costs the
// same whatever its N, and a narrow N takes little shared memory from the ring that the weights stream through.  A gated pair has two
// accumulators in the same lanes.
// A CTA has as many features as make one CTA for each SM, a multiple of eight up to 128: the instructions always work on 128 rows of shared
// memory, of which those behind the CTA's own are whatever comes next there and end in lanes that nobody reads.  Where few features would have
// every CTA read all of x, the CTAs of a cluster (up to eight) share n_in instead; their sums meet in shared memory: each CTA
// finishes some of the rows and gets what all have of them, added up in the order of the shares, so that a result has the same bits every time and
// wherever its row is in the call.
//   warp 0 TMA, warp 1 instructions, the other eight or sixteen results: 32 features and sixteen rows of x at a time.
#include <algorithm>
#include <cmath>

#include "launch.cuh"
#include "linear.cuh"

namespace mb {
namespace {

constexpr int RM = 128;  // rows of an instruction: features of a CTA at most
constexpr int MAX_STAGES = 24, EARLY = 4, AHEAD = 4;
constexpr int MAX_CLUSTER = 8, UNIT = 16, TURN = 2 * UNIT * RM * 4;  // (two turns of a unit for four warps)
constexpr int STATIC = 3 * 1024, DYNAMIC = 232448 - STATIC, DYNAMIC_TWO = (228 * 1024) / 2 - 1024 - STATIC;  // shared memory of a CTA, one or two to an SM
// A CTA of a cluster waits for others that may still be asking for tensor memory.  So that none of them can be kept from it by a CTA that waits
// in the same way, two such CTAs never share an SM: each takes more than half of its shared memory (and more than the other kernels
// of clusters leave, which take at least 104 KB a CTA).
constexpr size_t ALONE = 128 * 1024;

struct RowParams {
  LinearParams l;
  int rows_tile, row_tiles;         // rows of x of a CTA (a multiple of 16), tiles of them
  int features;                     // of a CTA (a multiple of 8)
  int cluster;                      // CTAs that share n_in
  int stages, stage_bytes;
  int parts_at;                     // the cluster's sums: where in shared memory (0: the ring, when it is done with)
  int turn_at;                      // where results are turned around, TURN bytes for four warps: the ring or behind the sums in it
  int tmem_cols, early;
};

// How the K blocks fall to the CTAs of a cluster, and units of rows for the finish: number i of `size` has [total i / size, total (i + 1) / size)
__host__ __device__ __forceinline__ int share_begin(int total, int i, int size) { return static_cast<int>(static_cast<unsigned>(total * i) / static_cast<unsigned>(size)); }

__device__ __forceinline__ void st_cluster4(uint32_t addr, const float* v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void result_warps_sync(int threads) { asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory"); }
__device__ __forceinline__ void four_warps_sync(int four) { asm volatile("bar.sync %0, 128;" ::"r"(2 + four) : "memory"); }
__device__ __forceinline__ void prefetch_line(const char* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// Eight values of a row as they lie in memory, 16 bytes (F32: 32); converted where they are added.
struct Eight {
  uint4 a, b;
};
__device__ __forceinline__ Eight fetch_eight(const char* p, int type, bool vec, int left) {
  Eight e = {};
  if (vec) {
    e.a = *reinterpret_cast<const uint4*>(p);
    if (type == MIMIR_B200_T_F32) e.b = *reinterpret_cast<const uint4*>(p + 16);
    return e;
  }
  uint32_t w[8] = {};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (j >= left) break;
    if (type == MIMIR_B200_T_F32) w[j] = reinterpret_cast<const uint32_t*>(p)[j];
    else w[j / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[j]) << (16 * (j & 1));
  }
  e.a = make_uint4(w[0], w[1], w[2], w[3]), e.b = make_uint4(w[4], w[5], w[6], w[7]);
  return e;
}
__device__ __forceinline__ void add_eight(const Eight& e, int type, float (&v)[8]) {
  const uint32_t w[8] = {e.a.x, e.a.y, e.a.z, e.a.w, e.b.x, e.b.y, e.b.z, e.b.w};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t h = w[j / 2] >> (16 * (j & 1));
    v[j] += type == MIMIR_B200_T_F32 ? __uint_as_float(w[j]) : type == MIMIR_B200_T_F16 ? __half2float(__ushort_as_half(static_cast<unsigned short>(h))) : __uint_as_float(h << 16);
  }
}

// FOURS: how many times four warps take the results.  Sixteen warps where a CTA has the SM to itself: each has its units one after the other, some
// 0.9 us for 16 rows of a gated pair.  HELD: not 0 where the CTA's share of n_in is more than a sum in tensor memory
// takes (linear.cuh): how many times 16 sums a thread holds then.
template <bool F8, bool GATED, int HELD, int FOURS>
__global__ void __launch_bounds__(64 + 128 * FOURS, FOURS == 2 ? 2 : 1)
linear_rows_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_up,
                   const __grid_constant__ RowParams rp) {
  constexpr int G = GATED ? 2 : 1, RESULT_THREADS = 128 * FOURS;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t bars[2 * MAX_STAGES + 5];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_word;
  __shared__ float x_scales[F8 ? 256 : 1];
  uint64_t *full_bar = bars, *empty_bar = bars + MAX_STAGES, *acc_full = bars + 2 * MAX_STAGES, *drained = acc_full + 2, *acc_empty = acc_full + 3;
  volatile int* abort_flag = &abort_word;

  const LinearParams& p = rp.l;
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int rank = rp.cluster > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int tile = static_cast<int>(blockIdx.x) / rp.cluster, ft = tile / rp.row_tiles, rt = tile - ft * rp.row_tiles, n = rp.rows_tile;
  const int feature0 = ft * rp.features, x_row0 = rt * n;
  const int b0 = share_begin(p.kblocks, rank, rp.cluster), b1 = share_begin(p.kblocks, rank + 1, rp.cluster);

  // The producer starts on its own: barriers and the first few blocks, before the others are through with their set-up.  (Not all that the ring
  // holds: asking for it takes as long as its bytes need, and the first instruction would wait for that.)
  constexpr int per_block = F8 ? LIN_BLOCK : LIN_BLOCK / 2;
  const int w_bytes = rp.features * LIN_BLOCK;
  const int at_once = min(min(rp.stages, b1 - b0), EARLY);
  auto load_block = [&](int stage, int b) {
    uint8_t* base = smem + stage * rp.stage_bytes;
    uint64_t* bar = &full_bar[stage];
    mbar_expect_tx(bar, static_cast<uint32_t>(rp.stage_bytes));
    tma_load_2d(base, &map_w, bar, b * per_block, feature0);
    if constexpr (GATED) tma_load_2d(base + w_bytes, &map_up, bar, b * per_block, feature0);
    tma_load_2d(base + G * w_bytes, &map_x, bar, b * per_block, x_row0);
  };
  if (warp == 0) {
    if (lane < rp.stages) {
      mbar_init(&full_bar[lane], 1);
      mbar_init(&empty_bar[lane], 1);
    } else if (lane >= 27) {
      mbar_init(&acc_full[lane - 27], lane < 30 ? 1 : RESULT_THREADS / 32);  // (acc_full[0, 1], drained, acc_empty[0, 1])
    } else if (lane == 26) {
      *abort_flag = 0;
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async_smem();
    __syncwarp();
    const bool one = elect_one();
    // the first weights into L2 while the kernel before this one finishes (what it may still write there is not lost: L2 is where both meet)
    for (int i = 0; i < min(AHEAD, b1 - b0); ++i) {
      if (one) {
        tma_prefetch_2d(&map_w, (b0 + i) * per_block, feature0);
        if constexpr (GATED) tma_prefetch_2d(&map_up, (b0 + i) * per_block, feature0);
      }
      __syncwarp();
    }
    pdl_wait();
    for (int i = 0; i < at_once; ++i) {
      if (one) load_block(i, b0 + i);
      __syncwarp();
    }
  } else if (warp == 1) {
    tmem_alloc(&tmem_slot, rp.tmem_cols);
    tmem_relinquish();
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = tmem_slot;
  if (rp.cluster > 1) cluster_arrive();  // (waited for before the first write into another CTA)
  pdl_early_if(rp.early);
  pdl_wait();

  // tensor memory: the sums; HELD: two such regions that the instructions add up in by turns, the whole in the first at the end
  const uint32_t region = static_cast<uint32_t>(G * n);
  const int quad = warp & 3, four = (warp - 2) >> 2;
  const uint32_t lanes = tmem + (static_cast<uint32_t>(quad * 32) << 16);

  if (warp == 0) {
    const bool one = elect_one();
    int stage = at_once == rp.stages ? 0 : at_once;
    uint32_t phase = at_once == rp.stages ? 1 : 0;
    int issued = at_once;
    for (; b0 + issued < b1; ++issued) {
      if (!mbar_wait_warp(&empty_bar[stage], phase ^ 1, abort_flag, p.err_word, 111)) break;
      if (one) load_block(stage, b0 + issued);
      __syncwarp();
      if (++stage == rp.stages) { stage = 0; phase ^= 1; }
    }
    // what was asked for has landed and been used (or the abort flag is up) before the ring becomes something else
    bool ok = true;
    for (int s = 0; s < rp.stages && ok; ++s) {
      ok = mbar_wait_warp(&empty_bar[stage], phase ^ 1, abort_flag, p.err_word, 112);
      if (++stage == rp.stages) { stage = 0; phase ^= 1; }
    }
    if (!ok) {  // a wait gave up: nothing may still be on its way into shared memory when the CTA ends
      int still = 0;
      for (int i = max(0, issued - rp.stages); i < issued; ++i)
        mbar_wait_warp(&full_bar[i % rp.stages], static_cast<uint32_t>((i / rp.stages) & 1), &still, p.err_word, 116);
    }
  } else if (warp == 1) {
    const bool one = elect_one();
    const uint32_t idesc = linear_idesc(RM, n) | p.formats;
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 0;
    bool ready = false, ok = true;
    for (int b = b0; b < b1 && ok;) {
      uint32_t d = tmem;
      if constexpr (HELD > 0) {
        if (!mbar_wait_warp(&acc_empty[acc], acc_phase ^ 1, abort_flag, p.err_word, 113)) { ok = false; break; }
        tcgen05_fence_after();
        d = tmem + acc * region;
      }
      const int from = b, end = HELD ? min(b1, b + p.chunk) : b1;
      for (; b < end; ++b) {
        if (!__all_sync(0xffffffffu, ready) && !mbar_wait_warp(&full_bar[stage], phase, abort_flag, p.err_word, 114)) { ok = false; break; }
        tcgen05_fence_after();
        const uint32_t sa = smem_u32(smem + stage * rp.stage_bytes);
        const uint64_t dw = make_smem_desc(sa, LIN_BLOCK), du = dw + (w_bytes >> 4), dx = dw + (G * w_bytes >> 4);
        uint64_t* done = &empty_bar[stage];
        if (++stage == rp.stages) { stage = 0; phase ^= 1; }
        ready = mbar_test(&full_bar[stage], phase);
        if (one) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {  // 32 bytes further in a descriptor's address field: 2
            const uint32_t add = (b != from || k != 0) ? 1u : 0u;
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
    if (!ok) {  // ... nor an instruction at work
      int still = 0;
      if (one) umma_commit(drained);
      __syncwarp();
      mbar_wait_warp(drained, 0, &still, p.err_word, 117);
    }
  }

  // ---- results: a lane has a feature, a register a row of x ----
  // (warps whose 32 lanes are all behind the CTA's features keep the barriers company)
  const bool results = warp >= 2, busy = results && quad * 32 < rp.features;
  const int size = p.out_type == MIMIR_B200_T_F32 ? 4 : 2, units = n / UNIT;
  const int u0 = share_begin(units, rank, rp.cluster), u1 = share_begin(units, rank + 1, rp.cluster);  // the units that this CTA finishes
  const int limit = min(p.n_out, feature0 + rp.features), feature = feature0 + quad * 32 + lane;
  float w_scale = 1.0f, up_scale = 1.0f, bias = 0.0f, up_bias = 0.0f;
  bool ok = true;
  // the four warps' number `fourth` writes eight features from `col` on of two rows of a unit; their residual is on its way a unit ahead
  const int mine = u0 + ((four - u0) & (FOURS - 1)), fourth = static_cast<int>(threadIdx.x - 64) & 127, col = feature0 + (fourth & 15) * 8;
  Eight next[2];
  auto fetch = [&](int u) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = x_row0 + u * UNIT + 8 * i + (fourth >> 4);
      if (u < u1 && row < p.rows && col < limit)
        next[i] = fetch_eight(p.residual + row * p.residual_row + static_cast<long long>(col) * size, p.out_type, col + 8 <= p.n_out && p.vec_res, limit - col);
    }
  };
  if (results) {
    if (!GATED && p.residual) fetch(mine);
    // all that the results need besides the sums, while these are made
    if (feature < limit) {
      if constexpr (F8) w_scale = load_float(p.w_scale + feature);
      if constexpr (F8 && GATED) up_scale = load_float(p.up_scale + feature);
      if (p.bias) bias = load_float(p.bias + feature);
      if (GATED && p.up_bias) up_bias = load_float(p.up_bias + feature);
      if (!GATED && p.residual)  // (into L2)
        for (int i = u0 * UNIT + four; i < u1 * UNIT && x_row0 + i < p.rows; i += FOURS)
          prefetch_line(p.residual + (x_row0 + i) * p.residual_row + static_cast<long long>(feature) * size);
    }
    if constexpr (F8) {
      const int i = static_cast<int>(threadIdx.x) - 64;
      if (i < n) x_scales[i] = x_row0 + i < p.rows ? load_float(p.x_scale + x_row0 + i) : 0.0f;
    }
    __syncwarp();
    if constexpr (HELD > 0) {
      // sums of a chunk at a time out of tensor memory, added up rounded, and the whole back into its first region (a warp's columns are its own)
      int acc = 0;
      uint32_t acc_phase = 0;
      float v[HELD][16];  // 16 rows each, of a gated pair first the one, then the other
#pragma unroll
      for (int i = 0; i < HELD; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) v[i][j] = 0.0f;
      for (int b = b0; b < b1; b += p.chunk) {
        ok = mbar_wait_warp(&acc_full[acc], acc_phase, abort_flag, p.err_word, 115);
        if (!ok) break;
        tcgen05_fence_after();
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
          const uint32_t col = static_cast<uint32_t>((FOURS * i + four) * 16);
          if (col >= region || !busy) continue;
          float w[16];
          tmem_ld_32x16(lanes + acc * region + col, w);
#pragma unroll
          for (int j = 0; j < 16; ++j) v[i][j] += w[j];
        }
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[acc]);
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
      }
#pragma unroll
      for (int i = 0; i < HELD; ++i) {
        const uint32_t col = static_cast<uint32_t>((FOURS * i + four) * 16);
        if (col >= region || !busy) continue;
        uint32_t w[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) w[j] = __float_as_uint(v[i][j]);
        tmem_st_32x16(lanes + col, w);
      }
      tmem_wait_st();
      tcgen05_fence_before();
    } else {
      ok = mbar_wait_warp(&acc_full[0], 0, abort_flag, p.err_word, 115);
    }
    // (the rows' scales are there; sums taken out change hands between a lane's warps)
    if (F8 || HELD > 0) result_warps_sync(RESULT_THREADS);
    tcgen05_fence_after();
  }
  if (rp.cluster > 1) {
    __syncwarp();
    cluster_wait();  // every CTA of the cluster has begun
    if (rp.parts_at == 0) {
      __syncthreads();
      cluster_sync_all();  // every ring of the cluster is done with
    }
    if (busy && ok) {
      int who = 0, r0 = 0, r1 = share_begin(units, 1, rp.cluster);  // who finishes a unit, and that one's units
      for (int u = four; u < units; u += FOURS) {
        while (u >= r1) r0 = r1, r1 = share_begin(units, ++who + 1, rp.cluster);
        // [sender][gate, up][unit][four rows][feature][row]
        const int wide = r1 - r0, at = rp.parts_at + (rank * G * wide + u - r0) * UNIT * RM * 4 + (quad * 32 + lane) * 16;
        const uint32_t dst = mapa_shared(smem_u32(smem + at), static_cast<uint32_t>(who));
        float z[16], y[16];
        tmem_ld_32x16(lanes + static_cast<uint32_t>(u * UNIT), z);
        if constexpr (GATED) tmem_ld_32x16(lanes + static_cast<uint32_t>(n + u * UNIT), y);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          st_cluster4(dst + j * RM * 16, z + 4 * j);
          if constexpr (GATED) st_cluster4(dst + static_cast<uint32_t>(wide * UNIT * RM * 4 + j * RM * 16), y + 4 * j);
        }
      }
    }
    __syncwarp();
    cluster_sync_all();  // every share has arrived
  }
  if (results) {
    // Sixteen rows at a time: a lane's sums of its feature, scaled and activated; by way of shared memory to lanes that have eight neighbouring
    // features of a row, for the residual and the result in 16 bytes (two bytes a lane took 0.5 us for eight rows, of 0.9 in all).
    float* const turns = reinterpret_cast<float*>(smem + rp.turn_at) + four * 2 * UNIT * RM;
    const float4* parts = reinterpret_cast<const float4*>(smem + rp.parts_at) + quad * 32 + lane;
    const int wide = u1 - u0;
    const bool go = ok && !*abort_flag;
    int flip = 0;
#pragma unroll 1
    for (int u = mine; u < u1; u += FOURS, flip ^= 1) {
      if (x_row0 + u * UNIT >= p.rows) break;
      Eight now[2];
      if (!GATED && p.residual) {
        now[0] = next[0], now[1] = next[1];
        fetch(u + FOURS);
      }
      float* turn = turns + flip * UNIT * RM;
      if (busy) {
        float z[16], y[16];
        if (rp.cluster == 1) {
          tmem_ld_32x16(lanes + static_cast<uint32_t>(u * UNIT), z);
          if constexpr (GATED) tmem_ld_32x16(lanes + static_cast<uint32_t>(n + u * UNIT), y);
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) z[j] = y[j] = 0.0f;
        }
        for (int o = 0; o < rp.cluster && rp.cluster > 1; ++o) {
          const float4* from = parts + (o * G * wide + u - u0) * 4 * RM;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 a = from[j * RM];
            z[4 * j] += a.x, z[4 * j + 1] += a.y, z[4 * j + 2] += a.z, z[4 * j + 3] += a.w;
            if constexpr (GATED) {
              const float4 b = from[(wide * 4 + j) * RM];
              y[4 * j] += b.x, y[4 * j + 1] += b.y, y[4 * j + 2] += b.z, y[4 * j + 3] += b.w;
            }
          }
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          if constexpr (F8) {
            const float sx = x_scales[u * UNIT + j];
            z[j] = fmaf(z[j] * sx, w_scale, bias);
            if constexpr (GATED) y[j] = fmaf(y[j] * sx, up_scale, up_bias);
          } else {
            z[j] += bias;
            if constexpr (GATED) y[j] += up_bias;
          }
        }
        activate(z, p.act, p.out_type);
#pragma unroll
        for (int j = 0; j < 16; ++j) turn[j * RM + quad * 32 + lane] = GATED ? z[j] * y[j] : z[j];
      }
      four_warps_sync(four);
      if (col < limit && go) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = x_row0 + u * UNIT + 8 * i + (fourth >> 4);
          if (row >= p.rows) break;
          const float4 a = *reinterpret_cast<const float4*>(turn + (i * 128 + fourth) * 8), b = *reinterpret_cast<const float4*>(turn + (i * 128 + fourth) * 8 + 4);
          float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
          if (!GATED && p.residual) add_eight(now[i], p.out_type, v);
          store_eight(p.out + row * p.out_row + static_cast<long long>(col) * size, p.out_type, col + 8 <= p.n_out && p.vec_out, limit - col, v);
        }
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
  int rows_tile, row_tiles, features, cluster, per_sm, stages, stage_bytes, parts_at, turn_at, tmem_cols;
  bool chunks;
  size_t smem;
  long long ctas;
  double us;
};

// The shape of a launch with that many features to a CTA, `cluster` CTAs that share n_in, per_sm of them on an SM; false where it does not fit.
bool shape_of(const MimirLinear& a, bool gated, int features, int cluster, int per_sm, RowShape* s) {
  const int g = gated ? 2 : 1, f32 = a.out_type == MIMIR_B200_T_F32;
  const int most = (f32 ? 128 : 256) / g;
  s->row_tiles = (a.rows + most - 1) / most;
  s->rows_tile = round_up((a.rows + s->row_tiles - 1) / s->row_tiles, UNIT);
  s->features = features, s->cluster = cluster, s->per_sm = per_sm;
  s->ctas = static_cast<long long>(s->row_tiles) * ((a.n_out + features - 1) / features) * cluster;
  const int kblocks = linear_kblocks(a), need = (kblocks + cluster - 1) / cluster;  // stages that a CTA can fill at all
  if (cluster > 1 && per_sm > 1) return false;
  if (s->ctas > 0x3fffffffLL || (cluster > 1 && kblocks < 2 * cluster)) return false;
  s->chunks = need > linear_chunk(a);
  s->tmem_cols = 32;
  while (s->tmem_cols < (s->chunks ? 2 : 1) * g * s->rows_tile) s->tmem_cols *= 2;
  if (s->tmem_cols > 512 / per_sm) return false;
  const int units = s->rows_tile / UNIT, parts = cluster == 1 ? 0 : cluster * ((units + cluster - 1) / cluster) * UNIT * g * RM * 4;
  s->stage_bytes = (g * features + s->rows_tile) * LIN_BLOCK;
  // (an instruction reads 128 rows from the start of the features' that it is given)
  const int pad = std::max(0, RM - features - s->rows_tile) * LIN_BLOCK;
  const int space = (per_sm == 2 ? DYNAMIC_TWO : DYNAMIC) - 1024;
  const int turns = (per_sm == 2 ? 2 : 4) * TURN;
  auto stages_in = [&](int bytes) { return bytes < 0 ? 0 : std::min(std::min(bytes / s->stage_bytes, MAX_STAGES), need); };
  s->stages = stages_in(space - pad - parts);
  s->parts_at = std::max(s->stages * s->stage_bytes + pad, turns);  // (results are turned around in the ring)
  if (s->parts_at + parts > space) s->stages = 0;
  if (parts == 0 || (s->stages < need && (s->stages < 4 || s->stages * s->stage_bytes < 96 * 1024))) {  // too little of a ring: the sums come into it afterwards
    s->stages = stages_in(space - pad);
    s->parts_at = 0;
  }
  if (s->stages < 2 && s->stages < need) return false;
  s->turn_at = s->parts_at ? 0 : parts;
  if (s->turn_at + turns > space) return false;
  s->smem = static_cast<size_t>(s->parts_at ? s->parts_at + parts : std::max(s->stages * s->stage_bytes + pad, s->turn_at + turns)) + 1024;
  if (cluster > 1) s->smem = std::max(s->smem, ALONE);
  return true;
}

// Stands for the kernel where the runtime is asked how many clusters run at the same time (of kernels that allocate tensor memory it counts one CTA
// to an SM).  A cluster lives in one GPC, whose SM count is no multiple of it.
__global__ void __launch_bounds__(64 + 512, 1) rows_footprint_kernel() {}
struct ClusterTable { int n[MAX_CLUSTER + 1]; };
const ClusterTable* active_clusters() {
  static PerDeviceOnce once;
  static ClusterTable table[64];  // (PerDeviceOnce counts as many devices)
  ClusterTable& t = table[ctx().device];
  const int rc = once.run([&]() -> int {
    MB_CUDA(cudaFuncSetAttribute(rows_footprint_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, DYNAMIC));
    for (int size = 1; size <= MAX_CLUSTER; ++size) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(static_cast<unsigned>(size * 512));
      cfg.blockDim = dim3(64 + 512);
      cfg.dynamicSmemBytes = DYNAMIC;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = static_cast<unsigned>(size);
      attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      MB_CUDA(cudaOccupancyMaxActiveClusters(&t.n[size], rows_footprint_kernel, &cfg));
    }
    return MIMIR_B200_OK;
  });
  return rc == MIMIR_B200_OK ? &t : nullptr;
}

// The quickest shape by an estimate in us.  A round of CTAs loads (at most 120 KB an us each, 18.4 MB in all; a ring that does not hold all of a
// CTA's blocks is waited for 0.34 us at a time) and multiplies (an instruction of 128 x N takes 46 cycles, from N = 61 on 0.75 N, a block 70
// more), or waits for the weights from memory, up to a tenth longer where SMs idle; then come 0.42 us for each unit of 16 rows that a warp
// finishes, and 1.85 and more for the meeting of a cluster; of equals, CTAs of middling size.  The numbers were fitted to earlier forms of both
// kernels.  With the present ones, over 228 products (1 to 2 048 rows, n_in 512 to 16 384, n_out 640 to 32 000, 16 and 8 bits, gated or not, up
// to 46 shapes each): the shape taken, or the kernel of tiles instead, is on average 2.7 % slower than the quickest, half of them at most 0.4 %,
// 20 more than 10 %, at worst 38 % (384 rows x 1 024 x 32 000 in 8 bits 29.2 us, in tiles 21.2).
RowShape row_shape(const MimirLinear& a, bool gated) {
  RowShape best = {};
  best.us = 1e30;
  const ClusterTable* active = active_clusters();
  if (!active) return best;
  const int g = gated ? 2 : 1, sms = ctx().sm_count;
  const double blocks = std::ceil(static_cast<double>(a.n_in) * type_bytes(a.type) / LIN_BLOCK), hbm = blocks * LIN_BLOCK * g * a.n_out / 6.55e6;
  for (int cluster = 1; cluster <= MAX_CLUSTER; ++cluster)
    for (int features = RM; features >= 16; features -= 8)
      for (int per_sm = 1; per_sm <= (cluster == 1 ? 2 : 1); ++per_sm) {
        RowShape s;
        if (!shape_of(a, gated, features, cluster, per_sm, &s)) continue;
        const double at_once = static_cast<double>(active->n[cluster]) * cluster * per_sm, rounds = std::ceil(s.ctas / at_once), mine = std::ceil(blocks / cluster);
        if (at_once <= 0) continue;
        const double load = std::max(s.stage_bytes / 120e3, s.stages < mine ? 0.34 / s.stages : 0.0);
        const double mma = (70.0 + g * 4 * std::max(46.0, 0.75 * s.rows_tile)) / 1850.0;
        const double busy = s.ctas / (std::ceil(static_cast<double>(s.ctas) / sms) * sms);  // share of the SMs, over the time
        const double loop = std::max({rounds * mine * std::max(load, mma) * per_sm, hbm * (1.1 - 0.1 * busy), s.ctas * mine * s.stage_bytes / 18.4e6});
        const int turns = per_sm == 2 ? 2 : 4, units = ((s.rows_tile / UNIT + cluster - 1) / cluster + turns - 1) / turns;
        const double meet = cluster == 1 ? 0.0 : 1.85 + 0.019 * s.rows_tile * g * (cluster - 1) / cluster + (s.parts_at ? 0.0 : 2.0);
        s.us = 1.9 + loop + (0.23 + 0.42 * g * units + meet) * (per_sm == 1 ? rounds : (rounds + 1) / 2) + 0.003 * std::abs(features - 64);
        if (s.us < best.us) best = s;
      }
  return best;
}

template <bool F8, bool GATED, int HELD, int FOURS>
int launch_as(const CUtensorMap (&maps)[3], const RowParams& p, const RowShape& s, cudaStream_t st) {
  auto kern = linear_rows_kernel<F8, GATED, HELD, FOURS>;
  static PerDeviceOnce once;
  MB_TRY(once.run([&]() -> int {
    MB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, DYNAMIC));
    return MIMIR_B200_OK;
  }));
  MB_TRY(launch_pdl(kern, dim3(static_cast<unsigned>(s.ctas)), dim3(64 + 128 * FOURS), s.smem, st, s.cluster, maps[0], maps[1], maps[2], p));
  count_launch();
  return MIMIR_B200_OK;
}
template <bool F8, bool GATED>
int launch_for(const CUtensorMap (&maps)[3], const RowParams& p, const RowShape& s, cudaStream_t st) {
  const int region = (GATED ? 2 : 1) * s.rows_tile;  // (at most 256, of two CTAs to an SM 128: tensor memory)
  if (s.per_sm == 2) {
    if (!s.chunks) return launch_as<F8, GATED, 0, 2>(maps, p, s, st);
    return region <= 64 ? launch_as<F8, GATED, 2, 2>(maps, p, s, st) : launch_as<F8, GATED, 4, 2>(maps, p, s, st);
  }
  if (!s.chunks) return launch_as<F8, GATED, 0, 4>(maps, p, s, st);
  return region <= 128 ? launch_as<F8, GATED, 2, 4>(maps, p, s, st) : launch_as<F8, GATED, 4, 4>(maps, p, s, st);
}

// The shapes that this thread asked for last (looking through all of them takes longer than a launch).
struct ShapeKey {
  int rows, n_in, n_out, type, f32, gated, device;
  bool operator==(const ShapeKey& o) const {
    return rows == o.rows && n_in == o.n_in && n_out == o.n_out && type == o.type && f32 == o.f32 && gated == o.gated && device == o.device;
  }
};
const RowShape& known_shape(const MimirLinear& a, bool gated) {
  struct Entry {
    ShapeKey key = {};  // (no rows: none)
    RowShape shape;
  };
  static thread_local Entry entries[64];
  const ShapeKey key = {a.rows, a.n_in, a.n_out, a.type, a.out_type == MIMIR_B200_T_F32, gated, ctx().device};
  const uint32_t h = (static_cast<uint32_t>(a.rows) * 0x9E3779B1u ^ static_cast<uint32_t>(a.n_in) * 0x85EBCA77u ^ static_cast<uint32_t>(a.n_out) * 0xC2B2AE3Du ^
                      static_cast<uint32_t>(key.type * 4 + key.f32 * 2 + key.gated) * 0x27D4EB2Fu) >> 26;
  Entry& e = entries[h];
  if (!(e.key == key)) {
    const RowShape s = row_shape(a, gated);
    if (s.us > 1e29) {  // (no cluster can be asked for: the caller's launch says so; not kept)
      static thread_local RowShape none;
      none = s;
      return none;
    }
    e.shape = s, e.key = key;
  }
  return e.shape;
}

}  // namespace

double linear_rows_us(const MimirLinear& a, bool gated) { return a.rows > 4096 ? 1e30 : known_shape(a, gated).us; }

int launch_linear_rows(const MimirLinear& a, const LinearParams& l, bool gated, cudaStream_t st) {
  const RowShape& s = known_shape(a, gated);
  CUtensorMap maps[3];
  MB_TRY(make_operand_map(&maps[0], a.x, a.type, a.rows, a.n_in, a.x_stride, s.rows_tile));
  MB_TRY(make_operand_map(&maps[1], a.w, a.type, a.n_out, a.n_in, a.w_stride, s.features));
  maps[2] = maps[1];
  if (gated) MB_TRY(make_operand_map(&maps[2], a.up, a.type, a.n_out, a.n_in, a.up_stride, s.features));
  RowParams p = {};
  p.l = l, p.rows_tile = s.rows_tile, p.row_tiles = s.row_tiles, p.features = s.features, p.cluster = s.cluster;
  p.stages = s.stages, p.stage_bytes = s.stage_bytes, p.parts_at = s.parts_at, p.turn_at = s.turn_at, p.tmem_cols = s.tmem_cols;
  p.early = pdl_small_grid(static_cast<unsigned>(s.ctas));
  if (a.type == MIMIR_B200_T_E4M3) return gated ? launch_for<true, true>(maps, p, s, st) : launch_for<true, false>(maps, p, s, st);
  return gated ? launch_for<false, true>(maps, p, s, st) : launch_for<false, false>(maps, p, s, st);
}

}  // namespace mb
