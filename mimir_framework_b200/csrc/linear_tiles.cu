// linear_tiles.cu — products of many rows.
//
// Clusters of two CTAs on neighbouring SMs share a tile of 256 rows x 256 features (tcgen05 with cta_group::2): each loads its own 128 rows of x
// and half of the weights' 256, so that a byte of operands in shared memory is used 256 times.  A gated pair's tile is 128 features of each matrix:
// the leader's half of the N side is the gate's, the other's is up's, and a thread finds both of an output in its own row of
// tensor memory.  The kernel is persistent, tensor memory holds two accumulators of 256 columns:
//   warp 0     TMA into a ring of five stages of 32 KB a CTA
//   warp 1     (the leader's) issues the instructions for both
//   the others results: two or four warps for each 32 rows, as many parts of the columns; 32 columns at a time through activation, gate and residual
// Four where the results bound the kernel, two where the instructions do, as a thread then has 168 registers.  The time with four over that with two, by the
// K blocks of a product (8 192 rows x 4 096 features, off their boundary 4 000 x 4 001; without an activation, and with GELU):
//                                           2          4          8         16         24         48         96
//   16 bits                             .87 .78    .88 .80    .99 .80   1.05 .94  1.03 1.01  1.05  .98  1.03 1.00
//   16 bits, residual                   .86 .77    .89 .78    .89 .82   1.02 .81  1.03  .90  1.01  .99   .99 1.01
//   16 bits, off the boundary           .65 .69    .68 .70    .69 .71    .77 .73   .88  .79  1.02 1.05  1.01 1.02
//   16 bits, off it with residual       .72 .72    .73 .72    .74 .73    .74 .74   .75  .74   .78  .82   .97  .96
//   16 bits, gated                      .96 .90   1.03 .91   1.08 .93   1.15 1.04 1.02  .97  1.01 1.04  1.01 1.01
//   16 bits, gated, off the boundary    .77 .78    .79 .79    .82 .80   1.01 .85  1.09 1.03  1.01 1.03  1.02 1.02
//   E4M3                               1.00 .89   1.00 .90   1.00 .90   1.05 .95  1.05 1.03  1.02 1.00  1.03 1.01
//   E4M3, residual                     1.00 .96   1.03 .97   1.06 .98   1.05 .98  1.06  .98  1.02 1.03   .95 1.02
//   E4M3, off the boundary              .78 .76    .78 .77    .80 .78    .85 .80   .93  .86  1.04 1.02   .99 1.02
//   E4M3, off it with residual          .70 .70    .71 .70    .71 .71    .73 .72   .74  .73   .85  .81  1.01  .95
//   E4M3, gated                         .93 .90    .93 .91    .94 .91   1.02 1.12 1.01 1.01  1.08 1.03  1.02 1.01
//   E4M3, gated, off the boundary       .78 .76    .80 .76    .81 .78    .85 .82  1.04 1.01  1.02 1.02  1.02  .99
// Sums of more inputs than linear.cuh leaves to the tensor core are taken out a chunk at a time and added up in registers (CHUNKS).
#include <algorithm>
#include <cmath>

#include "launch.cuh"
#include "linear.cuh"

namespace mb {
namespace {

constexpr int TM = 128, TN = 256;  // rows of a CTA, columns of an accumulator
constexpr int STAGES = 5, A_BYTES = TM * LIN_BLOCK, W_BYTES = TN / 2 * LIN_BLOCK, STAGE = A_BYTES + W_BYTES;
constexpr int OUT_TILE = 32 * 64;     // 32 rows x 64 bytes of results on their way out
constexpr int TURNS = 16 * OUT_TILE;  // eight warps: two such tiles each, or what turns 32 rows around; sixteen: one, or 16 rows
constexpr int COLS = 2 * TN * 4;      // scales and biases of the columns of four warps
constexpr int SMEM = STAGES * STAGE + TURNS + 4 * COLS + 256 + 1024;
static_assert(SMEM <= 232448, "exceeds the 227 KB of shared memory a CTA may use");

struct TileParams {
  LinearParams l;
  int tiles_m, tiles_n, group_n;
  int full;  // tiles from this one on run as two of half the columns: the last round's, where it would leave half of the SMs idle
};

// Work item t: its tile and, of one that is cut, which half of the columns (else -1).  Groups of group_n column tiles, so that the tiles
// at work at one time share rows and weights in L2.
__device__ __forceinline__ int tile_of(const TileParams& p, int t, int& tm, int& tn) {
  int cut = -1;
  if (t >= p.full) {
    cut = (t - p.full) & 1;
    t = p.full + ((t - p.full) >> 1);
  }
  const int per = p.group_n * p.tiles_m, g = t / per, r = t - g * per, n0 = g * p.group_n, wide = min(p.group_n, p.tiles_n - n0);
  tm = r / wide;
  tn = n0 + r % wide;
  return cut;
}

// scale and bias of 32 neighbouring features, from shared memory
template <bool F8>
__device__ __forceinline__ void scaled(float (&v)[32], float sx, const float* scale, const float* bias) {
#pragma unroll
  for (int j = 0; j < 32; j += 4) {
    const float4 b = *reinterpret_cast<const float4*>(bias + j);
    if constexpr (F8) {
      const float4 s = *reinterpret_cast<const float4*>(scale + j);
      v[j] = fmaf(v[j] * sx, s.x, b.x), v[j + 1] = fmaf(v[j + 1] * sx, s.y, b.y);
      v[j + 2] = fmaf(v[j + 2] * sx, s.z, b.z), v[j + 3] = fmaf(v[j + 3] * sx, s.w, b.w);
    } else {
      v[j] += b.x, v[j + 1] += b.y, v[j + 2] += b.z, v[j + 3] += b.w;
    }
  }
}

// 32 results of this lane's row, columns col0 on, to where they belong
template <int N>
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }
template <int ROWS, int BUFFERS>
__device__ __forceinline__ void write_out(const LinearParams& p, const CUtensorMap& map_out, float (&v)[32], int row0, int col0, float* turn, int& flip) {
  const int lane = threadIdx.x & 31, row = row0 + lane;
  const int size = p.out_type == MIMIR_B200_T_F32 ? 4 : 2;
  if (p.vec_out && (col0 + 32 <= p.n_out || (p.n_out * size) % 16 == 0)) {
    // rows on 16 bytes: tiles of 32 rows x 64 bytes in shared memory (64-byte swizzle: no conflicts), each one copy, which stops at the last row and, where
    // that is on 16 bytes too (else it would write behind it), the last column
    if (p.residual && row < p.rows) {
      const char* r = p.residual + row * p.residual_row + static_cast<long long>(col0) * size;
      if (p.vec_res && col0 + 32 <= p.n_out) {
        if (size == 4) {
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            float q[8];
            unpack8<MIMIR_B200_T_F32>(load8<MIMIR_B200_T_F32>(r + j * 4), q);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[j + e] += q[e];
          }
        } else {
          Raw8<MIMIR_B200_T_F16> raw[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) raw[j] = load8<MIMIR_B200_T_F16>(r + j * 16);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float q[8];
            if (p.out_type == MIMIR_B200_T_F16) {
              unpack8<MIMIR_B200_T_F16>(raw[j], q);
            } else {
              Raw8<MIMIR_B200_T_BF16> b;
#pragma unroll
              for (int e = 0; e < 4; ++e) b.w[e] = raw[j].w[e];
              unpack8<MIMIR_B200_T_BF16>(b, q);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) v[8 * j + e] += q[e];
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (col0 + j < p.n_out) v[j] += load_typed(r + j * size, p.out_type);
      }
    }
    const int copies = size == 4 ? 2 : 1;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (h == copies) break;
      uint32_t w[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        if (size == 4) {
          w[j] = __float_as_uint(v[16 * h + j]);
        } else if (p.out_type == MIMIR_B200_T_F16) {
          const __half2 x = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
          w[j] = *reinterpret_cast<const uint32_t*>(&x);
        } else {
          const __nv_bfloat162 x = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
          w[j] = *reinterpret_cast<const uint32_t*>(&x);
        }
      }
      uint8_t* const tile = reinterpret_cast<uint8_t*>(turn) + flip * OUT_TILE;
      if (BUFFERS == 2) flip ^= 1;
      if (lane == 0) bulk_wait_read<BUFFERS - 1>();  // the copy that was there has read it
      __syncwarp();
#pragma unroll
      for (int c = 0; c < 4; ++c)
        *reinterpret_cast<uint4*>(tile + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4)) = make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if (row0 < p.rows && col0 + 16 * h < p.n_out) tma_store_2d(&map_out, tile, col0 + 16 * h, row0);
        bulk_commit();
      }
    }
    return;
  }
  // rows off their boundary, and the last columns: turned around, so that a warp's lanes write neighbours, 16 columns of two rows at a time
  if (p.vec_out) {
    if (lane == 0) bulk_wait_read<0>();
    __syncwarp();
  }
  const int at = lane & 15;
#pragma unroll
  for (int c0 = 0; c0 < 32; c0 += 16) {
    const int col = col0 + c0 + at;
#pragma unroll
    for (int r0 = 0; r0 < 32; r0 += ROWS) {
      if (ROWS == 32 || (lane & 16) == r0) {
#pragma unroll
        for (int j = 0; j < 16; ++j) turn[(lane & (ROWS - 1)) * 17 + j] = v[c0 + j];
      }
      __syncwarp();
      const int rows = min(ROWS, p.rows - row0 - r0);
      if (col < p.n_out) {
        char* o = p.out + (row0 + r0) * p.out_row + static_cast<long long>(col) * size;
        const char* r = p.residual ? p.residual + (row0 + r0) * p.residual_row + static_cast<long long>(col) * size : nullptr;
#pragma unroll
        for (int i0 = 0; i0 < ROWS; i0 += 16) {
          float q[8];
          if (p.residual) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int k = i0 + 2 * i + (lane >> 4);
              q[i] = k < rows ? load_typed(r + k * p.residual_row, p.out_type) : 0.0f;
            }
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int k = i0 + 2 * i + (lane >> 4);
            if (k < rows) store_typed(o + k * p.out_row, p.out_type, p.residual ? turn[k * 17 + at] + q[i] : turn[k * 17 + at]);
          }
        }
      }
      __syncwarp();
    }
  }
}

template <bool F8, bool GATED, bool CHUNKS, int PARTS>
__global__ void __launch_bounds__(64 + 128 * PARTS, 1)
linear_tiles_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_up,
                    const __grid_constant__ CUtensorMap map_out, const __grid_constant__ TileParams tp) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* turns = reinterpret_cast<float*>(smem + STAGES * STAGE);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE + TURNS + 4 * COLS);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* acc_full = empty_bar + STAGES;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* drained = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const LinearParams& p = tp.l;
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1, all = tp.tiles_m * tp.tiles_n, items = 2 * all - tp.full;
  constexpr int OUT = GATED ? TN / 2 : TN;  // features of a tile
  constexpr int EPI_WARPS = 4 * PARTS, WARP_COLS = COLS / PARTS, TURN = TURNS / EPI_WARPS;
  static_assert(TURN >= (64 / PARTS) * 17 * 4, "a warp's results are turned around in it");

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 2 * EPI_WARPS);  // (the leader's collects both CTAs' warps)
    }
    mbar_init(drained, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async_smem();
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tcgen05_fence_before();
  __syncthreads();
  cluster_sync_all();  // the other's barriers are there
  tcgen05_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();

  if (warp == 0) {
    const bool one = elect_one();
    const CUtensorMap* const wmap = GATED && rank ? &map_up : &map_w;
    constexpr int per_block = F8 ? LIN_BLOCK : LIN_BLOCK / 2;
    int stage = 0, issued = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int t = first; t < items && ok; t += step) {
      int tm, tn;
      const int cut = tile_of(tp, t, tm, tn);
      const int x_row = (2 * tm + rank) * TM;
      int w_row = tn * OUT + (cut > 0 ? OUT / 2 : 0);
      if (!GATED) w_row += rank * (cut >= 0 ? TN / 4 : TN / 2);
      const uint32_t bytes = 2 * (A_BYTES + (cut >= 0 ? W_BYTES / 2 : W_BYTES));
      for (int kb = 0; kb < p.kblocks; ++kb) {
        if (!mbar_wait_warp(&empty_bar[stage], phase ^ 1, abort_flag, p.err_word, 101)) { ok = false; break; }
        if (one) {
          uint8_t* base = smem + stage * STAGE;
          // the leader's barrier counts the bytes of both CTAs, whichever arrive first
          if (rank == 0) mbar_expect_tx(&full_bar[stage], bytes);
          const uint32_t fb = mapa_shared(smem_u32(&full_bar[stage]), 0);
          tma_load_2d_pair(base, &map_x, fb, kb * per_block, x_row);
          tma_load_2d_pair(base + A_BYTES, wmap, fb, kb * per_block, w_row);
          if (cut < 0) tma_load_2d_pair(base + A_BYTES + W_BYTES / 2, wmap, fb, kb * per_block, w_row + LIN_W_BOX);
        }
        __syncwarp();
        if (issued < STAGES) ++issued;
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
      }
    }
    // what was asked for has landed and been used (or the abort flag is up) before the CTA leaves
    int last = stage;
    uint32_t last_phase = phase;
    for (int s = 0; s < STAGES; ++s) {
      if (!mbar_wait_warp(&empty_bar[stage], phase ^ 1, abort_flag, p.err_word, 102)) { ok = false; break; }
      if (++stage == STAGES) { stage = 0; phase ^= 1; }
    }
    if (!ok && rank == 0) {
      // a wait gave up: nothing may still be on its way into shared memory when the CTA ends (the barriers count both CTAs' copies, and the other leaves with
      // this one)
      int still = 0;
      for (int s = 0; s < issued; ++s) {
        if (--last < 0) { last = STAGES - 1; last_phase ^= 1; }
        mbar_wait_warp(&full_bar[last], last_phase, &still, p.err_word, 106);
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const bool one = elect_one();
      const uint32_t id_full = linear_idesc(2 * TM, TN) | p.formats, id_cut = linear_idesc(2 * TM, TN / 2) | p.formats;
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ready = false, ok = true;
      for (int t = first; t < items && ok; t += step) {
        const uint32_t idesc = t >= tp.full ? id_cut : id_full;
        for (int kb = 0; kb < p.kblocks && ok;) {
          if (!mbar_wait_warp(&acc_empty[acc], acc_phase ^ 1, abort_flag, p.err_word, 103)) { ok = false; break; }
          tcgen05_fence_after();
          const uint32_t d = tmem + static_cast<uint32_t>(acc * TN);
          const int from = kb, to = min(p.kblocks, kb + p.chunk);
          for (; kb < to; ++kb) {
            if (!__all_sync(0xffffffffu, ready) && !mbar_wait_warp(&full_bar[stage], phase, abort_flag, p.err_word, 104)) { ok = false; break; }
            tcgen05_fence_after();
            const uint32_t sa = smem_u32(smem + stage * STAGE);
            const uint64_t da = make_smem_desc(sa, LIN_BLOCK), dw = make_smem_desc(sa + A_BYTES, LIN_BLOCK);
            uint64_t* done = &empty_bar[stage];
            if (++stage == STAGES) { stage = 0; phase ^= 1; }
            ready = mbar_test(&full_bar[stage], phase);
            if (one) {
#pragma unroll
              for (int k = 0; k < 4; ++k) {  // 32 bytes further in a descriptor's address field: 2
                const uint32_t add = (kb != from || k != 0) ? 1u : 0u;
                if constexpr (F8) umma_f8_pair(d, da + 2 * k, dw + 2 * k, idesc, add);
                else umma_bf16_pair(d, da + 2 * k, dw + 2 * k, idesc, add);
              }
              umma_commit_pair(mapa_shared(smem_u32(done), 0));
              umma_commit_pair(mapa_shared(smem_u32(done), 1));
            }
            __syncwarp();
          }
          if (!ok) break;
          if (one) {
            umma_commit_pair(mapa_shared(smem_u32(&acc_full[acc]), 0));
            umma_commit_pair(mapa_shared(smem_u32(&acc_full[acc]), 1));
          }
          __syncwarp();
          if (++acc == 2) { acc = 0; acc_phase ^= 1; }
        }
      }
      if (!ok) {  // ... nor an instruction at work
        int still = 0;
        if (one) umma_commit_pair(mapa_shared(smem_u32(drained), 0));
        __syncwarp();
        mbar_wait_warp(drained, 0, &still, p.err_word, 107);
      }
    }
  } else {
    const int ew = warp - 2, quad = warp & 3, part = ew >> 2;
    float* const turn = turns + ew * (TURN / 4);
    float* const cols = turns + TURNS / 4 + ew * (WARP_COLS / 4);
    int acc = 0, flip = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    auto take = [&]() -> uint32_t {
      ok = mbar_wait_warp(&acc_full[acc], acc_phase, abort_flag, p.err_word, 105);
      tcgen05_fence_after();
      return tmem + (static_cast<uint32_t>(quad * 32) << 16) + static_cast<uint32_t>(acc * TN);
    };
    auto give_back = [&] {
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(mapa_shared(smem_u32(&acc_empty[acc]), 0));
      if (++acc == 2) { acc = 0; acc_phase ^= 1; }
    };
    // What a tile's results need besides its sums is on its way while the tile before it is finished: scales and biases of the warp's columns ([bias][of
    // up][scale][of up], EACH of them, in shared memory when their tile comes) and the scale of the lane's row.
    constexpr int EACH = OUT / PARTS, HOLD = WARP_COLS / 128;
    float next_cols[HOLD], next_sx = 1.0f;
    // this warp's columns of a tile, from its first on, as many as `each` (none where mine >= wide)
    auto my_columns = [&](int tn, int cut, int& wide, int& each, int& mine) -> int {
      wide = cut >= 0 ? OUT / 2 : OUT, each = max(32, wide / PARTS), mine = part * each;
      return tn * OUT + (cut > 0 ? OUT / 2 : 0) + mine;
    };
    auto fetch = [&](int t) {
      if (t >= items) return;
      int tm, tn, wide, each, mine;
      const int cut = tile_of(tp, t, tm, tn), col00 = my_columns(tn, cut, wide, each, mine), row = (2 * tm + rank) * TM + quad * 32 + lane;
      if (F8 && row < p.rows) next_sx = load_float(p.x_scale + row);
#pragma unroll
      for (int i = 0; i < HOLD; ++i) {
        const int which = i * 32 / EACH, col = col00 + i * 32 % EACH + lane;
        if (!F8 && which >= (GATED ? 2 : 1)) break;
        const float* from = GATED ? (which == 0 ? p.bias : which == 1 ? p.up_bias : which == 2 ? p.w_scale : p.up_scale) : which == 0 ? p.bias : p.w_scale;
        next_cols[i] = from && col < p.n_out ? load_float(from + col) : 0.0f;
      }
    };
    fetch(first);
    for (int t = first; t < items && ok; t += step) {
      int tm, tn, wide, each, mine;
      const int cut = tile_of(tp, t, tm, tn), col00 = my_columns(tn, cut, wide, each, mine), nch = mine < wide ? each / 32 : 0;
      const int row0 = (2 * tm + rank) * TM + quad * 32;
      const float sx = next_sx;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < HOLD; ++i)
        if (F8 || i * 32 / EACH < (GATED ? 2 : 1)) cols[i * 32 + lane] = next_cols[i];
      __syncwarp();
      fetch(t + step);
      const float* const my_cols = cols - col00;  // (+ column)
      auto finish = [&](float (&z)[32], float (&u)[32], int col0) {
        scaled<F8>(z, sx, my_cols + (GATED ? 2 : 1) * EACH + col0, my_cols + col0);
        activate(z, p.act, p.out_type);
        if constexpr (GATED) {
          scaled<F8>(u, sx, my_cols + 3 * EACH + col0, my_cols + EACH + col0);
#pragma unroll
          for (int j = 0; j < 32; ++j) z[j] *= u[j];
        }
        write_out<64 / PARTS, 4 / PARTS>(p, map_out, z, row0, col0, turn, flip);
      };
      if constexpr (CHUNKS) {
        constexpr int HELD = TN / PARTS / 32;
        float v[HELD][32];
#pragma unroll
        for (int i = 0; i < HELD; ++i)
#pragma unroll
          for (int j = 0; j < 32; ++j) v[i][j] = 0.0f;
        for (int kb = 0; kb < p.kblocks && ok; kb += p.chunk) {
          const uint32_t at = take();
          if (!ok) break;
#pragma unroll
          for (int i = 0; i < HELD; ++i) {
            // (of a gated pair: first the one's, then the other's)
            const int n = GATED ? i % (HELD / 2) : i;
            if (n >= nch) continue;
            float w[32];
            tmem_ld_32x32(at + static_cast<uint32_t>(mine + n * 32 + (GATED && i >= HELD / 2 ? wide : 0)), w);
#pragma unroll
            for (int j = 0; j < 32; ++j) v[i][j] += w[j];
          }
          give_back();
        }
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < (GATED ? HELD / 2 : HELD); ++i)
          if (i < nch && col00 + i * 32 < p.n_out) finish(v[i], v[GATED ? i + HELD / 2 : i], col00 + i * 32);
      } else {
        const uint32_t at = take();
        if (!ok) break;
#pragma unroll 1
        for (int i = 0; i < nch; ++i) {
          if (col00 + i * 32 >= p.n_out) break;
          float z[32], u[32];
          tmem_ld_32x32(at + static_cast<uint32_t>(mine + i * 32), z);
          if constexpr (GATED) tmem_ld_32x32(at + static_cast<uint32_t>(mine + i * 32 + wide), u);
          finish(z, u, col00 + i * 32);
        }
        give_back();
      }
    }
    if (lane == 0) bulk_wait_read<0>();  // no copy still reads shared memory when the CTA leaves
  }

  tcgen05_fence_before();
  __syncthreads();
  cluster_sync_all();  // neither leaves, or frees tensor memory, while the other may still signal it
  if (warp == 1) {
    tcgen05_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

struct TileShape {
  long long tiles_m, tiles_n;
  int pairs;
  long long full, items;
};
TileShape tile_shape(const MimirLinear& a, bool gated) {
  TileShape s;
  const int out = gated ? TN / 2 : TN;
  s.tiles_m = (a.rows + 2 * TM - 1) / (2 * TM);
  s.tiles_n = (a.n_out + out - 1) / out;
  s.pairs = ctx().sm_count / 2;
  const long long tiles = s.tiles_m * s.tiles_n, rest = tiles % s.pairs;
  s.full = 2 * rest <= s.pairs ? tiles - rest : tiles;
  s.items = 2 * tiles - s.full;
  return s;
}

template <bool F8, bool GATED, bool CHUNKS, int PARTS>
int launch_as(const CUtensorMap (&maps)[4], const TileParams& p, unsigned grid, cudaStream_t st) {
  auto kern = linear_tiles_kernel<F8, GATED, CHUNKS, PARTS>;
  static PerDeviceOnce once;
  MB_TRY(once.run([&]() -> int {
    MB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
    return MIMIR_B200_OK;
  }));
  MB_TRY(launch_pdl(kern, dim3(grid), dim3(64 + 128 * PARTS), SMEM, st, 2, maps[0], maps[1], maps[2], maps[3], p));
  count_launch();
  return MIMIR_B200_OK;
}
template <bool F8, bool GATED>
int launch_for(const CUtensorMap (&maps)[4], const TileParams& p, unsigned grid, cudaStream_t st) {
  if (p.l.kblocks > p.l.chunk) return launch_as<F8, GATED, true, 2>(maps, p, grid, st);
  const bool many = p.l.kblocks <= (p.l.vec_out ? (GATED ? 4 : p.l.residual ? 24 : 8) : p.l.residual ? 96 : 24);  // (both sides at the top)
  return many ? launch_as<F8, GATED, false, 4>(maps, p, grid, st) : launch_as<F8, GATED, false, 2>(maps, p, grid, st);
}

}  // namespace

// An estimate in us (see row_shape): 0.376 for a block of a round of tiles, 0.233 for one of halves.
double linear_tiles_us(const MimirLinear& a, bool gated) {
  const TileShape s = tile_shape(a, gated);
  if (s.items > 0x7fffffffLL / 4) return 1e30;
  const double blocks = std::ceil(static_cast<double>(a.n_in) * type_bytes(a.type) / LIN_BLOCK), rounds = std::ceil(static_cast<double>(s.full) / s.pairs);
  const double hbm = blocks * LIN_BLOCK * (gated ? 2 : 1) * a.n_out / 6.55e6;
  return std::max(blocks * (0.376 * rounds + (s.items > s.full ? 0.233 : 0.0)), hbm) + 6.5 + (a.type == MIMIR_B200_T_E4M3 ? 1.0 : 0.0);
}

int launch_linear_tiles(const MimirLinear& a, const LinearParams& l, bool gated, cudaStream_t st) {
  const TileShape s = tile_shape(a, gated);
  CUtensorMap maps[4];
  MB_TRY(make_operand_map(&maps[0], a.x, a.type, a.rows, a.n_in, a.x_stride, TM));
  MB_TRY(make_operand_map(&maps[1], a.w, a.type, a.n_out, a.n_in, a.w_stride, LIN_W_BOX));
  maps[2] = maps[1];
  if (gated) MB_TRY(make_operand_map(&maps[2], a.up, a.type, a.n_out, a.n_in, a.up_stride, LIN_W_BOX));
  maps[3] = maps[0];
  if (l.vec_out) MB_TRY(make_result_map(&maps[3], a.out, a.out_type, a.rows, a.n_out, a.out_stride));
  TileParams p = {};
  p.l = l, p.tiles_m = static_cast<int>(s.tiles_m), p.tiles_n = static_cast<int>(s.tiles_n), p.full = static_cast<int>(s.full);
  p.group_n = p.tiles_n < 8 ? p.tiles_n : 8;
  const unsigned grid = static_cast<unsigned>(2 * (s.items < s.pairs ? s.items : s.pairs));
  if (a.type == MIMIR_B200_T_E4M3) return gated ? launch_for<true, true>(maps, p, grid, st) : launch_for<true, false>(maps, p, grid, st);
  return gated ? launch_for<false, true>(maps, p, grid, st) : launch_for<false, false>(maps, p, grid, st);
}

}  // namespace mb
