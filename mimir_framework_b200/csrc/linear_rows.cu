// linear_rows.cu — products of few rows: the weights' bytes are the bound, or there are not tiles enough for the SMs.
//
// The weights are the M side (128 features, the lanes of tensor memory), up to 256 rows of x (of a gated pair 128) the N side: an instruction costs
// the same whatever its N, and a narrow N takes little shared memory from the ring that the weights stream through.  A gated pair has two
// accumulators in the same lanes.  Where features and rows make fewer tiles than there are SMs, a cluster of up to eight CTAs takes a few tiles and
// cuts all their K blocks into equal shares, so that a CTA has the end of one tile and the start of the next at most.  The shares of
// a tile meet in shared memory: each of its CTAs finishes some of the rows and gets what the others have of them, in a fixed order, so
// that a result has the same bits every time.
//   warp 0 TMA, warp 1 instructions, warps 2-9 results: two for each 32 features, eight rows of x at a time in turn.
#include <algorithm>

#include "launch.cuh"
#include "linear.cuh"

namespace mb {
namespace {

constexpr int RM = 128;  // features of a CTA
constexpr int MAX_STAGES = 16, THREADS = 320, RESULT_THREADS = 256, W_BYTES = RM * LIN_BLOCK;
constexpr int MAX_CLUSTER = 8, TURNS = 2 * 2 * 8 * RM * 4;
constexpr int STATIC = 3072, DYNAMIC = 232448 - STATIC, DYNAMIC_TWO = (228 * 1024) / 2 - 1024 - STATIC;  // shared memory of a CTA, one or two to an SM
// A CTA of a cluster waits for others that may still be asking for tensor memory.  So that none of them can be kept from it by a CTA that waits
// in the same way, two such CTAs never share an SM: each takes more than half of its shared memory (and more than the other kernels
// of clusters leave, which take at least 104 KB a CTA).
constexpr size_t ALONE = 128 * 1024;

struct RowParams {
  LinearParams l;
  int rows_tile, row_tiles, tiles;  // rows of x of a tile (a multiple of 16), tiles of them, tiles in all
  int group, cluster;               // tiles of a cluster, its CTAs
  int stages, stage_bytes;
  int parts_at, part_bytes;         // other CTAs' shares: where in shared memory (0: the ring, when it is done with), and how much for each of two tiles
  int turn_at;                      // where results are turned around, 16 KB: the ring or behind the shares in it
  int tmem_cols, early;
};

// How a cluster's K blocks fall to its CTAs: CTA c has blocks [total c / size, total (c + 1) / size) of its tiles' in order.
struct Shares {
  int kblocks, total, size;
  // (at most 2^17 blocks of a product, eight products: 32 bits do)
  __host__ __device__ int begin(int c) const { return static_cast<int>(static_cast<unsigned>(total * c) / static_cast<unsigned>(size)); }
  __host__ __device__ int holder(int block) const { return static_cast<int>(static_cast<unsigned>((block + 1) * size - 1) / static_cast<unsigned>(total)); }
};

__device__ __forceinline__ void st_cluster4(uint32_t addr, const float* v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void result_warps_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ void four_warps_sync(int half) { asm volatile("bar.sync %0, 128;" ::"r"(2 + half) : "memory"); }
__device__ __forceinline__ void prefetch_line(const char* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

template <bool F8, bool GATED, bool F32>
__global__ void __launch_bounds__(THREADS, 2)
linear_rows_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_up,
                   const __grid_constant__ RowParams rp) {
  constexpr int G = GATED ? 2 : 1;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t bars[2 * MAX_STAGES + 4];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_word;
  __shared__ float x_scales[F8 ? 2 : 1][F8 ? 256 : 1];
  uint64_t *full_bar = bars, *empty_bar = bars + MAX_STAGES, *acc_full = bars + 2 * MAX_STAGES, *acc_empty = acc_full + 2;
  volatile int* abort_flag = &abort_word;

  const LinearParams& p = rp.l;
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int rank = rp.cluster > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int tile0 = static_cast<int>(blockIdx.x) / rp.cluster * rp.group, n = rp.rows_tile;
  const Shares sh = {p.kblocks, min(rp.group, rp.tiles - tile0) * p.kblocks, rp.cluster};
  // this CTA's blocks: from b0 on in tile `first`, up to b1, which may be the next one's
  const int b0 = sh.begin(rank), b1 = sh.begin(rank + 1), first = b0 / p.kblocks, cut = min(b1, (first + 1) * p.kblocks);
  const int segments = b1 > cut ? 2 : 1;

  // The producer starts on its own: barriers, and what the ring holds at once, before the others are through with their set-up.
  constexpr int per_block = F8 ? LIN_BLOCK : LIN_BLOCK / 2;
  const uint32_t tx_bytes = static_cast<uint32_t>(G * W_BYTES + n * LIN_BLOCK);
  const int at_once = min(rp.stages, b1 - b0);
  auto load_block = [&](int stage, int b) {
    const int tile = tile0 + first + (b >= cut ? 1 : 0), ft = tile / rp.row_tiles, rt = tile - ft * rp.row_tiles;
    const int k = (b - (first + (b >= cut ? 1 : 0)) * p.kblocks) * per_block;
    uint8_t* base = smem + stage * rp.stage_bytes;
    uint64_t* bar = &full_bar[stage];
    mbar_expect_tx(bar, tx_bytes);
    tma_load_2d(base, &map_w, bar, k, ft * RM);
    if constexpr (GATED) tma_load_2d(base + W_BYTES, &map_up, bar, k, ft * RM);
    tma_load_2d(base + G * W_BYTES, &map_x, bar, k, rt * n);
  };
  if (warp == 0) {
    if (lane < rp.stages) {
      mbar_init(&full_bar[lane], 1);
      mbar_init(&empty_bar[lane], 1);
    } else if (lane >= 28) {
      mbar_init(&acc_full[lane - 28], lane < 30 ? 1 : RESULT_THREADS / 32);  // (acc_full[0, 1], acc_empty[0, 1])
    } else if (lane == 27) {
      *abort_flag = 0;
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async_smem();
    __syncwarp();
    pdl_wait();
    const bool one = elect_one();
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

  // tensor memory: a region for each of the two tiles' sums; behind them (results of F32) two that the instructions add up in
  const uint32_t region = static_cast<uint32_t>(G * n), scratch = static_cast<uint32_t>(rp.group > 1 ? 2 : 1) * region;
  const int quad = warp & 3, half = (warp - 2) >> 2;
  const uint32_t lanes = tmem + (static_cast<uint32_t>(quad * 32) << 16);

  if (warp == 0) {
    const bool one = elect_one();
    int stage = at_once == rp.stages ? 0 : at_once;
    uint32_t phase = at_once == rp.stages ? 1 : 0;
    for (int b = b0 + at_once; b < b1; ++b) {
      if (!mbar_wait_warp(&empty_bar[stage], phase ^ 1, abort_flag, p.err_word, 111)) break;
      if (one) load_block(stage, b);
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
    for (int s = 0; s < segments && ok; ++s) {
      const int to = s ? b1 : cut;
      for (int b = s ? cut : b0; b < to && ok;) {
        uint32_t d = tmem + s * region;
        if constexpr (F32) {
          if (!mbar_wait_warp(&acc_empty[acc], acc_phase ^ 1, abort_flag, p.err_word, 113)) { ok = false; break; }
          tcgen05_fence_after();
          d = tmem + scratch + acc * region;
        }
        const int from = b, end = F32 ? min(to, b + p.chunk) : to;
        for (; b < end; ++b) {
          if (!__all_sync(0xffffffffu, ready) && !mbar_wait_warp(&full_bar[stage], phase, abort_flag, p.err_word, 114)) { ok = false; break; }
          tcgen05_fence_after();
          const uint32_t sa = smem_u32(smem + stage * rp.stage_bytes);
          const uint64_t dw = make_smem_desc(sa, LIN_BLOCK), du = dw + (W_BYTES >> 4), dx = dw + (G * W_BYTES >> 4);
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
        if (one) umma_commit(&acc_full[F32 ? acc : s]);
        __syncwarp();
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
      }
    }
  }

  // ---- results: a lane has a feature, a register a row of x ----
  const bool results = warp >= 2;
  const int size = p.out_type == MIMIR_B200_T_F32 ? 4 : 2, eights = n / 8;
  bool ok = true;
  // A segment's tile: its features and rows, the CTAs that share it, and the eights of its rows that this one finishes
  struct Segment {
    int feature, feature0, row0, from, sharers, me, e0, e1;
    float w_scale, up_scale, bias, up_bias;
  };
  Segment seg[2];
  if (results) {
    // all that the results need besides the sums, while these are made
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (s >= segments) break;
      const int tile = tile0 + first + s, ft = tile / rp.row_tiles, rt = tile - ft * rp.row_tiles;
      Segment& g = seg[s];
      g.feature0 = ft * RM, g.feature = ft * RM + quad * 32 + lane, g.row0 = rt * n;
      g.from = sh.holder((first + s) * p.kblocks);
      g.sharers = sh.holder((first + s + 1) * p.kblocks - 1) - g.from + 1;
      g.me = rank - g.from;
      g.e0 = eights * g.me / g.sharers, g.e1 = eights * (g.me + 1) / g.sharers;
      g.w_scale = g.up_scale = 1.0f, g.bias = g.up_bias = 0.0f;
      if (g.feature < p.n_out) {
        if constexpr (F8) g.w_scale = __ldg(p.w_scale + g.feature);
        if constexpr (F8 && GATED) g.up_scale = __ldg(p.up_scale + g.feature);
        if (p.bias) g.bias = __ldg(p.bias + g.feature);
        if (GATED && p.up_bias) g.up_bias = __ldg(p.up_bias + g.feature);
      }
      if constexpr (F8) {
        const int i = static_cast<int>(threadIdx.x) - 64;
        if (i < n) x_scales[s][i] = g.row0 + i < p.rows ? __ldg(p.x_scale + g.row0 + i) : 0.0f;
      }
      if (!GATED && p.residual && g.feature < p.n_out)  // (into L2)
        for (int i = g.e0 * 8 + half; i < g.e1 * 8 && g.row0 + i < p.rows; i += 2)
          prefetch_line(p.residual + (g.row0 + i) * p.residual_row + static_cast<long long>(g.feature) * size);
    }
    __syncwarp();
  }
  if (results) {
    if constexpr (F32) {
      // sums of a chunk at a time out of tensor memory, added up rounded, and the whole back into the tile's region
      int acc = 0;
      uint32_t acc_phase = 0;
      for (int s = 0; s < segments && ok; ++s) {
        const int to = s ? b1 : cut;
        float v[4][16];  // 16 rows each, of a gated pair first the one, then the other
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 16; ++j) v[i][j] = 0.0f;
        for (int b = s ? cut : b0; b < to; b += p.chunk) {
          ok = mbar_wait_warp(&acc_full[acc], acc_phase, abort_flag, p.err_word, 115);
          if (!ok) break;
          tcgen05_fence_after();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t col = static_cast<uint32_t>((2 * i + half) * 16);
            if (col >= region) continue;
            float w[16];
            tmem_ld_32x16(lanes + scratch + acc * region + col, w);
#pragma unroll
            for (int j = 0; j < 16; ++j) v[i][j] += w[j];
          }
          tcgen05_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&acc_empty[acc]);
          if (++acc == 2) { acc = 0; acc_phase ^= 1; }
        }
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t col = static_cast<uint32_t>((2 * i + half) * 16);
          if (col >= region) continue;
          uint32_t w[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) w[j] = __float_as_uint(v[i][j]);
          tmem_st_32x16(lanes + s * region + col, w);
        }
        tmem_wait_st();
      }
      tcgen05_fence_before();
    } else {
      for (int s = 0; s < segments && ok; ++s) ok = mbar_wait_warp(&acc_full[s], 0, abort_flag, p.err_word, 115);
    }
    // (the rows' scales are there; sums of F32 change hands between a lane's two warps)
    if (F8 || F32) result_warps_sync();
    tcgen05_fence_after();
  }
  if (rp.cluster > 1) {
    __syncwarp();
    cluster_wait();  // every CTA of the cluster has begun
    if (rp.parts_at == 0) {
      __syncthreads();
      cluster_sync_all();  // every ring of the cluster is done with
    }
    if (results && ok) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        if (s >= segments) break;
        const Segment& g = seg[s];
        for (int e = half; e < eights; e += 2) {
          const int who = static_cast<int>(static_cast<unsigned>((e + 1) * g.sharers - 1) / static_cast<unsigned>(eights));  // finishes these rows
          if (who == g.me) continue;
          const int to = g.from + who, r0 = eights * who / g.sharers, wide = eights * (who + 1) / g.sharers - r0;
          // (of the receiver's tiles: its first or its second)
          const int at = rp.parts_at + (first + s - sh.begin(to) / p.kblocks) * rp.part_bytes +
                         ((g.me < who ? g.me : g.me - 1) * G * wide + e - r0) * 8 * RM * 4 + (quad * 32 + lane) * 16;
          const uint32_t dst = mapa_shared(smem_u32(smem + at), static_cast<uint32_t>(to));
          float z[8], u[8];
          tmem_ld_32x8(lanes + s * region + static_cast<uint32_t>(e * 8), z);
          if constexpr (GATED) tmem_ld_32x8(lanes + s * region + static_cast<uint32_t>(n + e * 8), u);
          st_cluster4(dst, z);
          st_cluster4(dst + RM * 16, z + 4);
          if constexpr (GATED) {
            st_cluster4(dst + static_cast<uint32_t>(wide * 8 * RM * 4), u);
            st_cluster4(dst + static_cast<uint32_t>(wide * 8 * RM * 4 + RM * 16), u + 4);
          }
        }
      }
    }
    __syncwarp();
    cluster_sync_all();  // every share has arrived
  }
  if (results) {
    // Eight rows at a time: a lane's sums of its feature, scaled and activated; by way of shared memory to lanes that have eight neighbouring
    // features of a row, for the residual and the result in 16 bytes (two bytes a lane took 0.5 us for eight rows, of 0.9 in all).
    const int fourth = static_cast<int>(threadIdx.x - 64) & 127;  // among the 128 threads that share eight rows
    float* const turns = reinterpret_cast<float*>(smem + rp.turn_at) + half * 2 * 8 * RM;
    const bool go = ok && !*abort_flag;
    int flip = 0;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (s >= segments) break;
      const Segment& g = seg[s];
      const int wide = g.e1 - g.e0;
      const float4* parts = reinterpret_cast<const float4*>(smem + rp.parts_at + s * rp.part_bytes) + quad * 32 + lane;
#pragma unroll 1
      for (int e = g.e0 + ((g.e0 ^ half) & 1); e < g.e1; e += 2, flip ^= 1) {
        const int row0 = g.row0 + e * 8;
        if (row0 >= p.rows) break;
        // the row and features that this thread writes, and their residual on its way
        const int row = row0 + (fourth >> 4), col = g.feature0 + (fourth & 15) * 8;
        const bool there = row < p.rows && col < p.n_out;
        const char* res = p.residual + row * p.residual_row + static_cast<long long>(col) * size;
        char* out = p.out + row * p.out_row + static_cast<long long>(col) * size;
        const bool whole = col + 8 <= p.n_out;
        float q[8];
        if (!GATED && p.residual && there) load_eight(res, p.out_type, whole && p.vec_res, p.n_out - col, q);
        float z[8], u[8];
        tmem_ld_32x8(lanes + s * region + static_cast<uint32_t>(e * 8), z);
        if constexpr (GATED) tmem_ld_32x8(lanes + s * region + static_cast<uint32_t>(n + e * 8), u);
        for (int o = 0; o < g.sharers - 1; ++o) {
          const float4* from = parts + (o * G * wide + e - g.e0) * 2 * RM;
#pragma unroll
          for (int w = 0; w < G; ++w) {
            const float4 a = from[w * wide * 2 * RM], b = from[w * wide * 2 * RM + RM];
            float(&v)[8] = w ? u : z;
            v[0] += a.x, v[1] += a.y, v[2] += a.z, v[3] += a.w, v[4] += b.x, v[5] += b.y, v[6] += b.z, v[7] += b.w;
          }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if constexpr (F8) {
            const float sx = x_scales[s][e * 8 + j];
            z[j] = fmaf(z[j] * sx, g.w_scale, g.bias);
            if constexpr (GATED) u[j] = fmaf(u[j] * sx, g.up_scale, g.up_bias);
          } else {
            z[j] += g.bias;
            if constexpr (GATED) u[j] += g.up_bias;
          }
        }
        activate(z, p.act);
        float* turn = turns + flip * 8 * RM;
#pragma unroll
        for (int j = 0; j < 8; ++j) turn[j * RM + quad * 32 + lane] = GATED ? z[j] * u[j] : z[j];
        four_warps_sync(half);
        if (there && go) {
          const float4 a = *reinterpret_cast<const float4*>(turn + fourth * 8), b = *reinterpret_cast<const float4*>(turn + fourth * 8 + 4);
          float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
          if (!GATED && p.residual) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += q[j];
          }
          store_eight(out, p.out_type, whole && p.vec_out, p.n_out - col, v);
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
  int rows_tile, row_tiles, group, cluster, per_sm, stages, stage_bytes, parts_at, part_bytes, turn_at, tmem_cols;
  size_t smem;
  long long tiles, ctas;
  double cycles;
};

// The shape of a launch with `group` tiles to a cluster of `cluster` CTAs, per_sm of them on an SM; false where it does not fit.
bool shape_of(const MimirLinear& a, bool gated, int group, int cluster, int per_sm, RowShape* s) {
  const int g = gated ? 2 : 1, f32 = a.out_type == MIMIR_B200_T_F32;
  // (two tiles' sums, and of F32 two more regions that they are made in: 512 columns)
  const int most = (f32 ? 128 : 256) / g;
  s->row_tiles = (a.rows + most - 1) / most;
  s->rows_tile = round_up((a.rows + s->row_tiles - 1) / s->row_tiles, 16);
  s->tiles = static_cast<long long>(s->row_tiles) * ((a.n_out + RM - 1) / RM);
  s->group = group, s->cluster = cluster, s->per_sm = per_sm;
  s->ctas = (s->tiles + group - 1) / group * cluster;
  const int kblocks = static_cast<int>((static_cast<long long>(a.n_in) * type_bytes(a.type) + LIN_BLOCK - 1) / LIN_BLOCK);
  if (cluster > 1 && per_sm > 1) return false;
  if (s->ctas > 0x3fffffffLL || (cluster > 1 && kblocks < 2 * cluster)) return false;
  s->tmem_cols = 32;
  while (s->tmem_cols < ((group > 1 ? 2 : 1) + (f32 ? 2 : 0)) * g * s->rows_tile) s->tmem_cols *= 2;
  if (s->tmem_cols > 512 / per_sm) return false;
  // what a CTA gets from others for one tile: the most over the tiles of a cluster, the last cluster's with fewer of them too
  s->part_bytes = 0;
  for (int tiles = group; tiles >= 1; --tiles) {
    const Shares sh = {kblocks, tiles * kblocks, cluster};
    for (int t = 0; t < tiles; ++t) {
      const int sharers = sh.holder((t + 1) * kblocks - 1) - sh.holder(t * kblocks) + 1, eights = s->rows_tile / 8;
      const int bytes = (sharers - 1) * ((eights + sharers - 1) / sharers) * 8 * g * RM * 4;
      if (bytes > s->part_bytes) s->part_bytes = bytes;
    }
  }
  const int parts = s->part_bytes * (group > 1 ? 2 : 1), space = (per_sm == 2 ? DYNAMIC_TWO : DYNAMIC) - 1024;
  s->stage_bytes = g * W_BYTES + s->rows_tile * LIN_BLOCK;
  const int need = (group * kblocks + cluster - 1) / cluster;  // stages that a CTA can fill at all
  auto stages_in = [&](int bytes) { return bytes < 0 ? 0 : std::min(std::min(bytes / s->stage_bytes, MAX_STAGES), need); };
  s->stages = stages_in(space - parts);
  s->parts_at = s->stages * s->stage_bytes;
  if (parts == 0 || (s->stages < need && s->stages * s->stage_bytes < 96 * 1024)) {  // too little of a ring: the shares come into it afterwards
    s->stages = stages_in(space);
    s->parts_at = 0;
  }
  if (s->stages < 2 && s->stages < need) return false;
  s->turn_at = s->parts_at ? 0 : parts;
  if (s->turn_at + TURNS > space) return false;
  s->smem = static_cast<size_t>(std::max(s->stages * s->stage_bytes + (s->parts_at ? parts : 0), s->turn_at + TURNS)) + 1024;
  if (cluster > 1) s->smem = std::max(s->smem, ALONE);
  return true;
}

// Stands for the kernel where the runtime is asked how many clusters run at the same time (of kernels that allocate tensor memory it counts one CTA
// to an SM).  A cluster lives in one GPC, whose SM count is no multiple of it.
__global__ void __launch_bounds__(THREADS, 2) rows_footprint_kernel() {}
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
      cfg.blockDim = dim3(THREADS);
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

RowShape row_shape(const MimirLinear& a, bool gated) {
  RowShape best = {};
  best.cycles = 1e30;
  const ClusterTable* active = active_clusters();
  if (!active) return best;
  for (int cluster = 1; cluster <= MAX_CLUSTER; ++cluster)
    for (int group = 1; group <= cluster; ++group)
      for (int per_sm = 1; per_sm <= 2; ++per_sm) {
        RowShape s;
        if ((group == cluster && cluster > 1) || !shape_of(a, gated, group, cluster, per_sm, &s)) continue;
        const double blocks = (static_cast<double>(a.n_in) * type_bytes(a.type) + LIN_BLOCK - 1) / LIN_BLOCK * group / cluster;
        const long long at_once = static_cast<long long>(active->n[cluster]) * cluster;
        if (at_once <= 0) continue;
        const double rounds = static_cast<double>((s.ctas + at_once - 1) / at_once);
        const double fill = std::max(s.stage_bytes / 31.0, (gated ? 2 : 1) * 4 * std::max(32.0, s.rows_tile / 2.0));
        s.cycles = rounds * blocks * fill + 4000.0 + (cluster > 1 ? 3000.0 + (s.parts_at ? 0 : 1000.0) : 0.0);
        if (s.cycles < best.cycles) best = s;
      }
  return best;
}

template <bool F8, bool GATED, bool F32>
int launch_as(const CUtensorMap (&maps)[3], const RowParams& p, const RowShape& s, cudaStream_t st) {
  auto kern = linear_rows_kernel<F8, GATED, F32>;
  static PerDeviceOnce once;
  MB_TRY(once.run([&]() -> int {
    MB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, DYNAMIC));
    return MIMIR_B200_OK;
  }));
  MB_TRY(launch_pdl(kern, dim3(static_cast<unsigned>(s.ctas)), dim3(THREADS), s.smem, st, s.cluster, maps[0], maps[1], maps[2], p));
  count_launch();
  return MIMIR_B200_OK;
}

}  // namespace

double linear_rows_cycles(const MimirLinear& a, bool gated) { return a.rows > 4096 ? 1e30 : row_shape(a, gated).cycles; }

int launch_linear_rows(const MimirLinear& a, const LinearParams& l, bool gated, cudaStream_t st) {
  const RowShape s = row_shape(a, gated);
  CUtensorMap maps[3];
  MB_TRY(make_operand_map(&maps[0], a.x, a.type, a.rows, a.n_in, a.x_stride, s.rows_tile));
  MB_TRY(make_operand_map(&maps[1], a.w, a.type, a.n_out, a.n_in, a.w_stride, RM));
  maps[2] = maps[1];
  if (gated) MB_TRY(make_operand_map(&maps[2], a.up, a.type, a.n_out, a.n_in, a.up_stride, RM));
  RowParams p = {};
  p.l = l, p.rows_tile = s.rows_tile, p.row_tiles = s.row_tiles, p.tiles = static_cast<int>(s.tiles), p.group = s.group, p.cluster = s.cluster;
  p.stages = s.stages, p.stage_bytes = s.stage_bytes, p.parts_at = s.parts_at, p.part_bytes = s.part_bytes, p.turn_at = s.turn_at, p.tmem_cols = s.tmem_cols;
  p.early = pdl_small_grid(static_cast<unsigned>(s.ctas));
  const bool f32 = a.out_type == MIMIR_B200_T_F32;
  if (a.type == MIMIR_B200_T_E4M3)
    return gated ? (f32 ? launch_as<true, true, true>(maps, p, s, st) : launch_as<true, true, false>(maps, p, s, st))
                 : (f32 ? launch_as<true, false, true>(maps, p, s, st) : launch_as<true, false, false>(maps, p, s, st));
  return gated ? (f32 ? launch_as<false, true, true>(maps, p, s, st) : launch_as<false, true, false>(maps, p, s, st))
               : (f32 ? launch_as<false, false, true>(maps, p, s, st) : launch_as<false, false, false>(maps, p, s, st));
}

}  // namespace mb
