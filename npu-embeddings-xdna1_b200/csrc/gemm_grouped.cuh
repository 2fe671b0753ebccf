// One matrix product per expert over ragged groups of rows, on the sm_100a
// tensor cores:
//
//   C[p] = act(A[src(p)] . W[e] + bias[e])   for p in [off[e], off[e + 1])
//
// off comes from device memory, so a pass needs no host round trip.  src(p)
// is row_src[p] (the routed row, gathered on the way into shared memory) or p.
// W is [experts, N, K] bf16, one matrix over all experts to the tensor map;
// a gated weight's N columns are interleaved in groups of 64 = [32 up |
// 32 gate] and the product is up * act(gate), N / 2 wide.
//
// Tiles are 128 x BN of one expert; a list of tile counts per expert, built
// by every block from off, gives a tile its expert.  The roles, the shared
// memory ring, the double-buffered accumulator and the bounded waits are
// gemm_tc_kernel's.  A's rows come by a tiled TMA load where they are grouped
// already (rows past the group are the next group's and are not stored), or
// by 32 four-row gathers, one from each lane of the producer warp, the lane
// keeping its four row indices in registers for the whole tile.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cstdint>

#include "gemm_tc.cuh"
#include "ptx.cuh"

namespace nebw {

constexpr int kGroupMaxExperts = 512;

enum GroupEpi : int {
  kGrpBf16 = 0,
  kGrpBf16Gelu8 = 1,
  kGrpBf16Erf = 2,
  kGrpF32 = 3,
  kGrpBf16SwiGLU = 4,
  kGrpBf16GeGLU = 5,
};
__host__ __device__ constexpr bool grp_gated(int e) { return e >= kGrpBf16SwiGLU; }

struct GroupedArgs {
  const int *off;      // [experts + 1]
  int experts;
  int rows;            // C's rows: the bound of off
  const int *row_src;  // [rows] or null
  int a_rows;          // A's rows
  int N, K;            // N as staged (2F for a gated weight)
  const float *bias;   // [experts, N] in the container's column order, or null
  void *out;           // [rows, N or N / 2]
  int *err;
};

// Four rows of a K-major map (box 64 x 1) into 512 consecutive bytes of a
// 128-byte-swizzled tile.
__device__ __forceinline__ void tma_gather4(void *smem_dst, const void *tmap, uint64_t *bar,
                                            int32_t c0, const int (&r)[4]) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(c0), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
      "r"(smem_u32(bar))
      : "memory");
}

// The groups in shared memory: off clamped to [0, rows] and ascending (a
// fault is reported), and the first tile of every expert.
struct GroupTable {
  int off[kGroupMaxExperts + 1];
  int tile[kGroupMaxExperts + 1];
};

__device__ __forceinline__ void group_table_build(GroupTable &g, const GroupedArgs &p, int bm,
                                                  int n_blocks) {
  for (int e = threadIdx.x; e <= p.experts; e += blockDim.x) g.off[e] = __ldg(p.off + e);
  __syncthreads();
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int hi = 0, tiles = 0;  // the running maximum of off, and the tiles so far
    bool bad = false;
    for (int e0 = 0; e0 <= p.experts; e0 += 32) {
      const int e = e0 + lane;
      const int raw = e <= p.experts ? g.off[e] : 0;
      int v = min(max(raw, 0), p.rows);
      bad |= e <= p.experts && raw != v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v = max(v, u);
      }
      v = max(v, hi);
      bad |= e <= p.experts && v > raw;
      // expert e - 1 is [off[e - 1], off[e]): its tiles end at tile[e]
      int before = __shfl_up_sync(0xffffffffu, v, 1);
      if (lane == 0) before = e0 ? hi : v;
      int t = (v - before + bm - 1) / bm * n_blocks;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, t, o);
        if (lane >= o) t += u;
      }
      t += tiles;
      if (e <= p.experts) {
        g.off[e] = v;
        g.tile[e] = t;
      }
      hi = __shfl_sync(0xffffffffu, v, 31);
      tiles = __shfl_sync(0xffffffffu, t, 31);
    }
    if (bad && blockIdx.x == 0) record_err(p.err, kDevBadGroup);
  }
  __syncthreads();
}

// A tile of the list: expert, its rows [row, end) and the column block.
struct GroupTile {
  int e, row, end, nb;
};

// The tile `t`, walking on from expert `e` (t does not decrease from call to call).
__device__ __forceinline__ GroupTile group_tile(const GroupTable &g, int t, int bm, int n_blocks,
                                                int &e) {
  while (t >= g.tile[e + 1]) ++e;
  const int i = t - g.tile[e];
  const int mb = i / n_blocks;
  return {e, g.off[e] + mb * bm, g.off[e + 1], i - mb * n_blocks};
}

// 32 accumulator columns [col0, col0 + 32) of one row, biased, activated and
// stored; a gated epilogue's come with the 32 columns of their gate.
template <int EPI>
__device__ __forceinline__ void grp_store32(const GroupedArgs &p, int e, int64_t row, int col0,
                                            const uint32_t (&r)[32], const uint32_t (&rg)[32]) {
  constexpr bool kGated = grp_gated(EPI);
  const int width = kGated ? p.N / 2 : p.N;
  const int c0 = kGated ? col0 / 2 : col0;  // col0 % 64 == 0 there
  const int ncols = min(32, width - c0);    // width % 8 == 0
  float v[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
  const float *bias = p.bias ? p.bias + static_cast<int64_t>(e) * p.N + c0 : nullptr;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    if (i < ncols) {
      if (bias) v[i] += __ldg(bias + i);
      if constexpr (kGated) {
        float g = __uint_as_float(rg[i]);
        if (bias) g += __ldg(bias + width + i);
        v[i] *= EPI == kGrpBf16SwiGLU ? silu_fast(g) : gelu_erf(g);
      } else if constexpr (EPI == kGrpBf16Gelu8) {
        v[i] = gelu8(v[i]);
      } else if constexpr (EPI == kGrpBf16Erf) {
        v[i] = gelu_erf(v[i]);
      }
    }
  }
  if constexpr (EPI == kGrpF32) {
    float4 *o = reinterpret_cast<float4 *>(static_cast<float *>(p.out) + row * width + c0);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i * 4 < ncols) o[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  } else {
    uint4 *o = reinterpret_cast<uint4 *>(static_cast<__nv_bfloat16 *>(p.out) + row * width + c0);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i * 8 < ncols)
        o[i] = make_uint4(pack_bf16x2(v[8 * i], v[8 * i + 1]),
                          pack_bf16x2(v[8 * i + 2], v[8 * i + 3]),
                          pack_bf16x2(v[8 * i + 4], v[8 * i + 5]),
                          pack_bf16x2(v[8 * i + 6], v[8 * i + 7]));
  }
}

template <int BN>
struct GroupedShape {
  using S = GemmShape<BN>;
  static constexpr int kSmemBytes = S::kSmemBytes + static_cast<int>(sizeof(GroupTable));
};

template <int BN, int EPI, bool GATHER>
__global__ void __launch_bounds__(kGemmThreads, 1)
    gemm_grouped_kernel(const __grid_constant__ CUtensorMap tmA,
                        const __grid_constant__ CUtensorMap tmW, const GroupedArgs p) {
  using S = GemmShape<BN>;
  constexpr int kStages = S::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t *sA = smem;
  uint8_t *sW = smem + kStages * S::kABytes;
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + kStages * S::kStageBytes);
  uint64_t *empty = full + kStages;
  uint64_t *tfull = empty + kStages;
  uint64_t *tempty = tfull + 2;
  uint64_t *drain = tempty + 2;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
  GroupTable &table = *reinterpret_cast<GroupTable *>(smem + kStages * S::kStageBytes + S::kBarBytes);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int n_blocks = (p.N + BN - 1) / BN;
  const int num_kb = (p.K + kGemmBK - 1) / kGemmBK;

  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmW);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 8);
    }
    mbar_init(drain, 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, S::kTmemCols);
    tmem_relinquish();
  }
  group_table_build(table, p, kGemmBM, n_blocks);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int num_tiles = table.tile[p.experts];
  auto wait_all = [&](uint64_t *bar, uint32_t parity) -> bool {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, p.err));
  };

  if (warp == 0) {
    // ---------------- TMA producer (the whole warp walks the schedule) -----
    int stage = 0, e = 0;
    uint32_t phase = 0;
    uint32_t issued_mask = 0, last_phase = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x) {
      const GroupTile t = group_tile(table, tile, kGemmBM, n_blocks, e);
      int src[4];
      if constexpr (GATHER) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // past the group: its last row again, not stored
          int r = __ldg(p.row_src + min(t.row + 4 * lane + i, t.end - 1));
          if (r < 0 || r >= p.a_rows) {
            record_err(p.err, kDevBadGroup);
            r = 0;
          }
          src[i] = r;
        }
      }
      for (int kb = 0; kb < num_kb; ++kb) {
        if (!wait_all(&empty[stage], phase ^ 1u)) {
          ok = false;
          break;
        }
        if (lane == 0) {
          mbar_arrive_expect_tx(&full[stage], S::kStageBytes);
          tma_load_2d(sW + stage * S::kBBytes, &tmW, &full[stage], kb * kGemmBK,
                      t.e * p.N + t.nb * BN);
          if constexpr (!GATHER)
            tma_load_2d(sA + stage * S::kABytes, &tmA, &full[stage], kb * kGemmBK, t.row);
        }
        __syncwarp();
        if constexpr (GATHER)
          tma_gather4(sA + stage * S::kABytes + lane * 512, &tmA, &full[stage], kb * kGemmBK, src);
        issued_mask |= 1u << stage;
        last_phase = (last_phase & ~(1u << stage)) | (phase << stage);
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    // Drain: every stage this warp loaded has landed before the CTA exits.
    for (int s = 0; s < kStages; ++s)
      if (issued_mask & (1u << s)) wait_all(&full[s], (last_phase >> s) & 1u);
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    constexpr uint32_t idesc = idesc_bf16_f32(kGemmBM, BN);
    const bool elect = elect_one_sync();
    int stage = 0;
    uint32_t phase = 0;
    bool issued_any = false, ok = true;
    int local = 0;
    for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x, ++local) {
      const int acc = local & 1;
      if (!wait_all(&tempty[acc], ((local >> 1) & 1) ^ 1u)) break;
      tc_fence_after();
      const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * BN);
      for (int kb = 0; kb < num_kb; ++kb) {
        if (!wait_all(&full[stage], phase)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint64_t da = sdesc_kmajor_sw128(smem_u32(sA + stage * S::kABytes));
        const uint64_t dw = sdesc_kmajor_sw128(smem_u32(sW + stage * S::kBBytes));
        if (elect) {
#pragma unroll
          for (int k = 0; k < kGemmBK / 16; ++k)
            umma_bf16(d_tmem, da + k * 2, dw + k * 2, idesc, (kb | k) != 0 ? 1u : 0u);
          umma_commit(&empty[stage]);
        }
        __syncwarp();
        issued_any = true;
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (ok && elect) umma_commit(&tfull[acc]);
      __syncwarp();
    }
    if (issued_any) {
      if (elect) umma_commit(drain);
      __syncwarp();
      wait_all(drain, 0);
    }
  } else {
    // ---------------- epilogue (warps 2..9) ----------------
    constexpr int kHalf = BN / 2;
    constexpr int kChunks = kHalf / 32;
    const int quarter = warp & 3;
    const int col_half = ((warp - 2) >> 2) * kHalf;
    int local = 0, e = 0;
    for (int tile = blockIdx.x; tile < num_tiles; tile += gridDim.x, ++local) {
      const int acc = local & 1;
      if (!wait_all(&tfull[acc], (local >> 1) & 1)) break;
      tc_fence_after();
      const GroupTile t = group_tile(table, tile, kGemmBM, n_blocks, e);
      const int row = t.row + quarter * 32 + lane;
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) +
                             static_cast<uint32_t>(acc * BN + col_half);
      constexpr int kStep = grp_gated(EPI) ? 2 : 1;
#pragma unroll
      for (int c = 0; c < kChunks; c += kStep) {
        uint32_t r[32], rg[32];
        tmem_ld_32x32b_x32(t_row + c * 32, r);
        if constexpr (kStep == 2) tmem_ld_32x32b_x32(t_row + (c + 1) * 32, rg);
        tmem_wait_ld_regs(r);
        if constexpr (kStep == 2) tmem_wait_ld_regs(rg);
        if (c + kStep == kChunks) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&tempty[acc]);
        }
        const int col0 = t.nb * BN + col_half + c * 32;
        if (row < t.end && col0 < p.N) grp_store32<EPI>(p, t.e, row, col0, r, rg);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, S::kTmemCols);
  }
}

// Expert weights [experts, K, N] (fp32 or bf16) to bf16 [experts, N, K], RNE;
// for a gated weight row n of the result takes column glu(n) of [up | gate].
__global__ void stage_experts_kernel(const void *__restrict__ src, int src_bf16, int K, int N,
                                     int gated, int e0, __nv_bfloat16 *__restrict__ dst) {
  __shared__ float tile[32][33];
  const int64_t e = blockIdx.z;
  const int k0 = blockIdx.y * 32, n0 = blockIdx.x * 32;
  // 32 rows of the result are 32 consecutive columns of the source either way
  int c0 = n0;
  if (gated) c0 = (n0 / 64) * 32 + (n0 % 64 ? N / 2 : 0);
  for (int i = threadIdx.y; i < 32; i += blockDim.y) {
    const int k = k0 + i, c = c0 + threadIdx.x;
    float v = 0.f;
    if (k < K && n0 + static_cast<int>(threadIdx.x) < N) {
      const int64_t at = (e * K + k) * N + c;
      v = src_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(src)[at])
                   : static_cast<const float *>(src)[at];
    }
    tile[i][threadIdx.x] = v;
  }
  __syncthreads();
  for (int i = threadIdx.y; i < 32; i += blockDim.y) {
    const int n = n0 + i, k = k0 + threadIdx.x;
    if (n < N && k < K)
      dst[((e0 + e) * N + n) * K + k] = __float2bfloat16_rn(tile[threadIdx.x][i]);
  }
}

}  // namespace nebw
