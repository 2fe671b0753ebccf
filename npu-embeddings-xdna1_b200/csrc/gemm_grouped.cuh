// One matrix product per expert over ragged groups of rows, on the sm_100a
// tensor cores:
//
//   C[p] = act(A[src(p)] . W[e] + bias[e])   for p in [off[e], off[e + 1])
//
// off comes from device memory, so a pass needs no host round trip.  src(p)
// is row_src[p] (the routed row, gathered on the way into shared memory) or p.
// W is staged in blocks of 128 columns by 64 of K (stage_experts_kernel); a
// gated weight's N columns are interleaved in groups of 64 = [32 up | 32 gate]
// and the product is up * act(gate), N / 2 wide.
//
// A CTA pair (tcgen05 cta_group::2) takes 256 columns of W and up to 256 rows
// of one group, with W as the product's M operand and the rows as its N
// operand, a multiple of 32, so that a part tile loads and finishes only the
// rows it has; the accumulator holds a column of C per TMEM lane.  The
// persistent pairs walk one list of tiles, whatever the groups are: every
// block builds it from off.
//
// Measured, replayed from a graph: 373 us for 65,542 grouped rows, K 4096, N
// 1024, 8 experts (1473 TFLOP/s, 0.89 of the measured cuBLAS burst); 830 us
// gathered, K 1024, gated N 8192 (1326 TFLOP/s; 717 us without the gather);
// 42.5 us for 16,088 rows of 64 experts, K 1024, gated N 1024; 14.0 us for 28
// rows of 8, K 768, N 3840.  In a loop of calls, where the power cap lowers the
// clock: 372 to 457 us (1200 TFLOP/s), 830 to 957 (1150), 45 to 53, 16.4.
// What bounds it: the tensor pipe for whole tiles, HBM for few rows a group,
// and between them that W streams through the M side at 128 columns in 128
// clocks a step of 16, however few the rows are (0.26 us a K-block for one
// pair and 8 rows, 60 GB/s an SM: more than HBM gives from about 110 SMs on,
// the bound of a product with fewer column tiles than that).  One CTA on 128
// rows by 128, 64 or 32 columns, rows as M, was no faster at any size tried:
// 8.2 / 9.0 / 12.8 us for the pair against 8.2 / 8.9 / 14.1 us at best on 1,
// 32 and 1024 rows of 2 of 8 experts, K and N 1024; 15.0 against 15.4 us on
// 64 rows, K 768, N 3840.  Prefetching W into L2 8 to 32 K-blocks ahead was
// slower throughout (53 against 51 us on 2011 rows of 64 experts, 16).
//
// Roles of a block:
//   warp 0        W by TMA (and A, where its rows are grouped already), and
//                 the stage's transaction bytes
//   warp 1        tcgen05.mma (the leader)
//   warps 2-9     epilogue: TMEM -> bias, activation -> shared memory -> TMA
//                 store of 32 x 32 chunks; the chunk in which a group ends is
//                 stored row by row
//   warps 10-17   GATHER: A's rows, four at a time (tile::gather4), each warp
//                 a share of the tile's rows with their indices in registers
// A gather is issued by one lane for uniform operands; from 32 lanes of one
// warp the same 32 gathers take turns on the issue path (80 clocks each).
// Eight warps: 850 us on 65,542 rows, K 1024, N 8192, against 893 for four and
// 962 for sixteen, whose registers the epilogue then lacks (717 us for rows
// that are grouped already).  Rows past the group are not loaded: what lies in their
// place in shared memory reaches only accumulators that are not stored.  All
// waits are bounded as in gemm_tc_pair_kernel, whose barriers these are.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cstdint>
#include <type_traits>

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
  int tile_rows;       // most rows of a tile: 256 or 128
  const float *bias;   // [experts, N] in the container's column order, or null
  void *out;           // [rows, N or N / 2]
  int *err;
};

// Shared memory of a CTA: a ring of stages of 128 rows of W and half a tile's
// rows of A, each 64 wide.  The fewer rows a tile may have (the launch's
// choice), the deeper the ring.
struct GroupedShape {
  static constexpr int kWBytes = 128 * kGemmBK * 2;
  static constexpr int kRingBytes = 168 * 1024;
  static constexpr int kMaxStages = 8;
  __host__ __device__ static constexpr int stages(int tile_rows) {
    const int n = kRingBytes / (kWBytes + tile_rows / 2 * kGemmBK * 2);
    return n < kMaxStages ? n : kMaxStages;
  }
  static constexpr int kWarpStaging = 6 * 1024;  // one fp32 or three bf16 chunks
  static constexpr int kStagingBytes = 8 * kWarpStaging;
  static constexpr int kBarBytes = 256;
  static constexpr int kList = 128;  // tiles of a block looked up beforehand
  static constexpr int kTableBytes = kList * 16 + 2 * (kGroupMaxExperts + 1) * 4 + 8;
  static constexpr int kSmemBytes =
      1024 + kRingBytes + kStagingBytes + kBarBytes + kTableBytes;
};
constexpr int kGroupedBox = 32;  // rows of the TMA boxes that end a group of A
constexpr int kGroupedThreads = 320;
constexpr int kGatherWarps = 8;
constexpr int kGatherRows = kGemmBM / kGatherWarps;
constexpr int kGroupedGatherThreads = 320 + 32 * kGatherWarps;

// Arrive on a barrier of this cluster without ordering any memory access of
// this thread before it.
__device__ __forceinline__ void grp_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar)
               : "memory");
}

// Four rows of a K-major map (box 64 x 1) into 512 consecutive bytes of a
// 128-byte-swizzled tile, completing on the barrier at `bar` (a
// shared::cluster address: the leader's).
__device__ __forceinline__ void grp_gather4(uint32_t dst, const void *tmap, uint32_t bar,
                                            int32_t c0, int32_t r0, int32_t r1, int32_t r2,
                                            int32_t r3) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes"
      ".cta_group::2 [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(c0), "r"(r0), "r"(r1), "r"(r2), "r"(r3), "r"(bar)
      : "memory");
}

// A tile of the list: expert, its rows [row, end) and the column block.
struct alignas(16) GroupTile {
  int e, row, end, nb;
};

// The groups in shared memory: off clamped to [0, rows] and ascending (a
// fault is reported), the first tile of every expert, and this block's first
// tiles.
struct GroupTable {
  GroupTile list[GroupedShape::kList];
  int off[kGroupMaxExperts + 1];
  int tile[kGroupMaxExperts + 1];
};
static_assert(sizeof(GroupTable) == GroupedShape::kTableBytes, "table size");

constexpr int kGroupTileCols = 256;

// Tile t: a group of m rows is cut into ceil(m / tile_rows) tiles of equal
// size, rounded up to 32 rows.
__device__ __forceinline__ GroupTile group_find(const GroupTable &g, const GroupedArgs &p, int t,
                                                int n_blocks) {
  int lo = 0, hi = p.experts;  // tile[lo] <= t < tile[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t >= g.tile[mid]) lo = mid;
    else hi = mid;
  }
  const int i = t - g.tile[lo], b = i / n_blocks;
  const int m = g.off[lo + 1] - g.off[lo];
  const int tiles = (m + p.tile_rows - 1) / p.tile_rows;
  const int size = ((m + tiles - 1) / tiles + 31) / 32 * 32;
  const int row = g.off[lo] + b * size;
  return {lo, row, min(row + size, g.off[lo + 1]), i - b * n_blocks};
}

// off and tile, by one warp: four consecutive experts a lane, 128 a round.
__device__ __forceinline__ void group_table_build(GroupTable &g, const GroupedArgs &p,
                                                  int n_blocks, int lane) {
  int top = 0, tiles = 0;  // off's running maximum, and the tiles so far
  bool bad = false;
  for (int e0 = 0; e0 <= p.experts; e0 += 128) {
    const int e = e0 + 4 * lane;
    int v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = e + i <= p.experts ? __ldg(p.off + e + i) : 0;
    // ascending and within [0, rows]: what is not is reported and clamped
    int most = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = max(min(max(v[i], 0), p.rows), most);
      bad |= e + i <= p.experts && c != v[i];
      most = v[i] = c;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int w = __shfl_up_sync(0xffffffffu, most, o);
      if (lane >= o) most = max(most, w);
    }
    int before = __shfl_up_sync(0xffffffffu, most, 1);
    before = lane ? max(before, top) : top;
    // expert e - 1 is [off[e - 1], off[e]): its tiles end at tile[e]
    int t[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      bad |= e + i <= p.experts && v[i] < before;
      v[i] = max(v[i], before);
      if (e + i > 0) sum += (v[i] - before + p.tile_rows - 1) / p.tile_rows * n_blocks;
      t[i] = sum;
      before = v[i];
    }
    int all = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int w = __shfl_up_sync(0xffffffffu, all, o);
      if (lane >= o) all += w;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (e + i <= p.experts) {
        g.off[e + i] = v[i];
        g.tile[e + i] = tiles + all - sum + t[i];
      }
    }
    top = max(top, __shfl_sync(0xffffffffu, most, 31));
    tiles += __shfl_sync(0xffffffffu, all, 31);
  }
  if (bad && blockIdx.x == 0) record_err(p.err, kDevBadGroup);
}

// This block's tile number `local`, tile t.
__device__ __forceinline__ GroupTile group_tile(const GroupTable &g, const GroupedArgs &p,
                                                int local, int t, int n_blocks) {
  return local < GroupedShape::kList ? g.list[local] : group_find(g, p, t, n_blocks);
}

// Both warps of an epilogue pair: wait, and whether `ok` held for both (each
// arrives however its own wait ended, so neither is left behind).
__device__ __forceinline__ bool grp_pair_and(int id, bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %2, 0;\n\t"
      "barrier.cta.red.and.pred q, %1, 64, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(static_cast<uint32_t>(ok))
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void grp_pair_sync(int id) {
  asm volatile("barrier.cta.sync %0, 64;" ::"r"(id) : "memory");
}

// A 32 x 32 chunk of the accumulator, 32 lanes of the warp's quarter by 32
// columns, as mma fragments (tcgen05.ld 16x256b): of lanes 8 q .. 8 q + 7 and
// columns 8 c .. 8 c + 7, thread T holds lane T / 4, columns 2 (T % 4) and + 1,
// in r[16 (q / 2) + 4 c + 2 (q % 2)] and the one after.
__device__ __forceinline__ void grp_load_chunk(uint32_t taddr, uint32_t (&r)[32]) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[16 * h]), "=r"(r[16 * h + 1]), "=r"(r[16 * h + 2]), "=r"(r[16 * h + 3]),
          "=r"(r[16 * h + 4]), "=r"(r[16 * h + 5]), "=r"(r[16 * h + 6]), "=r"(r[16 * h + 7]),
          "=r"(r[16 * h + 8]), "=r"(r[16 * h + 9]), "=r"(r[16 * h + 10]), "=r"(r[16 * h + 11]),
          "=r"(r[16 * h + 12]), "=r"(r[16 * h + 13]), "=r"(r[16 * h + 14]), "=r"(r[16 * h + 15])
        : "r"(taddr + (static_cast<uint32_t>(16 * h) << 16))
        : "memory");
  tmem_wait_ld_regs(r);
}

// x / (1 + 2^(-x log2 e)) on two values: 2^x and 1 / x on the SFU (relative
// errors of 2^-22 and 2^-23), far below the rounding of the product to bf16.
__device__ __forceinline__ void grp_silu_x2(float &a, float &b) {
  float t0, t1;
  unpk2(mul_x2(pk2(a, b), pk2(-1.4426950408889634f, -1.4426950408889634f)), t0, t1);
  unpk2(add_x2(pk2(ex2_approx(t0), ex2_approx(t1)), pk2(1.0f, 1.0f)), t0, t1);
  unpk2(mul_x2(pk2(a, b), pk2(rcp_approx(t0), rcp_approx(t1))), a, b);
}

// The biases of this thread's columns of a chunk (0 where there are none).
__device__ __forceinline__ void grp_bias4(const float *bias, int c, int width, float (&b)[4]) {
#pragma unroll
  for (int q = 0; q < 4; ++q) b[q] = bias && c + 8 * q < width ? __ldg(bias + c + 8 * q) : 0.f;
}

// The chunk as rows of C in shared memory, in the output map's swizzle
// (make_tmap_out): bf16 by stmatrix.trans, four 8 x 8 blocks an instruction
// (the four column blocks of eight rows: each lane names a 16-byte piece, and
// the pieces of a block lie in different banks); fp32 value by value.
__device__ __forceinline__ void grp_stage_t(const float (&v)[32], uint8_t *chunk, int lane) {
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const int c = (lane >> 2) + 8 * (2 * (i / 16) + (i % 4) / 2);
    const int row = 8 * (i / 4 % 4) + 2 * (lane & 3) + i % 2;
    *reinterpret_cast<float *>(chunk + row * 128 + (((c >> 2) ^ (row & 7)) << 4) + (c & 3) * 4) =
        v[i];
  }
}
// m[i]: entries 2 i and 2 i + 1 of the chunk as bf16.
__device__ __forceinline__ void grp_stage_t(const uint32_t (&m)[16], uint8_t *chunk, int lane) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // rows 8 i .. 8 i + 7
    const int row = 8 * i + (lane & 7), q = lane >> 3;
    const uint32_t at = smem_u32(chunk + row * 64 + ((q ^ ((row >> 1) & 3)) << 4));
    asm volatile(
        "stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(at),
        "r"(m[2 * i]), "r"(m[2 * i + 1]), "r"(m[8 + 2 * i]), "r"(m[8 + 2 * i + 1])
        : "memory");
  }
}

// The staged rows [row0, end) of a chunk in which a group ends, by 16-byte
// pieces (the width is a multiple of 8 elements).
template <int EPI>
__device__ __forceinline__ void grp_store_rows(void *out, const uint8_t *chunk, int row0, int end,
                                               int c0, int width, int lane) {
  constexpr int kPieces = EPI == kGrpF32 ? 8 : 4, kRows = 32 / kPieces;
  constexpr int kSize = EPI == kGrpF32 ? 4 : 2, kPer = 16 / kSize;
  const int piece = lane % kPieces;
  if (c0 + piece * kPer >= width) return;
  for (int i = lane / kPieces; i < 32 && row0 + i < end; i += kRows) {
    const int sw = EPI == kGrpF32 ? i & 7 : (i >> 1) & 3;
    const uint4 u = *reinterpret_cast<const uint4 *>(chunk + i * (kPieces * 16) +
                                                     ((piece ^ sw) << 4));
    *reinterpret_cast<uint4 *>(
        static_cast<uint8_t *>(out) +
        (static_cast<int64_t>(row0 + i) * width + c0 + piece * kPer) * kSize) = u;
  }
}

template <int EPI, bool GATHER>
__global__ void __cluster_dims__(2, 1, 1)
    __launch_bounds__(GATHER ? kGroupedGatherThreads : kGroupedThreads, 1)
    gemm_grouped_kernel(const __grid_constant__ CUtensorMap tmA,
                        const __grid_constant__ CUtensorMap tmA128,
                        const __grid_constant__ CUtensorMap tmW,
                        const __grid_constant__ CUtensorMap tmC, const GroupedArgs p) {
  using S = GroupedShape;
  const int stages = S::stages(p.tile_rows);
  const int a_bytes = p.tile_rows / 2 * kGemmBK * 2;
  constexpr int kAccCols = 256;  // TMEM columns of an accumulator: the tile's rows
  // bf16 output: two accumulators, the epilogue of one tile under the products
  // of the next.  fp32 output shows what the tensor core cuts off as it adds up
  // (towards zero, once a step of 16): all of TMEM goes to one tile, K in as
  // many parts as fit (two of 256 rows, four of 128), which the epilogue adds.
  // Error against 64 bits at K 1024 / 2048: one part 1.0e-6 / 2.1e-6, two
  // 4.7e-7 / 1.0e-6, four - / 4.7e-7 (fp32 sums in torch: 2.5e-7 / 3.9e-7).
  constexpr int kBuffers = EPI == kGrpF32 ? 1 : 2;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t *sW = smem;
  uint8_t *sA = smem + stages * S::kWBytes;
  uint8_t *staging = smem + S::kRingBytes;
  uint64_t *full = reinterpret_cast<uint64_t *>(staging + S::kStagingBytes);
  uint64_t *empty = full + S::kMaxStages;
  uint64_t *tfull = empty + S::kMaxStages;
  uint64_t *tempty = tfull + 2;
  uint64_t *drain = tempty + 2;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
  GroupTable &table =
      *reinterpret_cast<GroupTable *>(staging + S::kStagingBytes + S::kBarBytes);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const bool leader = rank == 0;
  const int n_blocks = (p.N + 255) / 256;
  const int num_kb = (p.K + kGemmBK - 1) / kGemmBK;
  const int parts_fit = 512 / p.tile_rows;  // of K, fp32 output
  const int part_kb = (num_kb + parts_fit - 1) / parts_fit;
  const int parts = (num_kb + part_kb - 1) / part_kb;
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1;

  if (warp == 0) {
    group_table_build(table, p, n_blocks, lane);
  } else if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 2 * kAccCols);
    tmem_relinquish_pair();
  } else if (warp == 2 && lane == 0) {
    for (int s = 0; s < stages; ++s) {
      // every gather warp arrives on every stage, also with no row to load:
      // one that did not could fall a phase behind the ring, whose parity
      // then reads the wrong way round
      mbar_init(&full[s], 1 + (GATHER ? 2 * kGatherWarps : 0));
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 16);
    }
    mbar_init(drain, 1);
    fence_mbar_init();
  } else if (warp == 3 && lane == 0) {
    tma_prefetch_desc(&tmA);
    if (!GATHER) tma_prefetch_desc(&tmA128);
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmC);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < S::kList; i += blockDim.x) {
    const int64_t t = first + static_cast<int64_t>(i) * step;
    if (t < table.tile[p.experts])
      table.list[i] = group_find(table, p, static_cast<int>(t), n_blocks);
  }
  tc_fence_before();
  cluster_sync();  // barriers and TMEM of both CTAs, this CTA's list
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int num_tiles = table.tile[p.experts];
  auto wait_all = [&](uint64_t *bar, uint32_t parity) -> bool {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, p.err));
  };
  // the product's N, a multiple of 32, and how many of the tile's rows lie in
  // CTA c's half of it
  auto tile_n = [](const GroupTile &t) -> int { return (t.end - t.row + 31) / 32 * 32; };
  auto cta_rows = [&](const GroupTile &t, int c) -> int {
    const int half = tile_n(t) / 2;
    return min(max(t.end - t.row - c * half, 0), half);
  };

  if (warp == 0) {
    // ---------------- W (and grouped A) producer, both CTAs ----------------
    if (lane == 0) {
      int stage = 0, local = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = first; tile < num_tiles && ok; tile += step, ++local) {
        const GroupTile t = group_tile(table, p, local, tile, n_blocks);
        uint32_t bytes = 2 * S::kWBytes;
        for (int c = 0; c < 2; ++c) {
          const int m = cta_rows(t, c);
          bytes += GATHER ? (m + 3) / 4 * 512
                          : (m + kGroupedBox - 1) / kGroupedBox * (kGroupedBox * 128);
        }
        const int boxes = GATHER ? 0 : (cta_rows(t, rank) + kGroupedBox - 1) / kGroupedBox;
        const int a_row = t.row + rank * (tile_n(t) / 2);
        const int w_block = ((t.e * n_blocks + t.nb) * 2 + rank) * num_kb;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1u, p.err)) {
            ok = false;
            break;
          }
          if (leader) mbar_arrive_expect_tx(&full[stage], bytes);
          const uint32_t bar = map_to_cta(smem_u32(&full[stage]), 0);
          tma_load_2d_pair(sW + stage * S::kWBytes, &tmW, bar, 0, (w_block + kb) * 128);
          if (boxes == kGemmBM / kGroupedBox) {
            tma_load_2d_pair(sA + stage * a_bytes, &tmA128, bar, kb * kGemmBK, a_row);
          } else {
            for (int i = 0; i < boxes; ++i)
              tma_load_2d_pair(sA + stage * a_bytes + i * kGroupedBox * 128, &tmA, bar,
                               kb * kGemmBK, a_row + i * kGroupedBox);
          }
          if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // Tail: the MMAs have released every stage, so all loads of this CTA
      // (the gathers too) have landed and all commits aimed at its barriers
      // have arrived before it may exit.
      for (int i = 0; i < stages && ok; ++i) {
        if (!mbar_wait(&empty[stage], phase ^ 1u, p.err)) break;
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer (the leader) ----------------
    if (leader) {
      const bool elect = elect_one_sync();
      int stage = 0;
      uint32_t phase = 0;
      bool issued_any = false, ok = true;
      int local = 0;
      for (int tile = first; tile < num_tiles && ok; tile += step, ++local) {
        const GroupTile t = group_tile(table, p, local, tile, n_blocks);
        const uint32_t idesc = idesc_bf16_f32(256, tile_n(t));
        const int acc = local % kBuffers;
        if (!wait_all(&tempty[acc], ((local / kBuffers) & 1) ^ 1u)) break;
        tc_fence_after();
        for (int kb = 0; kb < num_kb; ++kb) {
          int kb0 = 0;  // where the accumulator begins
          uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * kAccCols);
          if constexpr (EPI == kGrpF32) {
            const int part = kb / part_kb;
            kb0 = part * part_kb;
            d_tmem += static_cast<uint32_t>(part * p.tile_rows);
          }
          if (!wait_all(&full[stage], phase)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t da = sdesc_kmajor_sw128(smem_u32(sA + stage * a_bytes));
          const uint64_t dw = sdesc_kmajor_sw128(smem_u32(sW + stage * S::kWBytes));
          if (elect) {
#pragma unroll
            for (int k = 0; k < kGemmBK / 16; ++k)
              umma_bf16_pair(d_tmem, dw + k * 2, da + k * 2, idesc, kb != kb0 || k != 0 ? 1u : 0u);
            umma_commit_pair(&empty[stage], 0x3);
          }
          __syncwarp();
          issued_any = true;
          if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (ok && elect) umma_commit_pair(&tfull[acc], 0x3);
        __syncwarp();
      }
      if (issued_any) {
        if (elect) umma_commit_pair(drain, 0x1);
        __syncwarp();
        wait_all(drain, 0);
      }
    }
  } else if (warp < 10) {
    // ---------------- epilogue ----------------
    // TMEM lanes are W's columns: 32 of them a quarter, a warp for each half
    // of the tile's rows, 32 x 32 chunks in the fragment layout that stmatrix
    // turns over.  A gated weight's quarters alternate between up and gate of
    // the same 32 output columns, so the warps of quarters 2q and 2q + 1 work
    // on two chunks together: each hands the other its values of one chunk
    // through shared memory and finishes the other.
    constexpr bool kGated = grp_gated(EPI);
    constexpr int kChunkBytes = EPI == kGrpF32 ? 4096 : 2048;
    constexpr int kSlots = kGated ? 1 : S::kWarpStaging / kChunkBytes;
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const int gate = kGated ? quarter & 1 : 0;
    const int pair = half * 2 + (quarter >> 1);  // gated: pair of warps
    float4 *send = reinterpret_cast<float4 *>(staging + pair * 8192 + gate * 4096) + lane;
    const float4 *receive =
        reinterpret_cast<float4 *>(staging + pair * 8192 + (gate ^ 1) * 4096) + lane;
    uint8_t *mine = kGated ? staging + 32768 + (warp - 2) * 2048
                           : staging + (warp - 2) * S::kWarpStaging;
    const int width = kGated ? p.N / 2 : p.N;
    int slot = 0;
    int local = 0;
    for (int tile = first; tile < num_tiles; tile += step, ++local) {
      const int acc = local % kBuffers;
      const GroupTile t = group_tile(table, p, local, tile, n_blocks);
      // first W column of the quarter (of the pair of quarters), and of C
      const int col = t.nb * 256 + rank * 128 + (kGated ? quarter & 2 : quarter) * 32;
      const int c0 = kGated ? col / 2 : col;
      // this thread's columns of a chunk: c0 + lane / 4 + {0, 8, 16, 24}
      float b[4], bg[4];
      grp_bias4(p.bias ? p.bias + static_cast<int64_t>(t.e) * p.N : nullptr, c0 + (lane >> 2),
                width, b);
      if constexpr (kGated)
        grp_bias4(p.bias ? p.bias + static_cast<int64_t>(t.e) * p.N + width : nullptr,
                  c0 + (lane >> 2), width, bg);
      bool ok = wait_all(&tfull[acc], (local / kBuffers) & 1);
      if constexpr (kGated) ok = grp_pair_and(1 + pair, ok);
      if (!ok) break;
      tc_fence_after();
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) +
                             static_cast<uint32_t>(acc * kAccCols);
      const int chunks = tile_n(t) / 32;
      const int split = (chunks + 1) / 2;
      const int begin = half ? split : 0, end = half ? chunks : split;
      if (c0 < width) {  // the same for both warps of a pair
#pragma unroll 1
        for (int c = begin; c < end; c += kGated ? 2 : 1) {
          uint32_t r[32];
          int at = c;  // the chunk this warp finishes
          if constexpr (kGated) {
            // up: keeps c, hands over c + 1; gate: hands over c, keeps c + 1
            const bool two = c + 1 < end;
            if (gate || two) {
              grp_load_chunk(t_row + (gate ? c : c + 1) * 32, r);
              // the other warp has read what this one handed over before
              grp_pair_sync(1 + pair);
#pragma unroll
              for (int i = 0; i < 8; ++i)
                send[i * 32] = make_float4(__uint_as_float(r[4 * i]), __uint_as_float(r[4 * i + 1]),
                                           __uint_as_float(r[4 * i + 2]),
                                           __uint_as_float(r[4 * i + 3]));
            } else {
              grp_pair_sync(1 + pair);
            }
            at = gate ? c + 1 : c;
            if (at < end) grp_load_chunk(t_row + at * 32, r);
            grp_pair_sync(1 + pair);
            if (at >= end) continue;
          } else {
            grp_load_chunk(t_row + c * 32, r);
            if constexpr (EPI == kGrpF32) {
              for (int part = 1; part < parts; ++part) {
                uint32_t s[32];
                grp_load_chunk(t_row + part * p.tile_rows + c * 32, s);
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  r[i] = __float_as_uint(__uint_as_float(r[i]) + __uint_as_float(s[i]));
              }
            }
          }
          // entry 4 i + j: column lane / 4 + 8 * (2 * (i / 4) + j / 2), row
          // 8 * (i % 4) + 2 * (lane % 4) + j % 2, finished two at a time and
          // narrowed as they are made (16 registers a chunk instead of 32)
          std::conditional_t<EPI == kGrpF32, float[32], uint32_t[16]> v;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float4 o;
            if constexpr (kGated) o = receive[i * 32];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int q = 2 * (i / 4) + j;
              uint64_t x =
                  pk2(__uint_as_float(r[4 * i + 2 * j]), __uint_as_float(r[4 * i + 2 * j + 1]));
              if constexpr (kGated) {
                uint64_t g = j ? pk2(o.z, o.w) : pk2(o.x, o.y);
                if (gate) {  // the same for the whole warp
                  const uint64_t y = x;
                  x = g;
                  g = y;
                }
                float g0, g1;
                unpk2(add_x2(g, pk2(bg[q], bg[q])), g0, g1);
                if constexpr (EPI == kGrpBf16SwiGLU) grp_silu_x2(g0, g1);
                else gelu_erf_x2(g0, g1);
                x = mul_x2(add_x2(x, pk2(b[q], b[q])), pk2(g0, g1));
              } else {
                x = add_x2(x, pk2(b[q], b[q]));
              }
              float x0, x1;
              unpk2(x, x0, x1);
              if constexpr (EPI == kGrpBf16Gelu8) gelu8_x2(x0, x1);
              if constexpr (EPI == kGrpBf16Erf) gelu_erf_x2(x0, x1);
              if constexpr (EPI == kGrpF32) {
                v[4 * i + 2 * j] = x0;
                v[4 * i + 2 * j + 1] = x1;
              } else {
                v[2 * i + j] = pack_bf16x2(x0, x1);
              }
            }
          }
          uint8_t *chunk = mine + slot * kChunkBytes;
          if (lane == 0) bulk_wait_group_read<kSlots - 1>();
          __syncwarp();
          grp_stage_t(v, chunk, lane);
          const int row0 = t.row + at * 32;
          if (row0 + 32 <= t.end) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&tmC, chunk, c0, row0);
              bulk_commit_group();
            }
            if (++slot == kSlots) slot = 0;
          } else {
            __syncwarp();
            grp_store_rows<EPI>(p.out, chunk, row0, t.end, c0, width, lane);
          }
          __syncwarp();
        }
      }
      tc_fence_before();
      __syncwarp();
      // (the fence orders the TMEM reads; a releasing arrive at cluster scope
      // would also wait for this thread's outstanding accesses, a microsecond)
      if (lane == 0) grp_arrive(map_to_cta(smem_u32(&tempty[acc]), 0));
    }
    if (lane == 0) bulk_wait_group_all();
  } else if constexpr (GATHER) {
    // ---------------- A by gathers (warps 10..17) ----------------
    const int part = warp - 10;  // a share of this CTA's 128 rows
    const bool elect = elect_one_sync();
    int stage = 0, local = 0;
    uint32_t phase = 0;
    bool ok = true;
    // this warp's rows of a tile, and the lane's row of A for one of them;
    // a tile's are read while the one before is loaded
    auto count_of = [&](const GroupTile &t) -> int {
      return min(max(cta_rows(t, rank) - kGatherRows * part, 0), kGatherRows);
    };
    auto index_of = [&](int l, int tile) -> int {
      if (tile >= num_tiles) return 0;
      const GroupTile t = group_tile(table, p, l, tile, n_blocks);
      const int count = count_of(t);
      // past the group: its last row again, to fill a gather of four
      return count ? __ldg(p.row_src + t.row + rank * (tile_n(t) / 2) + kGatherRows * part +
                           min(lane, count - 1))
                   : 0;
    };
    int next = index_of(0, first);
    for (int tile = first; tile < num_tiles && ok; tile += step, ++local) {
      const int count = count_of(group_tile(table, p, local, tile, n_blocks));
      int mine = next;
      next = index_of(local + 1, tile + step);
      if (mine < 0 || mine >= p.a_rows) {
        record_err(p.err, kDevBadGroup);
        mine = 0;
      }
      int src[kGatherRows];
#pragma unroll
      for (int i = 0; i < kGatherRows; ++i) src[i] = __shfl_sync(0xffffffffu, mine, i);
      for (int kb = 0; kb < num_kb; ++kb) {
        if (!wait_all(&empty[stage], phase ^ 1u)) {
          ok = false;
          break;
        }
        if (elect) {
          const uint32_t dst = smem_u32(sA + stage * a_bytes) + part * (kGatherRows * 128);
          const uint32_t bar = map_to_cta(smem_u32(&full[stage]), 0);
#pragma unroll
          for (int i = 0; i < kGatherRows / 4; ++i)
            if (4 * i < count)
              grp_gather4(dst + i * 512, &tmA, bar, kb * kGemmBK, src[4 * i], src[4 * i + 1],
                          src[4 * i + 2], src[4 * i + 3]);
          grp_arrive(bar);
        }
        __syncwarp();
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  }

  tc_fence_before();
  cluster_sync();  // no CTA leaves while its pair may still signal it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 2 * kAccCols);
  }
}

#ifdef NEBW_LAYER_KERNELS
// Expert weights [experts, K, N] (fp32 or bf16) to bf16 RNE blocks of 128
// columns by 64 of K, [experts][column block][K block][128][64]: a block is
// 16 KB in one piece, which a TMA box reads as 128 consecutive rows of 128
// bytes (2 to 4% faster than the same boxes from [N, K] rows: 43.1 against
// 44.0 us on 2011 rows of 64 experts, 15.2 against 16.0 on 128 rows of 8).
// Column blocks come in twos; columns past N and K are zero.  A gated weight's
// column n takes column glu(n) of [up | gate].
__global__ void stage_experts_kernel(const void *__restrict__ src, int src_bf16, int K, int N,
                                     int gated, int e0, int col_blocks, int k_blocks,
                                     __nv_bfloat16 *__restrict__ dst) {
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
    const int64_t block = ((e0 + e) * col_blocks + n / 128) * k_blocks + k / 64;
    dst[(block * 128 + n % 128) * 64 + k % 64] = __float2bfloat16_rn(tile[threadIdx.x][i]);
  }
}
#endif

}  // namespace nebw
