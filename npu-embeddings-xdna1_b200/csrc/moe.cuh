// Expert routing: the top-k experts of every row with their weights, the
// rows grouped by expert, and the weighted sum of the experts' rows.
//
//   chosen(t)   the k largest logits of row t, ties to the lower expert; a
//               logit of -inf (a masked expert) or NaN is never chosen
//   softmax     p_e = exp(l_e - max l) / sum_e exp(l_e - max l)
//   sigmoid     p_e = 1 / (1 + exp(-l_e))
//   weights     p_e, or p_e / (sum of the chosen p) with renorm; times scale
//   grouping    stable: expert by expert, rows ascending within one; places
//               group_off[e] .. group_off[e + 1]
//
// Everything whole is exact and has one order whatever the schedule: the
// choice compares the logits themselves, and places come from counts, never
// from the order in which blocks reach an atomic.
#pragma once

#include <cuda_bf16.h>
#include <cstdint>

#include "ptx.cuh"
#include "rowops.cuh"

namespace nebw {

constexpr int kRouteWarps = 16;
constexpr int kRouteThreads = kRouteWarps * 32;
constexpr int kRouteWarpRows = 32;
constexpr int kRouteBlockRows = kRouteWarps * kRouteWarpRows;  // rows a block
constexpr int kRouteMaxExperts = 512;
constexpr int kRouteMaxK = 16;

struct RouteArgs {
  const void *logits;  // [rows, stride], fp32 or bf16
  int64_t stride;
  int64_t rows;
  const int *rows_dev;  // if set, the live row count is min(*rows_dev, rows)
  int experts, k;
  int sigmoid, renorm;
  float scale;
  int *ids;         // [rows, k], -1 where fewer than k could be chosen
  float *weights;   // [rows, k]
  int *group_off;   // [experts + 1]
  int *row_src;     // [rows * k]: the row at each grouped place
  int *row_dst;     // [rows, k]: the place of each row's expert, -1 if none
  int *hist;        // [blocks, experts]
  int blocks;
};

__device__ __forceinline__ int64_t route_rows(const RouteArgs &p) {
  if (!p.rows_dev) return p.rows;
  return min(p.rows, static_cast<int64_t>(max(0, __ldg(p.rows_dev))));
}

// A logit as an unsigned key of the same order; 0 for -inf and NaN.  -0 and
// +0 are one value.
__device__ __forceinline__ uint32_t route_key(float v) {
  if (!(v > -INFINITY)) return 0u;
  const uint32_t u = __float_as_uint(v + 0.0f);
  return u ^ (u & 0x80000000u ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float route_value(uint32_t key) {
  return __uint_as_float(key ^ (key & 0x80000000u ? 0x80000000u : 0xffffffffu));
}

// One row's choice by one warp; lane j < k returns its j-th expert (or -1)
// and weight.  NV logits a lane: expert i * 32 + lane.
template <typename T, int NV>
__device__ __forceinline__ void route_row(const RouteArgs &p, int64_t row, int lane, int &id,
                                          float &weight) {
  const T *l = static_cast<const T *>(p.logits) + row * p.stride;
  uint32_t key[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = i * 32 + lane;
    float v = -INFINITY;
    if (e < p.experts) {
      if constexpr (sizeof(T) == 4) v = l[e];
      else v = __bfloat162float(l[e]);
    }
    key[i] = route_key(v);
  }
  float sum_all = 0.f, top = 0.f;
  uint32_t mine = 0;
  id = -1;
  for (int j = 0; j < p.k; ++j) {
    uint32_t best = 0;
    int at = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (key[i] > best) {
        best = key[i];
        at = i;
      }
    const uint32_t m = __reduce_max_sync(0xffffffffu, best);
    if (m == 0) break;
    const unsigned e =
        __reduce_min_sync(0xffffffffu, best == m ? static_cast<unsigned>(at * 32 + lane) : ~0u);
    if (j == 0) {
      top = route_value(m);
      if (!p.sigmoid && !p.renorm) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const float v = route_value(key[i]);
          if (key[i]) sum_all += v == top ? 1.0f : expf(v - top);
        }
        sum_all = warp_sum(sum_all);
      }
    }
    if (static_cast<int>(e & 31) == lane) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (i == static_cast<int>(e >> 5)) key[i] = 0;
    }
    if (lane == j) {
      id = static_cast<int>(e);
      mine = m;
    }
  }
  weight = 0.f;
  if (mine) {
    const float v = route_value(mine);
    weight = p.sigmoid ? 1.0f / (1.0f + expf(-v)) : v == top ? 1.0f : expf(v - top);
  }
  if (p.renorm) {
    const float s = warp_sum(weight);
    weight = s > 0.f ? weight / s : 0.f;
  } else if (!p.sigmoid && mine) {
    weight /= sum_all;
  }
  weight *= p.scale;
}

// The choice of every row, and each block's count of rows per expert.
template <typename T, int NV>
__global__ void __launch_bounds__(kRouteThreads) route_topk_kernel(const RouteArgs p) {
  __shared__ int count[kRouteMaxExperts];
  for (int e = threadIdx.x; e < p.experts; e += kRouteThreads) count[e] = 0;
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t rows = route_rows(p);
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * kRouteBlockRows + warp * kRouteWarpRows;
  for (int r = 0; r < kRouteWarpRows && r0 + r < rows; ++r) {
    int id;
    float w;
    route_row<T, NV>(p, r0 + r, lane, id, w);
    if (lane < p.k) {
      p.ids[(r0 + r) * p.k + lane] = id;
      p.weights[(r0 + r) * p.k + lane] = w;
      if (id >= 0) atomicAdd(&count[id], 1);
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.experts; e += kRouteThreads)
    p.hist[static_cast<int64_t>(blockIdx.x) * p.experts + e] = count[e];
}

// The grouped place of every chosen (row, expert): the counts of all blocks
// give each expert's start and this block's start within it; the order inside
// a block comes from a count per warp and a match within 32 entries.
__global__ void __launch_bounds__(kRouteThreads) route_place_kernel(const RouteArgs p) {
  extern __shared__ int sh[];
  int *start = sh;                    // [experts]
  int *cnt = sh + p.experts;          // [warps, experts]
  const int E = p.experts;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int e = threadIdx.x; e < E; e += kRouteThreads) {
    int before = 0, all = 0;
    for (int b = 0; b < p.blocks; ++b) {
      const int c = p.hist[static_cast<int64_t>(b) * E + e];
      if (b < static_cast<int>(blockIdx.x)) before += c;
      all += c;
    }
    start[e] = before;
    cnt[e] = all;
  }
  __syncthreads();
  if (warp == 0) {  // exclusive scan of the totals over the experts
    int run = 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
      const int e = e0 + lane;
      const int c = e < E ? cnt[e] : 0;
      int inc = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      if (e < E) {
        start[e] += run + inc - c;
        if (blockIdx.x == 0) p.group_off[e] = run + inc - c;
      }
      run += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (blockIdx.x == 0 && lane == 0) p.group_off[E] = run;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kRouteWarps * E; i += kRouteThreads) cnt[i] = 0;
  __syncthreads();
  const int64_t rows = route_rows(p);
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * kRouteBlockRows + warp * kRouteWarpRows;
  const int64_t i0 = r0 * p.k;
  const int64_t i1 = min(rows, r0 + kRouteWarpRows) * p.k;
  int *mine = cnt + warp * E;
  for (int64_t i = i0; i < i1; i += 32) {
    const int id = i + lane < i1 ? p.ids[i + lane] : -1;
    const unsigned same = __match_any_sync(0xffffffffu, id);
    if (id >= 0 && (same & ((1u << lane) - 1)) == 0) mine[id] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += kRouteThreads) {
    int run = start[e];
    for (int w = 0; w < kRouteWarps; ++w) {
      const int c = cnt[w * E + e];
      cnt[w * E + e] = run;
      run += c;
    }
  }
  __syncthreads();
  for (int64_t i = i0; i < i1; i += 32) {
    const int id = i + lane < i1 ? p.ids[i + lane] : -1;
    const unsigned same = __match_any_sync(0xffffffffu, id);
    const unsigned below = same & ((1u << lane) - 1);
    int place = -1;
    if (id >= 0) place = mine[id] + __popc(below);
    __syncwarp();
    if (id >= 0 && below == 0) mine[id] += __popc(same);
    __syncwarp();
    if (i + lane < i1) {
      p.row_dst[i + lane] = place;
      if (place >= 0) p.row_src[place] = static_cast<int>((i + lane) / p.k);
    }
  }
}

// out[t] = residual[t] + sum_j weights[t, j] * y[row_dst[t, j]], j ascending,
// in fp32 with one rounding at the end; an entry without a place (row_dst
// < 0) adds nothing and is not read.
struct CombineArgs {
  const void *y;
  const int *row_dst;
  const float *weights;
  const float *residual;
  void *out;
  int64_t rows, y_rows;
  const int *rows_dev;
  int k;
  int64_t H;
  int *err;
};

template <typename TY, typename TO, int V>
__global__ void __launch_bounds__(256) moe_combine_kernel(const CombineArgs p) {
  const int64_t per_row = p.H / V;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  int64_t rows = p.rows;
  if (p.rows_dev) rows = min(rows, static_cast<int64_t>(max(0, __ldg(p.rows_dev))));
  const int64_t row = i / per_row;
  if (row >= rows) return;
  const int64_t c = (i - row * per_row) * V;
  float acc[V];
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] = 0.f;
  for (int j = 0; j < p.k; ++j) {
    const int at = __ldg(p.row_dst + row * p.k + j);
    if (at < 0) continue;
    if (at >= p.y_rows) {
      record_err(p.err, kDevBadGroup);
      continue;
    }
    const float w = __ldg(p.weights + row * p.k + j);
    const TY *y = static_cast<const TY *>(p.y) + static_cast<int64_t>(at) * p.H + c;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float f;
      if constexpr (sizeof(TY) == 4) f = y[v];
      else f = __bfloat162float(y[v]);
      acc[v] = fmaf(w, f, acc[v]);
    }
  }
  const int64_t o = row * p.H + c;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if (p.residual) acc[v] += p.residual[o + v];
    if constexpr (sizeof(TO) == 4) static_cast<float *>(p.out)[o + v] = acc[v];
    else static_cast<__nv_bfloat16 *>(p.out)[o + v] = __float2bfloat16_rn(acc[v]);
  }
}

}  // namespace nebw
