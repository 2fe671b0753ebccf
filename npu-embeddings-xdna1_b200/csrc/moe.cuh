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

constexpr int kRouteThreads = 512;
constexpr int kRouteWarps = kRouteThreads / 32;
constexpr int kRouteMaxExperts = 512;
constexpr int kRouteMaxK = 16;
constexpr int kRouteFusedRows = 256;  // up to here one block does it all

struct RouteArgs {
  const void *logits;  // [rows, stride], fp32 or bf16
  int64_t stride;
  int rows;
  const int *rows_dev;  // if set, the live row count is min(*rows_dev, rows)
  int experts, k;
  int sigmoid, renorm;
  float scale;
  int *ids;         // [rows, k], -1 where fewer than k could be chosen
  float *weights;   // [rows, k]
  int *group_off;   // [experts + 1]
  int *row_src;     // [rows * k]: the row at each grouped place
  int *row_dst;     // [rows, k]: the place of each row's expert, -1 if none
  int *hist;        // [blocks, experts]; unused by one block
  int lg;           // 2^lg lanes share a row,
  int per;          // each with `per` consecutive experts (a multiple of 8)
  int vec;          // rows of whole, aligned 16-byte vectors
  int block_rows;   // rows a block
};

__device__ __forceinline__ int route_rows(const RouteArgs &p) {
  return p.rows_dev ? min(p.rows, max(0, __ldg(p.rows_dev))) : p.rows;
}

// A logit and its expert as one unsigned key: the larger logit first, then
// the lower expert; 0 for -inf and NaN.  -0 and +0 are one value.  bf16 keys
// fit 32 bits (16 of the value, 16 of the expert), fp32 keys take 64.
template <typename T>
struct RouteKey;
template <>
struct RouteKey<__nv_bfloat16> {
  using Key = uint32_t;
  static __device__ __forceinline__ Key make(uint32_t bits16, int e) {
    const uint32_t u = bits16 == 0x8000u ? 0u : bits16;
    const uint32_t o = u & 0x8000u ? u ^ 0xffffu : u | 0x8000u;  // ascending
    // above -inf (0x007f) and up to +inf (0xff80); NaN of either sign is outside
    return o > 0x007fu && o <= 0xff80u ? (o << 16) | (0xffffu - e) : 0u;
  }
  static __device__ __forceinline__ float value(Key k) {
    const uint32_t o = k >> 16;
    return __uint_as_float((o & 0x8000u ? o & 0x7fffu : o ^ 0xffffu) << 16);
  }
  static __device__ __forceinline__ int expert(Key k) { return 0xffff - (k & 0xffffu); }
  // eight consecutive logits
  static __device__ __forceinline__ void load8(const __nv_bfloat16 *l, int e, int n, bool vec,
                                               Key (&k)[8]) {
    if (vec) {
      const uint4 u = __ldg(reinterpret_cast<const uint4 *>(l + e));
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) k[i] = make(i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu, e + i);
    } else {
      const unsigned short *s = reinterpret_cast<const unsigned short *>(l);
#pragma unroll
      for (int i = 0; i < 8; ++i) k[i] = e + i < n ? make(__ldg(s + e + i), e + i) : 0u;
    }
  }
};
template <>
struct RouteKey<float> {
  using Key = unsigned long long;
  static __device__ __forceinline__ Key make(float v, int e) {
    const uint32_t u = __float_as_uint(v + 0.0f);  // -0 + 0 = +0
    const uint32_t o = u ^ (u & 0x80000000u ? 0xffffffffu : 0x80000000u);
    return v > -INFINITY ? (static_cast<Key>(o) << 32) | (0xffffu - e) : 0ull;
  }
  static __device__ __forceinline__ float value(Key k) {
    const uint32_t o = static_cast<uint32_t>(k >> 32);
    return __uint_as_float(o ^ (o & 0x80000000u ? 0x80000000u : 0xffffffffu));
  }
  static __device__ __forceinline__ int expert(Key k) {
    return 0xffff - static_cast<int>(k & 0xffffu);
  }
  static __device__ __forceinline__ void load8(const float *l, int e, int n, bool vec,
                                               Key (&k)[8]) {
    if (vec) {
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        const float4 v = __ldg(reinterpret_cast<const float4 *>(l + e + i));
        k[i] = make(v.x, e + i);
        k[i + 1] = make(v.y, e + i + 1);
        k[i + 2] = make(v.z, e + i + 2);
        k[i + 3] = make(v.w, e + i + 3);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) k[i] = e + i < n ? make(__ldg(l + e + i), e + i) : 0ull;
    }
  }
};

// a >= b afterwards.
template <typename Key>
__device__ __forceinline__ void route_order(Key &a, Key &b) {
  const Key hi = max(a, b), lo = min(a, b);
  a = hi;
  b = lo;
}

// One row's choice by the 2^lg lanes that share it: each keeps the K largest
// keys of its experts in order (insertion, unrolled and without a branch),
// then lanes merge in pairs: the K largest of two ordered lists are max(a[i],
// b[K - 1 - i]), which a bitonic pass orders again.  Every lane ends with the
// row's list.
template <typename T, int K>
__device__ __forceinline__ void route_row(const RouteArgs &p, const T *l, int sub,
                                          typename RouteKey<T>::Key (&top)[K]) {
  using R = RouteKey<T>;
  using Key = typename R::Key;
#pragma unroll
  for (int i = 0; i < K; ++i) top[i] = 0;
  const int end = min(p.experts, (sub + 1) * p.per);
  for (int e = sub * p.per; e < end; e += 8) {
    Key k[8];
    R::load8(l, e, p.experts, p.vec, k);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
      for (int j = 0; j < K; ++j) route_order(top[j], k[i]);
    }
  }
  for (int o = 1; o < 1 << p.lg; o <<= 1) {
    Key other[K];
#pragma unroll
    for (int i = 0; i < K; ++i) other[i] = __shfl_xor_sync(0xffffffffu, top[i], o);
#pragma unroll
    for (int i = 0; i < K; ++i) top[i] = max(top[i], other[K - 1 - i]);
#pragma unroll
    for (int d = K / 2; d > 0; d >>= 1) {
#pragma unroll
      for (int i = 0; i < K; ++i)
        if ((i & d) == 0) route_order(top[i], top[i + d]);
    }
  }
}

// The choice of this block's rows, written out and counted per expert.
template <typename T, int K>
__device__ __forceinline__ void route_choose(const RouteArgs &p, int r0, int r1, int *count) {
  using R = RouteKey<T>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = lane & ((1 << p.lg) - 1);
  const int rows_warp = 32 >> p.lg;
  for (int rb = r0 + warp * rows_warp; rb < r1; rb += kRouteWarps * rows_warp) {
    const int row = rb + (lane >> p.lg);
    const bool live = row < r1;
    // lanes of a row that is not there walk the last one
    const T *l = static_cast<const T *>(p.logits) +
                 static_cast<int64_t>(live ? row : r1 - 1) * p.stride;
    typename R::Key top[K];
    route_row<T, K>(p, l, sub, top);
    const float first = R::value(top[0]);
    float sum = 0.f;
    if (!p.sigmoid && !p.renorm) {
      const int end = min(p.experts, (sub + 1) * p.per);
      for (int e = sub * p.per; e < end; e += 8) {
        typename R::Key k[8];
        R::load8(l, e, p.experts, p.vec, k);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float v = R::value(k[i]);
          if (k[i]) sum += v == first ? 1.0f : expf(v - first);  // inf - inf is no number
        }
      }
      for (int o = 1; o < 1 << p.lg; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    if (!live || sub != 0) continue;
    float w[K];
    float chosen = 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      w[j] = 0.f;
      if (j < p.k && top[j]) {
        const float v = R::value(top[j]);
        w[j] = p.sigmoid ? 1.0f / (1.0f + expf(-v)) : v == first ? 1.0f : expf(v - first);
        chosen += w[j];
      }
    }
    if (p.renorm) sum = chosen;
    const bool divide = p.renorm || !p.sigmoid;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      if (j < p.k) {
        const int id = top[j] ? R::expert(top[j]) : -1;
        if (divide) w[j] = sum > 0.f ? w[j] / sum : 0.f;
        p.ids[static_cast<int64_t>(row) * p.k + j] = id;
        p.weights[static_cast<int64_t>(row) * p.k + j] = w[j] * p.scale;
        if (id >= 0) atomicAdd(&count[id], 1);
      }
    }
  }
}

// The grouped places of this block's rows.  start [experts]: the first place
// of each expert for this block; cnt [warps, experts]: scratch.  The order
// inside a block comes from a count per warp and a match within 32 entries.
__device__ __forceinline__ void route_place(const RouteArgs &p, int r0, int r1, const int *start,
                                            int *cnt) {
  const int E = p.experts;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < kRouteWarps * E; i += kRouteThreads) cnt[i] = 0;
  __syncthreads();
  // each warp a run of whole groups of 32 entries
  const int n = (r1 - r0) * p.k;
  const int run = (n + kRouteThreads - 1) / kRouteThreads * 32;
  const int i0 = min(n, warp * run), i1 = min(n, i0 + run);
  const int *ids = p.ids + static_cast<int64_t>(r0) * p.k;
  int *mine = cnt + warp * E;
  for (int i = i0; i < i1; i += 32) {
    const int id = i + lane < i1 ? ids[i + lane] : -1;
    const unsigned same = __match_any_sync(0xffffffffu, id);
    if (id >= 0 && (same & ((1u << lane) - 1)) == 0) mine[id] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += kRouteThreads) {
    int at = start[e];
    for (int w = 0; w < kRouteWarps; ++w) {
      const int c = cnt[w * E + e];
      cnt[w * E + e] = at;
      at += c;
    }
  }
  __syncthreads();
  for (int i = i0; i < i1; i += 32) {
    const int id = i + lane < i1 ? ids[i + lane] : -1;
    const unsigned same = __match_any_sync(0xffffffffu, id);
    const unsigned below = same & ((1u << lane) - 1);
    int place = -1;
    if (id >= 0) place = mine[id] + __popc(below);
    __syncwarp();
    if (id >= 0 && below == 0) mine[id] += __popc(same);
    __syncwarp();
    if (i + lane < i1) {
      p.row_dst[static_cast<int64_t>(r0) * p.k + i + lane] = place;
      if (place >= 0) p.row_src[place] = r0 + (i + lane) / p.k;
    }
  }
}

// Exclusive scan of total [experts] over the experts by warp 0, added to
// start; the totals' scan is group_off.
__device__ __forceinline__ void route_scan(const RouteArgs &p, const int *total, int *start,
                                           bool write) {
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int run = 0;
    for (int e0 = 0; e0 < p.experts; e0 += 32) {
      const int e = e0 + lane;
      const int c = e < p.experts ? total[e] : 0;
      int inc = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      if (e < p.experts) {
        start[e] += run + inc - c;
        if (write) p.group_off[e] = run + inc - c;
      }
      run += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (write && lane == 0) p.group_off[p.experts] = run;
  }
}

// The choice of every row, and each block's count of rows per expert.
template <typename T, int K>
__global__ void __launch_bounds__(kRouteThreads) route_choose_kernel(const RouteArgs p) {
  __shared__ int count[kRouteMaxExperts];
  for (int e = threadIdx.x; e < p.experts; e += kRouteThreads) count[e] = 0;
  __syncthreads();
  const int rows = route_rows(p);
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * p.block_rows;
  if (r0 < rows)
    route_choose<T, K>(p, static_cast<int>(r0),
                       static_cast<int>(min(static_cast<int64_t>(rows), r0 + p.block_rows)), count);
  __syncthreads();
  for (int e = threadIdx.x; e < p.experts; e += kRouteThreads)
    p.hist[static_cast<int64_t>(blockIdx.x) * p.experts + e] = count[e];
}

// The places: the counts of all blocks give each expert's start and this
// block's start within it.
__global__ void __launch_bounds__(kRouteThreads) route_place_kernel(const RouteArgs p) {
  extern __shared__ int sh[];
  const int E = p.experts;
  int *start = sh, *total = sh + E, *cnt = sh + 2 * E;
  for (int e = threadIdx.x; e < 2 * E; e += kRouteThreads) sh[e] = 0;
  __syncthreads();
  // threads share the blocks' counts out among them, expert by expert
  int lanes = 32;
  while (lanes < E && lanes < kRouteThreads) lanes <<= 1;
  for (int e = threadIdx.x & (lanes - 1); e < E; e += lanes) {
    int before = 0, all = 0;
    for (int b = threadIdx.x / lanes; b < gridDim.x; b += kRouteThreads / lanes) {
      const int c = p.hist[static_cast<int64_t>(b) * E + e];
      if (b < static_cast<int>(blockIdx.x)) before += c;
      all += c;
    }
    atomicAdd(&start[e], before);
    atomicAdd(&total[e], all);
  }
  __syncthreads();
  route_scan(p, total, start, blockIdx.x == 0);
  __syncthreads();
  const int rows = route_rows(p);
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * p.block_rows;
  if (r0 < rows)
    route_place(p, static_cast<int>(r0),
                static_cast<int>(min(static_cast<int64_t>(rows), r0 + p.block_rows)), start, cnt);
}

// Few rows: one block chooses and places.
template <typename T, int K>
__global__ void __launch_bounds__(kRouteThreads) route_fused_kernel(const RouteArgs p) {
  extern __shared__ int sh[];
  const int E = p.experts;
  int *start = sh, *total = sh + E, *cnt = sh + 2 * E;
  for (int e = threadIdx.x; e < 2 * E; e += kRouteThreads) sh[e] = 0;
  __syncthreads();
  const int rows = route_rows(p);
  if (rows > 0) route_choose<T, K>(p, 0, rows, total);
  __syncthreads();
  route_scan(p, total, start, true);
  __syncthreads();
  route_place(p, 0, rows, start, cnt);
}

// out[t] = residual[t] + sum_j weights[t, j] * y[row_dst[t, j]], j ascending,
// in fp32 with one rounding at the end; an entry without a place (row_dst
// < 0) adds nothing and is not read.  HBM bounds it: k rows of y are read for
// one written.  V = 8 columns a thread by 16-byte accesses (1 where the width
// or an address does not allow them); the loads of four entries are issued
// together.
struct CombineArgs {
  const void *y;
  const int *row_dst;
  const float *weights;
  const float *residual;
  void *out;
  int rows, y_rows;
  const int *rows_dev;
  int k;
  int H;
  int *err;
};

template <int V>
__device__ __forceinline__ void combine_load(const float *y, float (&f)[V]) {
  if constexpr (V == 8) {
    const float4 a = __ldg(reinterpret_cast<const float4 *>(y));
    const float4 b = __ldg(reinterpret_cast<const float4 *>(y) + 1);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
    f[0] = __ldg(y);
  }
}
template <int V>
__device__ __forceinline__ void combine_load(const __nv_bfloat16 *y, float (&f)[V]) {
  if constexpr (V == 8) {
    const uint4 u = __ldg(reinterpret_cast<const uint4 *>(y));
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
    f[0] = __bfloat162float(*y);
  }
}

template <typename TY, typename TO, int V>
__global__ void __launch_bounds__(256) moe_combine_kernel(const CombineArgs p) {
  const int row = blockIdx.x * blockDim.y + threadIdx.y;
  const int rows = p.rows_dev ? min(p.rows, max(0, __ldg(p.rows_dev))) : p.rows;
  if (row >= rows) return;
  const int *dst = p.row_dst + static_cast<int64_t>(row) * p.k;
  const float *weights = p.weights + static_cast<int64_t>(row) * p.k;
  for (int c = threadIdx.x * V; c < p.H; c += blockDim.x * V) {
    const int64_t o = static_cast<int64_t>(row) * p.H + c;
    float acc[V];
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] = 0.f;
    for (int j0 = 0; j0 < p.k; j0 += 4) {
      float f[4][V], w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = j0 + j < p.k ? __ldg(dst + j0 + j) : -1;
        w[j] = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) f[j][v] = 0.f;
        if (at >= p.y_rows) {
          record_err(p.err, kDevBadGroup);
        } else if (at >= 0) {
          w[j] = __ldg(weights + j0 + j);
          combine_load<V>(static_cast<const TY *>(p.y) + static_cast<int64_t>(at) * p.H + c, f[j]);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] = fmaf(w[j], f[j][v], acc[v]);
      }
    }
    if (p.residual) {
      float r[V];
      if constexpr (V == 8) {  // not __ldg: residual may be out
        const float4 *r4 = reinterpret_cast<const float4 *>(p.residual + o);
        const float4 a = r4[0], b = r4[1];
        r[0] = a.x; r[1] = a.y; r[2] = a.z; r[3] = a.w;
        r[4] = b.x; r[5] = b.y; r[6] = b.z; r[7] = b.w;
      } else {
        r[0] = p.residual[o];
      }
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] += r[v];
    }
    if constexpr (sizeof(TO) == 4) {
      float *out = static_cast<float *>(p.out) + o;
      if constexpr (V == 8) {
        reinterpret_cast<float4 *>(out)[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
        reinterpret_cast<float4 *>(out)[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
      } else {
        *out = acc[0];
      }
    } else {
      __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(p.out) + o;
      if constexpr (V == 8)
        *reinterpret_cast<uint4 *>(out) =
            make_uint4(pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3]),
                       pack_bf16x2(acc[4], acc[5]), pack_bf16x2(acc[6], acc[7]));
      else
        *out = __float2bfloat16_rn(acc[0]);
    }
  }
}

}  // namespace nebw
