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
//
// Measured: 26.8 us replayed from a graph (31 as a call among others) for
// 131,071 rows of 64 bf16 logits by 8, whose bytes take 5.2.  The choice is
// about 17 of it.  A lane orders 16 keys and merges twice with another (86
// exchanges, 204 min and max instructions with what picks the larger): the ALU
// pipe is 77% busy while an SM works, 59% over the whole launch, and the rest
// is waiting, for logits that are read and used in one turn and for a fourth
// turn that is half empty (896 rows a block, 256 a turn).  The places are the
// other third, a chain of counts and barriers with the issue slots 23% busy.
// (One warp a row, with a warp-wide maximum for every chosen expert, and places
// by a match within 32 entries took 141 us.)  fp32 logits, whose keys take 64
// bits, are 1.5 times as long; lists of 16 of them spill 96 bytes.  A few rows
// cost one launch: 3.1 us for 21 rows of 8 by 2.
#pragma once

#include <cuda_bf16.h>
#include <cstdint>

#include "ptx.cuh"
#include "rowops.cuh"

namespace nebw {

constexpr int kRouteThreads = 1024;
constexpr int kRouteWarps = kRouteThreads / 32;
constexpr int kRouteMaxExperts = 512;
constexpr int kRouteMaxK = 16;

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
  int per;          // consecutive experts a lane looks at, a multiple of 8
  int vec;          // rows of whole, aligned 16-byte vectors
  int block_rows;   // rows a block, a multiple of 32
  int tiles;        // tiles of 32 rows placed at once
  int whole;        // k is the list's length and rows of ids and row_dst are 16-byte vectors
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
  // v: a bf16 value's bits in the upper half
  static __device__ __forceinline__ Key make(uint32_t v, int e) {
    const float f = __uint_as_float(v) + 0.0f;  // -0 + 0 = +0
    const int u = __float_as_int(f);
    const uint32_t o = static_cast<uint32_t>(u ^ ((u >> 31) | static_cast<int>(0x80000000)));
    return f > -INFINITY ? (o & 0xffff0000u) | (0xffffu - e) : 0u;
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
      for (int i = 0; i < 8; ++i)
        k[i] = make(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16, e + i);
    } else {
      const unsigned short *s = reinterpret_cast<const unsigned short *>(l);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        k[i] = e + i < n ? make(static_cast<uint32_t>(__ldg(s + e + i)) << 16, e + i) : 0u;
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

// The D stages of a bitonic merge over N elements: descending order from a
// bitonic sequence.
template <int N, typename Key>
__device__ __forceinline__ void route_merge(Key (&k)[N]) {
#pragma unroll
  for (int d = N / 2; d > 0; d >>= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if ((i & d) == 0) route_order(k[i], k[i + d]);
  }
}

// Eight keys in descending order (Batcher's odd-even merge sort, 19
// exchanges).
template <typename Key>
__device__ __forceinline__ void route_sort8(Key (&k)[8]) {
  constexpr int kNet[19][2] = {{0, 1}, {2, 3}, {4, 5}, {6, 7}, {0, 2}, {1, 3}, {4, 6},
                               {5, 7}, {1, 2}, {5, 6}, {0, 4}, {1, 5}, {2, 6}, {3, 7},
                               {2, 4}, {3, 5}, {1, 2}, {3, 4}, {5, 6}};
#pragma unroll
  for (int i = 0; i < 19; ++i) route_order(k[kNet[i][0]], k[kNet[i][1]]);
}

// Eight more keys into the ordered list of the K largest.  Up to four places
// an insertion is the shortest; longer lists sort the eight first: the K
// largest of two ordered lists are max(a[i], b[K - 1 - i]), a bitonic
// sequence that a merge orders again (35 exchanges for K = 8 against 64).
template <int K, typename Key>
__device__ __forceinline__ void route_add8(Key (&top)[K], Key (&k)[8]) {
  if constexpr (K <= 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
      for (int j = 0; j < K; ++j) route_order(top[j], k[i]);
    }
  } else {
    route_sort8(k);
#pragma unroll
    for (int i = 0; i < 8; ++i) top[K - 1 - i] = max(top[K - 1 - i], k[i]);
    route_merge<K>(top);
  }
}

// One row's choice by the 2^LG lanes that share it: each keeps the K largest
// keys of its experts in order, then lanes merge in pairs.  Every lane ends
// with the row's list.
template <typename T, int K, int LG>
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
    route_add8<K>(top, k);
  }
#pragma unroll
  for (int o = 1; o < 1 << LG; o <<= 1) {
    Key other[K];
#pragma unroll
    for (int i = 0; i < K; ++i) other[i] = __shfl_xor_sync(0xffffffffu, top[i], o);
#pragma unroll
    for (int i = 0; i < K; ++i) top[i] = max(top[i], other[K - 1 - i]);
    route_merge<K>(top);
  }
}

// The score of a chosen expert before it is normalised; `first` is the row's
// largest logit.  Sigmoids that are divided by their sum are taken times
// exp(-first) where first < 0: sigmoid(v) = exp(v) / (1 + exp(v)), so the first
// one is 1 / (1 + exp(first)) > 1/2 and the sum neither vanishes (all logits
// below -88.7) nor becomes so small that scale / sum overflows.  A row whose
// first is below kRouteMasked, where exp(-first) leaves 64 bits too, is one
// masked by some lowest value: its scores are 0.
constexpr float kRouteMasked = -709.78f;  // -ln of the largest double
__device__ __forceinline__ float route_score(const RouteArgs &p, float v, float first) {
  if (p.sigmoid) {
    if (p.renorm && first < 0.f)
      return first < kRouteMasked ? 0.f : expf(v - first) / (1.0f + expf(v));
    return 1.0f / (1.0f + expf(-v));
  }
  return v == first ? 1.0f : expf(v - first);  // inf - inf is no number
}

// The choice of this block's rows, written out and counted per expert.
template <typename T, int K, int LG>
__device__ __forceinline__ void route_choose(const RouteArgs &p, int r0, int r1, int *count) {
  using R = RouteKey<T>;
  using Key = typename R::Key;
  constexpr int kLanes = 1 << LG, kRowsWarp = 32 >> LG;
  constexpr int kMine = (K + kLanes - 1) / kLanes;  // entries a lane writes
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = lane & (kLanes - 1);
  for (int rb = r0 + warp * kRowsWarp; rb < r1; rb += kRouteWarps * kRowsWarp) {
    const int row = rb + (lane >> LG);
    const bool live = row < r1;
    // lanes of a row that is not there walk the last one
    const T *l = static_cast<const T *>(p.logits) +
                 static_cast<int64_t>(live ? row : r1 - 1) * p.stride;
    Key top[K];
    route_row<T, K, LG>(p, l, sub, top);
    const float first = R::value(top[0]);
    float sum = 0.f;
    if (!p.sigmoid && !p.renorm) {
      const int end = min(p.experts, (sub + 1) * p.per);
      for (int e = sub * p.per; e < end; e += 8) {
        Key k[8];
        R::load8(l, e, p.experts, p.vec, k);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (k[i]) sum += route_score(p, R::value(k[i]), first);
      }
    }
    // the row's lanes share its entries out: entry (i << LG) + sub, by halving
    // the list once per bit of sub
    Key mine[K];
#pragma unroll
    for (int i = 0; i < K; ++i) mine[i] = top[i];
#pragma unroll
    for (int b = 0; b < LG; ++b) {
#pragma unroll
      for (int i = 0; i < (K >> b) / 2; ++i)
        mine[i] = (sub >> b) & 1 ? mine[2 * i + 1] : mine[2 * i];
    }
    float w[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int j = (i << LG) + sub;
      // (a list shorter than the lanes: lanes from K on have no entry)
      if (j >= p.k) mine[i] = 0;
      w[i] = mine[i] ? route_score(p, R::value(mine[i]), first) : 0.f;
      if (p.renorm) sum += w[i];
    }
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    float by = p.scale;
    if (p.renorm || !p.sigmoid) by = sum > 0.f ? p.scale / sum : 0.f;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int j = (i << LG) + sub;
      if (live && j < p.k) {
        const int id = mine[i] ? R::expert(mine[i]) : -1;
        const int64_t at = static_cast<int64_t>(row) * p.k + j;
        p.ids[at] = id;
        p.weights[at] = w[i] * by;
        if (mine[i]) atomicAdd(&count[id], 1);
      }
    }
    __syncwarp();
  }
}

// A row's chosen experts, -1 past the last.
template <int K>
__device__ __forceinline__ void route_ids(const RouteArgs &p, int row, bool live, int (&id)[K]) {
  const int *ids = p.ids + static_cast<int64_t>(row) * p.k;
  if constexpr (K % 4 == 0) {
    if (p.whole) {
#pragma unroll
      for (int j = 0; j < K; j += 4) {
        const int4 v = live ? *reinterpret_cast<const int4 *>(ids + j) : make_int4(-1, -1, -1, -1);
        id[j] = v.x;
        id[j + 1] = v.y;
        id[j + 2] = v.z;
        id[j + 3] = v.w;
      }
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < K; ++j) id[j] = live && j < p.k ? ids[j] : -1;
}

// A row's places.
template <int K>
__device__ __forceinline__ void route_put(const RouteArgs &p, int row, const int (&place)[K]) {
  int *dst = p.row_dst + static_cast<int64_t>(row) * p.k;
  if constexpr (K % 4 == 0) {
    if (p.whole) {
#pragma unroll
      for (int j = 0; j < K; j += 4)
        *reinterpret_cast<int4 *>(dst + j) =
            make_int4(place[j], place[j + 1], place[j + 2], place[j + 3]);
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < K; ++j)
    if (j < p.k) dst[j] = place[j];
}

// The grouped places of this block's rows.  id: the experts of the first
// tiles' rows; start [experts]: the first place of each expert for this
// block; mask, pre [tiles, experts]: scratch.  A warp takes a tile of 32
// rows, a lane a row: bit r of mask[tile][e] says that row
// r of the tile chose e, so an entry's place is its expert's count before the
// tile and the bits below its own -- whatever order the bits were set in.
template <int K>
__device__ __forceinline__ void route_place(const RouteArgs &p, int r0, int r1, int *start,
                                            int *mask, int *pre, int (&id)[K]) {
  const int E = p.experts;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int rb = r0; rb < r1; rb += p.tiles * 32) {
    const int tiles = min(p.tiles, (r1 - rb + 31) / 32);
    for (int i = threadIdx.x; i < tiles * E; i += kRouteThreads) mask[i] = 0;
    __syncthreads();
    const int row = rb + warp * 32 + lane;
    const bool mine = warp < tiles && row < r1;
    if (rb != r0) route_ids<K>(p, row, mine, id);
    if (mine) {
#pragma unroll
      for (int j = 0; j < K; ++j)
        if (id[j] >= 0) atomicOr(&mask[warp * E + id[j]], static_cast<int>(1u << lane));
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += kRouteThreads) {
      int run = start[e];
#pragma unroll 8
      for (int t = 0; t < tiles; ++t) {
        pre[t * E + e] = run;
        run += __popc(mask[t * E + e]);
      }
      start[e] = run;
    }
    __syncthreads();
    if (mine) {
      int place[K];
#pragma unroll
      for (int j = 0; j < K; ++j) {
        place[j] = -1;
        if (id[j] >= 0) {
          place[j] = pre[warp * E + id[j]] + __popc(mask[warp * E + id[j]] & ((1u << lane) - 1u));
          p.row_src[place[j]] = row;
        }
      }
      route_put<K>(p, row, place);
    }
    __syncthreads();
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
template <typename T, int K, int LG>
__global__ void __launch_bounds__(kRouteThreads) route_choose_kernel(const RouteArgs p) {
  __shared__ int count[kRouteMaxExperts];
  for (int e = threadIdx.x; e < p.experts; e += kRouteThreads) count[e] = 0;
  __syncthreads();
  const int rows = route_rows(p);
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * p.block_rows;
  if (r0 < rows)
    route_choose<T, K, LG>(p, static_cast<int>(r0),
                           static_cast<int>(min(static_cast<int64_t>(rows), r0 + p.block_rows)),
                           count);
  __syncthreads();
  for (int e = threadIdx.x; e < p.experts; e += kRouteThreads)
    p.hist[static_cast<int64_t>(blockIdx.x) * p.experts + e] = count[e];
}

// The places: the counts of all blocks give each expert's start and this
// block's start within it.
template <int K>
__global__ void __launch_bounds__(kRouteThreads) route_place_kernel(const RouteArgs p) {
  extern __shared__ int sh[];
  const int E = p.experts;
  int *start = sh, *total = sh + E, *mask = sh + 2 * E, *pre = mask + p.tiles * E;
  const int rows = route_rows(p);
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * p.block_rows;
  const int64_t r1 = min(static_cast<int64_t>(rows), r0 + p.block_rows);
  int id[K];  // on their way while the counts are summed
  const int warp = threadIdx.x >> 5;
  route_ids<K>(p, static_cast<int>(r0) + static_cast<int>(threadIdx.x),
               warp < p.tiles && r0 + threadIdx.x < r1, id);
  for (int e = threadIdx.x; e < 2 * E; e += kRouteThreads) sh[e] = 0;
  __syncthreads();
  // threads share the blocks' counts out among them, expert by expert
  int lanes = 32;
  while (lanes < E && lanes < kRouteThreads) lanes <<= 1;
  for (int e = threadIdx.x & (lanes - 1); e < E; e += lanes) {
    int before = 0, all = 0;
#pragma unroll 8
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
  if (r0 < rows)
    route_place<K>(p, static_cast<int>(r0), static_cast<int>(r1), start, mask, pre, id);
}

// Few rows: one block chooses and places.
template <typename T, int K, int LG>
__global__ void __launch_bounds__(kRouteThreads) route_fused_kernel(const RouteArgs p) {
  extern __shared__ int sh[];
  const int E = p.experts;
  int *start = sh, *total = sh + E, *mask = sh + 2 * E, *pre = mask + p.tiles * E;
  for (int e = threadIdx.x; e < 2 * E; e += kRouteThreads) sh[e] = 0;
  __syncthreads();
  const int rows = route_rows(p);
  if (rows > 0) route_choose<T, K, LG>(p, 0, rows, total);
  __syncthreads();
  route_scan(p, total, start, true);
  __syncthreads();
  int id[K];
  route_ids<K>(p, threadIdx.x, (threadIdx.x >> 5) < p.tiles && threadIdx.x < rows, id);
  route_place<K>(p, 0, rows, start, mask, pre, id);
}

// out[t] = residual[t] + sum_j weights[t, j] * y[row_dst[t, j]], j ascending,
// in fp32 with one rounding at the end; an entry without a place (row_dst
// < 0) adds nothing and is not read.  HBM bounds it: k rows of y are read for
// one written, 120 us at 6.7 TB/s (1.03 of the copy rate) for 32,771 rows of
// 8 x 1024 bf16 onto fp32 rows.
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

// Eight columns of a row as they are stored, and their sum into acc.
template <typename T>
struct CombineVec;
template <>
struct CombineVec<__nv_bfloat16> {
  uint4 u;
  __device__ __forceinline__ void load(const __nv_bfloat16 *y) {
    u = __ldg(reinterpret_cast<const uint4 *>(y));
  }
  __device__ __forceinline__ void zero() { u = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void add(float w, float (&acc)[8]) const {
    const uint32_t v[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      acc[2 * i] = fmaf(w, __uint_as_float(v[i] << 16), acc[2 * i]);
      acc[2 * i + 1] = fmaf(w, __uint_as_float(v[i] & 0xffff0000u), acc[2 * i + 1]);
    }
  }
};
template <>
struct CombineVec<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float *y) {
    a = __ldg(reinterpret_cast<const float4 *>(y));
    b = __ldg(reinterpret_cast<const float4 *>(y) + 1);
  }
  __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void add(float w, float (&acc)[8]) const {
    const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = fmaf(w, v[i], acc[i]);
  }
};

// A row's places and weights, one entry a lane; entries without a place (or
// with a bad one, which is reported) have place -1 and weight 0.
__device__ __forceinline__ void combine_entries(const CombineArgs &p, int64_t row, int lane,
                                                int &at, float &w) {
  at = -1;
  w = 0.f;
  if (lane < p.k) {
    at = __ldg(p.row_dst + row * p.k + lane);
    w = __ldg(p.weights + row * p.k + lane);
    if (at >= p.y_rows) {
      record_err(p.err, kDevBadGroup);
      at = -1;
    }
    if (at < 0) w = 0.f;
  }
}

// A warp takes 256 columns of one row; the entries are read by as many lanes
// at once, and the loads of up to BATCH rows of y are in flight together.
template <typename TY, typename TO, int BATCH>
__global__ void __launch_bounds__(256) moe_combine_kernel(const CombineArgs p, int segments) {
  const int lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int rows = p.rows_dev ? min(p.rows, max(0, __ldg(p.rows_dev))) : p.rows;
  // items fit 32 bits where rows do not need more (checked by the caller)
  const int row = static_cast<int>(static_cast<uint32_t>(item) / static_cast<uint32_t>(segments));
  if (row >= rows) return;
  const int c = (static_cast<int>(item) - row * segments) * 256 + lane * 8;
  int at;
  float w;
  combine_entries(p, row, lane, at, w);
  const bool live = c < p.H;
  float acc[8];
#pragma unroll
  for (int v = 0; v < 8; ++v) acc[v] = 0.f;
  for (int j0 = 0; j0 < p.k; j0 += BATCH) {
    CombineVec<TY> f[BATCH];
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      const int a = __shfl_sync(0xffffffffu, at, j0 + j);  // lanes from k on hold -1
      f[j].zero();
      if (live && a >= 0)
        f[j].load(static_cast<const TY *>(p.y) + static_cast<int64_t>(a) * p.H + c);
    }
#pragma unroll
    for (int j = 0; j < BATCH; ++j) f[j].add(__shfl_sync(0xffffffffu, w, j0 + j), acc);
  }
  if (!live) return;
  const int64_t o = static_cast<int64_t>(row) * p.H + c;
  if (p.residual) {  // not __ldg: residual may be out
    const float4 *r4 = reinterpret_cast<const float4 *>(p.residual + o);
    const float4 a = r4[0], b = r4[1];
    acc[0] += a.x; acc[1] += a.y; acc[2] += a.z; acc[3] += a.w;
    acc[4] += b.x; acc[5] += b.y; acc[6] += b.z; acc[7] += b.w;
  }
  if constexpr (sizeof(TO) == 4) {
    float4 *out = reinterpret_cast<float4 *>(static_cast<float *>(p.out) + o);
    out[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
    out[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
  } else {
    *reinterpret_cast<uint4 *>(static_cast<__nv_bfloat16 *>(p.out) + o) =
        make_uint4(pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3]),
                   pack_bf16x2(acc[4], acc[5]), pack_bf16x2(acc[6], acc[7]));
  }
}

// Any width and alignment, a column a lane.
template <typename TY, typename TO>
__global__ void __launch_bounds__(256) moe_combine_any_kernel(const CombineArgs p) {
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int rows = p.rows_dev ? min(p.rows, max(0, __ldg(p.rows_dev))) : p.rows;
  if (row >= rows) return;
  int at;
  float w;
  combine_entries(p, row, lane, at, w);
  for (int c0 = 0; c0 < p.H; c0 += 32) {
    const int c = c0 + lane;
    float acc = 0.f;
    for (int j = 0; j < p.k; ++j) {
      const int a = __shfl_sync(0xffffffffu, at, j);
      const float wj = __shfl_sync(0xffffffffu, w, j);
      if (a < 0 || c >= p.H) continue;
      const TY *y = static_cast<const TY *>(p.y) + static_cast<int64_t>(a) * p.H + c;
      if constexpr (sizeof(TY) == 4) acc = fmaf(wj, *y, acc);
      else acc = fmaf(wj, __bfloat162float(*y), acc);
    }
    if (c < p.H) {
      const int64_t o = static_cast<int64_t>(row) * p.H + c;
      if (p.residual) acc += p.residual[o];
      if constexpr (sizeof(TO) == 4) static_cast<float *>(p.out)[o] = acc;
      else static_cast<__nv_bfloat16 *>(p.out)[o] = __float2bfloat16_rn(acc);
    }
  }
}

}  // namespace nebw
