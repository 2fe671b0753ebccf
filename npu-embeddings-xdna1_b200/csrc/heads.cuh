// Query and key heads of packed rows: rotary positions, and a norm of every
// head with the rotation in the same pass.
//
// Row r's head h is head_dim elements at x + r * stride + h * head_dim.  With
// n = rot_dim / 2 frequencies, the pair i of a head at position p turns by
// the angle t = p * inv_freq[i]:
//
//   a' = a cos t - b sin t,   b' = b cos t + a sin t
//
//   half   a = element i, b = element n + i
//   pairs  a = element 2i, b = element 2i + 1
//
// and the elements from 2n on stay as they are.  cos and sin come from a
// table [max_pos, n] of float2 made in double when the frequencies are staged
// (a position of 10^5 times a frequency near 1 keeps no fraction in fp32).
// The norm before it is y = x * rms(x)^-1 * gamma, or LayerNorm's two-pass
// (x - mean) * std^-1 * gamma + beta, over the head, in fp32; there is one
// rounding, of the rotated value, at the end.
//
// Each element is read once and written once and takes a handful of fp32
// operations, so HBM bounds it.
#pragma once

#include <cuda_bf16.h>
#include <cstdint>

#include "ptx.cuh"
#include "rowops.cuh"

namespace nebw {

enum HeadNorm : int { kHeadNormNone = 0, kHeadNormRms = 1, kHeadNormLayer = 2 };

struct HeadSide {      // the query or the key heads
  const void *x;
  void *out;           // == x (in place) or elsewhere
  int64_t stride, out_stride;  // elements between rows
  int heads;
  const float *gamma, *beta;   // [head_dim]; beta LayerNorm only
};

struct HeadArgs {
  HeadSide q, k;
  int64_t rows;
  const int *rows_dev;  // if set, the live row count is min(*rows_dev, rows)
  int head_dim, n;      // n = rot_dim / 2 (0: no rotation)
  const float2 *table;  // [max_pos, n] (cos, sin)
  int64_t max_pos;
  const int *pos;       // [rows]
  float eps;
  int *err;
};

// cos and sin of every position and frequency, in double, scaled and rounded
// once.
__global__ void __launch_bounds__(256)
    rope_table_kernel(const double *__restrict__ inv_freq, int n, int64_t max_pos, double scale,
                      float2 *__restrict__ table) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= max_pos * n) return;
  const int64_t p = i / n;
  double s, c;
  sincos(static_cast<double>(p) * inv_freq[i - p * n], &s, &c);
  table[i] = make_float2(static_cast<float>(c * scale), static_cast<float>(s * scale));
}

__device__ __forceinline__ int64_t head_position(const HeadArgs &p, int64_t row) {
  int64_t at = p.pos[row];
  if (at < 0 || at >= p.max_pos) {  // reported; a valid entry is read instead
    record_err(p.err, kDevBadPosition);
    at = at < 0 ? 0 : p.max_pos - 1;
  }
  return at;
}

__device__ __forceinline__ float head_load(const float *p) { return *p; }
__device__ __forceinline__ float head_load(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
__device__ __forceinline__ void head_store(float *p, float v) { *p = v; }
__device__ __forceinline__ void head_store(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

// Any even head_dim up to 256 and any even rot_dim, elements one by one: a
// warp per head, up to four pairs a lane.
constexpr int kHeadMaxDim = 256;

template <typename T, int NORM, bool PAIRS>
__global__ void __launch_bounds__(256) heads_any_kernel(const HeadArgs p) {
  const int lane = threadIdx.x & 31;
  const int heads = p.q.heads + p.k.heads;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int64_t row = item / heads;
  int64_t rows = p.rows;
  if (p.rows_dev) rows = min(rows, static_cast<int64_t>(max(0, __ldg(p.rows_dev))));
  if (row >= rows) return;
  const int h = static_cast<int>(item - row * heads);
  const bool key = h >= p.q.heads;
  const HeadSide &side = key ? p.k : p.q;
  const int64_t hh = key ? h - p.q.heads : h;
  const T *x = static_cast<const T *>(side.x) + row * side.stride + hh * p.head_dim;
  T *out = static_cast<T *>(side.out) + row * side.out_stride + hh * p.head_dim;
  const float2 *cs = p.n ? p.table + head_position(p, row) * p.n : nullptr;
  constexpr int kMax = kHeadMaxDim / 64;  // pairs a lane
  const int half = p.head_dim / 2;
  float a[kMax], b[kMax];
  int ia[kMax], ib[kMax];
#pragma unroll
  for (int i = 0; i < kMax; ++i) {
    const int s = lane + 32 * i;
    const bool turn = s < p.n;
    ia[i] = turn ? (PAIRS ? 2 * s : s) : 2 * s;
    ib[i] = turn ? (PAIRS ? 2 * s + 1 : p.n + s) : 2 * s + 1;
    a[i] = s < half ? head_load(x + ia[i]) : 0.f;
    b[i] = s < half ? head_load(x + ib[i]) : 0.f;
  }
  if constexpr (NORM != kHeadNormNone) {
    float mean = 0.f;
    if constexpr (NORM == kHeadNormLayer) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < kMax; ++i) s += a[i] + b[i];
      mean = warp_sum(s) / static_cast<float>(p.head_dim);
    }
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < kMax; ++i) {
      if (lane + 32 * i < half) {
        a[i] -= mean;
        b[i] -= mean;
        q = fmaf(a[i], a[i], q);
        q = fmaf(b[i], b[i], q);
      }
    }
    const float is = 1.0f / sqrtf(warp_sum(q) / static_cast<float>(p.head_dim) + p.eps);
#pragma unroll
    for (int i = 0; i < kMax; ++i) {
      if (lane + 32 * i < half) {
        a[i] = a[i] * is * __ldg(side.gamma + ia[i]);
        b[i] = b[i] * is * __ldg(side.gamma + ib[i]);
        if constexpr (NORM == kHeadNormLayer) {
          a[i] += __ldg(side.beta + ia[i]);
          b[i] += __ldg(side.beta + ib[i]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kMax; ++i) {
    const int s = lane + 32 * i;
    if (s >= half) continue;
    if (s < p.n) {
      const float2 t = __ldg(cs + s);
      head_store(out + ia[i], fmaf(-b[i], t.y, a[i] * t.x));
      head_store(out + ib[i], fmaf(a[i], t.y, b[i] * t.x));
    } else {
      head_store(out + ia[i], a[i]);
      head_store(out + ib[i], b[i]);
    }
  }
}

// The same with 16-byte accesses, where head_dim and rot_dim are multiples of
// two vectors (V = 8 bf16 or 4 fp32 elements) and the rows and weights lie on
// 16-byte boundaries.  A thread owns V pairs of a head: two vectors, at i and
// n + i of the half layout, adjacent of the pairs layout (and of the part
// that does not turn), so the rotation needs no exchange and a norm only the
// shuffles of the 2^lg lanes that share a head.  A warp takes 32 / 2^lg heads
// of one side of one row at a time, IT times: the table entries and the
// norm's weights are read once for all of them, and all loads are issued
// before the first is used.
template <typename T>
struct HeadVec;
template <>
struct HeadVec<__nv_bfloat16> {
  static constexpr int V = 8;
  static __device__ __forceinline__ void unpack(const uint4 &u, float (&f)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                      pack_bf16x2(f[6], f[7]));
  }
};
template <>
struct HeadVec<float> {
  static constexpr int V = 4;
  static __device__ __forceinline__ void unpack(const uint4 &u, float (&f)[4]) {
    f[0] = __uint_as_float(u.x);
    f[1] = __uint_as_float(u.y);
    f[2] = __uint_as_float(u.z);
    f[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                      __float_as_uint(f[3]));
  }
};

template <int V>
__device__ __forceinline__ void head_weights(const float *w, float (&f)[V]) {
#pragma unroll
  for (int i = 0; i < V; i += 4) {
    const float4 x = __ldg(reinterpret_cast<const float4 *>(w + i));
    f[i] = x.x;
    f[i + 1] = x.y;
    f[i + 2] = x.z;
    f[i + 3] = x.w;
  }
}

template <typename T, int NORM, bool PAIRS, int IT>
__global__ void __launch_bounds__(256)
    heads_vec_kernel(const HeadArgs p, int lg, int q_chunks, int chunks) {
  constexpr int V = HeadVec<T>::V;
  const int lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int64_t row = item / chunks;
  int64_t rows = p.rows;
  if (p.rows_dev) rows = min(rows, static_cast<int64_t>(max(0, __ldg(p.rows_dev))));
  if (row >= rows) return;
  int chunk = static_cast<int>(item - row * chunks);
  const bool key = chunk >= q_chunks;
  if (key) chunk -= q_chunks;
  const T *x = static_cast<const T *>(key ? p.k.x : p.q.x);
  T *out = static_cast<T *>(key ? p.k.out : p.q.out);
  const int heads = key ? p.k.heads : p.q.heads;
  const bool in_place = x == out;
  x += row * (key ? p.k.stride : p.q.stride);
  out += row * (key ? p.k.out_stride : p.q.out_stride);

  const int per = 32 >> lg, slot = lane & ((1 << lg) - 1);
  const int head0 = chunk * IT * per + (lane >> lg);
  const bool turn = slot * V < p.n;
  bool live = slot * 2 * V < p.head_dim;
  // what does not turn and is not normed stays where it is
  if (NORM == kHeadNormNone && in_place) live = live && turn;
  const int e0 = turn && !PAIRS ? slot * V : slot * 2 * V;
  const int e1 = turn && !PAIRS ? p.n + slot * V : e0 + V;

  uint4 ua[IT], ub[IT];
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int h = head0 + i * per;
    ua[i] = ub[i] = make_uint4(0, 0, 0, 0);
    if (live && h < heads) {
      ua[i] = *reinterpret_cast<const uint4 *>(x + h * p.head_dim + e0);
      ub[i] = *reinterpret_cast<const uint4 *>(x + h * p.head_dim + e1);
    }
  }
  float c[V], s[V];  // of the thread's pairs
  if (turn) {
    const float4 *t =
        reinterpret_cast<const float4 *>(p.table + head_position(p, row) * p.n + slot * V);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float4 v = __ldg(t + i);
      c[2 * i] = v.x;
      s[2 * i] = v.y;
      c[2 * i + 1] = v.z;
      s[2 * i + 1] = v.w;
    }
  }
  float ga[V], gb[V], ba[V], bb[V];
  if constexpr (NORM != kHeadNormNone) {
    if (live) {
      const float *g = key ? p.k.gamma : p.q.gamma;
      head_weights<V>(g + e0, ga);
      head_weights<V>(g + e1, gb);
      if constexpr (NORM == kHeadNormLayer) {
        const float *b = key ? p.k.beta : p.q.beta;
        head_weights<V>(b + e0, ba);
        head_weights<V>(b + e1, bb);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    float a[V], b[V];
    HeadVec<T>::unpack(ua[i], a);
    HeadVec<T>::unpack(ub[i], b);
    if constexpr (NORM != kHeadNormNone) {
      float mean = 0.f;
      if constexpr (NORM == kHeadNormLayer) {
#pragma unroll
        for (int v = 0; v < V; ++v) mean += a[v] + b[v];
        for (int o = 1; o < 1 << lg; o <<= 1) mean += __shfl_xor_sync(0xffffffffu, mean, o);
        mean /= static_cast<float>(p.head_dim);
      }
      float q = 0.f;
      if (live) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          a[v] -= mean;
          b[v] -= mean;
          q = fmaf(a[v], a[v], q);
          q = fmaf(b[v], b[v], q);
        }
      }
      for (int o = 1; o < 1 << lg; o <<= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
      const float is = 1.0f / sqrtf(q / static_cast<float>(p.head_dim) + p.eps);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if constexpr (NORM == kHeadNormLayer) {
          a[v] = fmaf(a[v] * is, ga[v], ba[v]);
          b[v] = fmaf(b[v] * is, gb[v], bb[v]);
        } else {
          a[v] = a[v] * is * ga[v];
          b[v] = b[v] * is * gb[v];
        }
      }
    }
    if (turn) {
      if constexpr (PAIRS) {
#pragma unroll
        for (int v = 0; v < V; v += 2) {
          const float a0 = a[v], b0 = b[v];
          a[v] = fmaf(-a[v + 1], s[v / 2], a0 * c[v / 2]);
          a[v + 1] = fmaf(a0, s[v / 2], a[v + 1] * c[v / 2]);
          b[v] = fmaf(-b[v + 1], s[(V + v) / 2], b0 * c[(V + v) / 2]);
          b[v + 1] = fmaf(b0, s[(V + v) / 2], b[v + 1] * c[(V + v) / 2]);
        }
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float a0 = a[v];
          a[v] = fmaf(-b[v], s[v], a0 * c[v]);
          b[v] = fmaf(a0, s[v], b[v] * c[v]);
        }
      }
    }
    const int h = head0 + i * per;
    if (live && h < heads) {
      *reinterpret_cast<uint4 *>(out + h * p.head_dim + e0) = HeadVec<T>::pack(a);
      *reinterpret_cast<uint4 *>(out + h * p.head_dim + e1) = HeadVec<T>::pack(b);
    }
  }
}

}  // namespace nebw
