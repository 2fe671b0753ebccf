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

}  // namespace nebw
