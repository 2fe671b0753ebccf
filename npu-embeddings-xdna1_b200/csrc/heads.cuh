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
// operations, so HBM bounds it.  Replayed from a graph: rotation alone 83 us at
// 6.5 TB/s (1.00 of the copy rate) on 65,539 rows of 32 heads of 64, RMS norm
// and rotation 142 us at 5.9 TB/s (0.91) on 49,999 rows of 32 heads of 128; as
// calls among others 89 and 157.  LayerNorm keeps half as
// many warps on an SM and reads at 0.75; heads whose lanes are no power of two
// (80, 96) leave lanes idle, at 0.66 to 0.91.  Sharing a warp's lanes out over
// such heads without a gap was slower (159 against 129 us, heads of 80).
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

#ifdef NEBW_LAYER_KERNELS
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
#endif

// The table row of position `at`.
__device__ __forceinline__ int64_t head_position(const HeadArgs &p, int64_t at) {
  if (at < 0 || at >= p.max_pos) {  // reported; a valid entry is read instead
    record_err(p.err, kDevBadPosition);
    at = at < 0 ? 0 : p.max_pos - 1;
  }
  return at;
}

__device__ __forceinline__ float head_load(const float *p) { return *p; }
__device__ __forceinline__ float head_load(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
__device__ __forceinline__ void head_store(float *p, float v) { *p = v; }
__device__ __forceinline__ void head_store(__nv_bfloat16 *p, float v) {
  *p = __float2bfloat16_rn(v);
}

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
  const float2 *cs = p.n ? p.table + head_position(p, p.pos[row]) * p.n : nullptr;
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

// The same in vectors of V elements, where head_dim is a multiple of two of
// them, n of one, and the rows and weights lie on their boundaries: 16 bytes
// (V = 8 bf16 or 4 fp32), or 8 or 4 for heads of odd widths.  A thread owns V
// pairs of a head: two vectors, at i and n + i of the half layout, adjacent of
// the pairs layout (and of the part that does not turn), so the rotation
// needs no exchange and a norm only the shuffles of the 2^lg lanes that share
// a head.  A warp takes 32 / 2^lg heads of one side of one row at a time, IT
// times: the table entries and the norm's weights are read once for all of
// them, and all loads are issued before the first is used.  IT = 0 is for fewer
// heads than a turn takes: a warp then goes over heads of several rows (18.7
// us against 36.8 for 65,539 rows of 4 + 1 heads of 64).  The arithmetic is
// packed, two values an instruction, which keeps the issue slots below half of
// what the bytes take.
template <int BYTES>
struct HeadWord;
template <>
struct HeadWord<16> {
  using U = uint4;
  static __device__ __forceinline__ void split(const uint4 &u, uint32_t (&w)[4]) {
    w[0] = u.x;
    w[1] = u.y;
    w[2] = u.z;
    w[3] = u.w;
  }
  static __device__ __forceinline__ uint4 join(const uint32_t (&w)[4]) {
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct HeadWord<8> {
  using U = uint2;
  static __device__ __forceinline__ void split(const uint2 &u, uint32_t (&w)[2]) {
    w[0] = u.x;
    w[1] = u.y;
  }
  static __device__ __forceinline__ uint2 join(const uint32_t (&w)[2]) {
    return make_uint2(w[0], w[1]);
  }
};
template <>
struct HeadWord<4> {
  using U = uint32_t;
  static __device__ __forceinline__ void split(const uint32_t &u, uint32_t (&w)[1]) { w[0] = u; }
  static __device__ __forceinline__ uint32_t join(const uint32_t (&w)[1]) { return w[0]; }
};

template <typename T, int V>
struct HeadVec {
  static constexpr int P = V / 2, W = V * static_cast<int>(sizeof(T)) / 4;
  using Word = HeadWord<4 * W>;
  using U = typename Word::U;
  static __device__ __forceinline__ void unpack(const U &u, uint64_t (&f)[P]) {
    uint32_t w[W];
    Word::split(u, w);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      if constexpr (sizeof(T) == 2)
        f[i] = pk2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
      else
        f[i] = pk2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    }
  }
  static __device__ __forceinline__ U pack(const uint64_t (&f)[P]) {
    uint32_t w[W];
#pragma unroll
    for (int i = 0; i < P; ++i) {
      float a, b;
      unpk2(f[i], a, b);
      if constexpr (sizeof(T) == 2) {
        w[i] = pack_bf16x2(a, b);
      } else {
        w[2 * i] = __float_as_uint(a);
        w[2 * i + 1] = __float_as_uint(b);
      }
    }
    return Word::join(w);
  }
};

template <int P>
__device__ __forceinline__ void head_weights(const float *w, uint64_t (&f)[P]) {
  if constexpr (P == 1) {
    const float2 x = __ldg(reinterpret_cast<const float2 *>(w));
    f[0] = pk2(x.x, x.y);
  } else {
#pragma unroll
    for (int i = 0; i < P; i += 2) {
      const float4 x = __ldg(reinterpret_cast<const float4 *>(w + 2 * i));
      f[i] = pk2(x.x, x.y);
      f[i + 1] = pk2(x.z, x.w);
    }
  }
}

// cos and sin of the thread's pair number i from its packed entries.
template <int P>
__device__ __forceinline__ void head_entry(const uint64_t (&c2)[P], const uint64_t (&s2)[P], int i,
                                           float &c, float &s) {
  float lo, hi;
  unpk2(c2[i / 2], lo, hi);
  c = i & 1 ? hi : lo;
  unpk2(s2[i / 2], lo, hi);
  s = i & 1 ? hi : lo;
}

// The weights (and biases) of pair number i, one packed value, folded into its
// rotation: w the factors of the pair itself, x those of the pair with its
// elements exchanged, c the constant part.
template <int P, int NORM>
__device__ __forceinline__ void head_fold_pair(const uint64_t (&c2)[P], const uint64_t (&s2)[P],
                                               int i, uint64_t &w, uint64_t &x, uint64_t &c) {
  float t, u, g0, g1;
  head_entry<P>(c2, s2, i, t, u);
  unpk2(w, g0, g1);
  x = pk2(-g1 * u, g0 * u);
  w = pk2(g0 * t, g1 * t);
  if constexpr (NORM == kHeadNormLayer) {
    float b0, b1;
    unpk2(c, b0, b1);
    c = pk2(fmaf(-b1, u, b0 * t), fmaf(b0, u, b1 * t));
  }
}

// Blocks an SM must hold, which bounds the registers.  Measured (us, at 4 / 3 /
// 2 blocks; 49,999 rows of 16 + 16 heads of 128, bf16, V = 8): no norm 132 /
// 131 / 157 (and 83 / 92 / 92 for 65,539 rows of 32 heads of 64, pairs, a
// quarter of the work), RMS 188 / 144 / 156, LayerNorm 270 / 234 / 173.  Half
// the vector holds half the state: RMS 106 / 115 / 115 (25,000 rows, fp32,
// heads of 96), LayerNorm 141 / 128 / 163 there and 174 / 194 / 198 for bf16
// in 8-byte vectors (heads of 80, turning 40).  The bounds were chosen by time
// and cost some spills with four turns a warp: 48 bytes (half layout) and 20
// (pairs) for bf16 without a norm, 28 and 8 with RMS, 8 for fp32 RMS.
constexpr int head_blocks(int norm, int v, int bytes) {
  if (norm == kHeadNormNone) return 4;
  if (norm == kHeadNormRms) return v < 8 ? 4 : 3;
  return v >= 8 ? 2 : bytes == 16 ? 3 : 4;
}

template <typename T, int V, int NORM, bool PAIRS, int IT>
__global__ void __launch_bounds__(256, head_blocks(NORM, V, V * static_cast<int>(sizeof(T))))
    heads_vec_kernel(const HeadArgs p, int lg, int q_chunks, float inv_dim) {
  using Vec = HeadVec<T, V>;
  using U = typename Vec::U;
  constexpr int P = Vec::P;
  constexpr bool FLAT = IT == 0;
  constexpr int TURNS = FLAT ? 1 : IT;
  const int lane = threadIdx.x & 31;
  int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  int64_t rows = p.rows;
  if (p.rows_dev) rows = min(rows, static_cast<int64_t>(max(0, __ldg(p.rows_dev))));
  const uint32_t item = static_cast<uint32_t>(row) * (32 >> lg);  // FLAT: the warp's first head
  if (!FLAT && row >= rows) return;
  const bool key = static_cast<int>(blockIdx.y) >= q_chunks;
  const int chunk = key ? blockIdx.y - q_chunks : blockIdx.y;
  const T *x = static_cast<const T *>(key ? p.k.x : p.q.x);
  T *out = static_cast<T *>(key ? p.k.out : p.q.out);
  const int heads = key ? p.k.heads : p.q.heads;
  const bool in_place = x == out;
  const int per = 32 >> lg, slot = lane & ((1 << lg) - 1);
  int head0 = chunk * TURNS * per + (lane >> lg);
  const bool turn = slot * V < p.n;
  bool live = slot * 2 * V < p.head_dim;
  if constexpr (FLAT) {
    if (item >= static_cast<uint64_t>(rows) * heads) return;
    row = (item + (lane >> lg)) / static_cast<uint32_t>(heads);
    head0 = static_cast<int>(item + (lane >> lg) - static_cast<uint32_t>(row) * heads);
    if (row >= rows) {  // (row 0 is read in its place)
      live = false;
      row = 0;
    }
  }
  // what does not turn and is not normed stays where it is
  if (NORM == kHeadNormNone && in_place) live = live && turn;
  const int e0 = turn && !PAIRS ? slot * V : slot * 2 * V;
  const int e1 = turn && !PAIRS ? p.n + slot * V : e0 + V;
  x += row * (key ? p.k.stride : p.q.stride) + head0 * p.head_dim;
  out += row * (key ? p.k.out_stride : p.q.out_stride) + head0 * p.head_dim;
  const int hop = per * p.head_dim;  // elements between a lane's heads

  const int pos = turn ? __ldg(p.pos + row) : 0;  // looked at once the rows are on their way
  U ua[TURNS], ub[TURNS];
#pragma unroll
  for (int i = 0; i < TURNS; ++i) {
    ua[i] = ub[i] = U{};
    if (live && head0 + i * per < heads) {
      ua[i] = *reinterpret_cast<const U *>(x + i * hop + e0);
      ub[i] = *reinterpret_cast<const U *>(x + i * hop + e1);
    }
  }
  // cos and sin of the thread's V pairs, two a packed value
  uint64_t c2[P], s2[P];
  if (turn) {
    const float4 *t =
        reinterpret_cast<const float4 *>(p.table + head_position(p, pos) * p.n + slot * V);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const float4 v = __ldg(t + i);
      c2[i] = pk2(v.x, v.z);
      s2[i] = pk2(v.y, v.w);
    }
  }
  // A normed head's weights go into the rotation: with n = x / std (less its
  // mean), a' = n_a (g_a c) - n_b (g_b s) + (b_a c - b_b s), and so for b'.
  // That makes wa, wb the factors of a thread's own elements, xa, xb those of
  // the ones they turn with, ca, cb the constant part.
  uint64_t wa[P], wb[P], xa[P], xb[P], ca[P], cb[P];
  if constexpr (NORM != kHeadNormNone) {
    if (live) {
      const float *g = key ? p.k.gamma : p.q.gamma;
      head_weights<P>(g + e0, wa);
      head_weights<P>(g + e1, wb);
      if constexpr (NORM == kHeadNormLayer) {
        const float *w = key ? p.k.beta : p.q.beta;
        head_weights<P>(w + e0, ca);
        head_weights<P>(w + e1, cb);
      }
      if (turn) {
        if constexpr (PAIRS) {
#pragma unroll
          for (int v = 0; v < P; ++v) {
            head_fold_pair<P, NORM>(c2, s2, v, wa[v], xa[v], ca[v]);
            head_fold_pair<P, NORM>(c2, s2, P + v, wb[v], xb[v], cb[v]);
          }
        } else {
#pragma unroll
          for (int v = 0; v < P; ++v) {
            const uint64_t ns = s2[v] ^ 0x8000000080000000ull;
            xa[v] = mul_x2(wb[v], ns);
            xb[v] = mul_x2(wa[v], s2[v]);
            wa[v] = mul_x2(wa[v], c2[v]);
            wb[v] = mul_x2(wb[v], c2[v]);
            if constexpr (NORM == kHeadNormLayer) {
              const uint64_t a0 = ca[v];
              ca[v] = fma_x2(cb[v], ns, mul_x2(a0, c2[v]));
              cb[v] = fma_x2(a0, s2[v], mul_x2(cb[v], c2[v]));
            }
          }
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < TURNS; ++i) {
    uint64_t a[P], b[P];
    Vec::unpack(ua[i], a);
    Vec::unpack(ub[i], b);
    if constexpr (NORM != kHeadNormNone) {
      if constexpr (NORM == kHeadNormLayer) {
        uint64_t m2 = 0;
#pragma unroll
        for (int v = 0; v < P; ++v) m2 = add_x2(m2, add_x2(a[v], b[v]));
        float mean, m1;
        unpk2(m2, mean, m1);
        mean += m1;
        for (int o = 1; o < 1 << lg; o <<= 1) mean += __shfl_xor_sync(0xffffffffu, mean, o);
        mean *= -inv_dim;
        const uint64_t n2 = live ? pk2(mean, mean) : 0;
#pragma unroll
        for (int v = 0; v < P; ++v) {
          a[v] = add_x2(a[v], n2);
          b[v] = add_x2(b[v], n2);
        }
      }
      uint64_t q2 = 0;
#pragma unroll
      for (int v = 0; v < P; ++v) {
        q2 = fma_x2(a[v], a[v], q2);
        q2 = fma_x2(b[v], b[v], q2);
      }
      float q, q1;
      unpk2(q2, q, q1);
      q += q1;
      for (int o = 1; o < 1 << lg; o <<= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
      const float is = rsqrtf(fmaf(q, inv_dim, p.eps));
      const uint64_t is2 = pk2(is, is);
#pragma unroll
      for (int v = 0; v < P; ++v) {
        uint64_t ya = mul_x2(a[v], wa[v]), yb = mul_x2(b[v], wb[v]);
        if (turn) {
          uint64_t pa = b[v], pb = a[v];  // what they turn with
          if constexpr (PAIRS) {
            float lo, hi;
            unpk2(a[v], lo, hi);
            pa = pk2(hi, lo);
            unpk2(b[v], lo, hi);
            pb = pk2(hi, lo);
          }
          ya = fma_x2(pa, xa[v], ya);
          yb = fma_x2(pb, xb[v], yb);
        }
        if constexpr (NORM == kHeadNormLayer) {
          a[v] = fma_x2(ya, is2, ca[v]);
          b[v] = fma_x2(yb, is2, cb[v]);
        } else {
          a[v] = mul_x2(ya, is2);
          b[v] = mul_x2(yb, is2);
        }
      }
    } else if (turn) {
      if constexpr (PAIRS) {
        // a[v] and b[v] are a pair each, number v and P + v of the thread's
#pragma unroll
        for (int v = 0; v < P; ++v) {
          float c, t, x0, x1;
          head_entry<P>(c2, s2, v, c, t);
          unpk2(a[v], x0, x1);
          a[v] = pk2(fmaf(-x1, t, x0 * c), fmaf(x0, t, x1 * c));
          head_entry<P>(c2, s2, P + v, c, t);
          unpk2(b[v], x0, x1);
          b[v] = pk2(fmaf(-x1, t, x0 * c), fmaf(x0, t, x1 * c));
        }
      } else {
#pragma unroll
        for (int v = 0; v < P; ++v) {
          const uint64_t a0 = a[v], ns = s2[v] ^ 0x8000000080000000ull;
          a[v] = fma_x2(b[v], ns, mul_x2(a0, c2[v]));
          b[v] = fma_x2(a0, s2[v], mul_x2(b[v], c2[v]));
        }
      }
    }
    if (live && head0 + i * per < heads) {
      *reinterpret_cast<U *>(out + i * hop + e0) = Vec::pack(a);
      *reinterpret_cast<U *>(out + i * hop + e1) = Vec::pack(b);
    }
  }
}

}  // namespace nebw
