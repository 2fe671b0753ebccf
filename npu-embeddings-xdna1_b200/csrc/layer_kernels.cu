// The kernels of rotary and expert layers and the choice among their variants:
// one translation unit, launched through layer_kernels.h.
#define NEBW_LAYER_KERNELS  // ptx.cuh and rowops.cuh leave out their own kernels

#include "layer_kernels.h"

namespace nebw {
namespace {

bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// ---------------------------------------------------------------------------
// heads
// ---------------------------------------------------------------------------

template <typename T, int V, int NORM, bool PAIRS, int IT>
void launch_heads_it(const HeadArgs &a, int lg, int per, cudaStream_t st) {
  int q_chunks, chunks;
  int64_t warps = a.rows;
  if constexpr (IT == 0) {  // heads of all rows in one list a side
    q_chunks = a.q.heads > 0;
    chunks = q_chunks + (a.k.heads > 0);
    warps = (a.rows * std::max(a.q.heads, a.k.heads) + per - 1) / per;
  } else {
    q_chunks = (a.q.heads + per * IT - 1) / (per * IT);
    chunks = q_chunks + (a.k.heads + per * IT - 1) / (per * IT);
  }
  const dim3 grid(static_cast<unsigned>((warps + 7) / 8), chunks);
  heads_vec_kernel<T, V, NORM, PAIRS, IT>
      <<<grid, 256, 0, st>>>(a, lg, q_chunks, 1.0f / static_cast<float>(a.head_dim));
}

bool heads_vec_side(const HeadSide &s, size_t esz, int v) {
  const size_t bytes = v * esz, weights = std::min<size_t>(16, v * sizeof(float));
  return aligned(s.x, bytes) && aligned(s.out, bytes) && s.stride * esz % bytes == 0 &&
         s.out_stride * esz % bytes == 0 && aligned(s.gamma, weights) && aligned(s.beta, weights);
}

// Whether vectors of v elements fit the heads (and a head a warp).
bool heads_vec_fit(const HeadArgs &a, size_t esz, int v) {
  return a.head_dim % (2 * v) == 0 && a.head_dim <= 64 * v && a.n % v == 0 &&
         heads_vec_side(a.q, esz, v) && heads_vec_side(a.k, esz, v);
}

template <typename T, int V, int NORM, bool PAIRS>
void launch_heads_vec(const HeadArgs &a, cudaStream_t st) {
  int lg = 0;  // lanes a head
  while ((2 * V << lg) < a.head_dim) ++lg;
  const int per = 32 >> lg;  // heads a warp takes at once
  if constexpr (V * sizeof(T) == 16) {
    // four turns a warp share its table entries and weights (144 us against
    // 170 for two, on the RMS case at heads_vec_kernel); one or two where the
    // heads end there
    const int most = std::max(a.q.heads, a.k.heads);
    if (most < per && a.rows * most < (1ll << 31))
      return launch_heads_it<T, V, NORM, PAIRS, 0>(a, lg, per, st);
    if (most <= per) return launch_heads_it<T, V, NORM, PAIRS, 1>(a, lg, per, st);
    if (most <= 2 * per) return launch_heads_it<T, V, NORM, PAIRS, 2>(a, lg, per, st);
  }
  return launch_heads_it<T, V, NORM, PAIRS, 4>(a, lg, per, st);
}

// The blocks of heads_any_kernel.
int64_t heads_any_blocks(const HeadArgs &a) { return (a.rows * (a.q.heads + a.k.heads) + 7) / 8; }

// The vectors' elements, or 0 for heads that no vectors fit.
template <typename T>
int heads_vec(const HeadArgs &a) {
  constexpr int V = 16 / sizeof(T);
  if (heads_vec_fit(a, sizeof(T), V)) return V;
  if (sizeof(T) == 2 && heads_vec_fit(a, sizeof(T), 4)) return 4;
  return heads_vec_fit(a, sizeof(T), 2) ? 2 : 0;
}

template <typename T, int NORM, bool PAIRS>
void launch_heads_of(const HeadArgs &a, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const int v = heads_vec<T>(a);
  if (v == V) return launch_heads_vec<T, V, NORM, PAIRS>(a, st);
  if constexpr (sizeof(T) == 2)
    if (v == 4) return launch_heads_vec<T, 4, NORM, PAIRS>(a, st);
  if (v == 2) return launch_heads_vec<T, 2, NORM, PAIRS>(a, st);
  heads_any_kernel<T, NORM, PAIRS>
      <<<static_cast<unsigned>(heads_any_blocks(a)), 256, 0, st>>>(a);
}

template <typename T, int NORM>
void launch_heads_layout(const HeadArgs &a, bool pairs, cudaStream_t st) {
  if (pairs) launch_heads_of<T, NORM, true>(a, st);
  else launch_heads_of<T, NORM, false>(a, st);
}

template <typename T>
void launch_heads_norm(const HeadArgs &a, int norm, bool pairs, cudaStream_t st) {
  switch (norm) {
    case kHeadNormRms: return launch_heads_layout<T, kHeadNormRms>(a, pairs, st);
    case kHeadNormLayer: return launch_heads_layout<T, kHeadNormLayer>(a, pairs, st);
    default: return launch_heads_layout<T, kHeadNormNone>(a, pairs, st);
  }
}

// ---------------------------------------------------------------------------
// routing
// ---------------------------------------------------------------------------

size_t route_smem(int experts) {
  return (2 + 2 * static_cast<size_t>(route_tiles(experts))) * experts * sizeof(int);
}

// A kernel's room for more than the 48 KB that every kernel has, once: `bit` is
// the kernel's own.
template <typename Kernel>
cudaError_t route_room(Kernel *kernel, size_t smem, std::atomic<uint32_t> &ready, int bit) {
  if (smem <= 48 * 1024 || ready.load(std::memory_order_acquire) >> bit & 1u) return cudaSuccess;
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRouteSmem);
  if (e == cudaSuccess) ready.fetch_or(1u << bit, std::memory_order_release);
  return e;
}

template <typename T, int K, int LG>
cudaError_t launch_route_lg(const RouteArgs &a, int blocks, std::atomic<uint32_t> &ready,
                            cudaStream_t st) {
  const size_t smem = route_smem(a.experts);
  // five kernels for each of the five list lengths 1, 2, 4, 8, 16
  constexpr int kBit = 5 * (K >= 16 ? 4 : K >= 8 ? 3 : K / 2);
  if (blocks == 0) {
    constexpr int kOwn = kBit + (sizeof(T) == 4 ? 0 : 2) + (LG ? 1 : 0);
    if (cudaError_t e = route_room(route_fused_kernel<T, K, LG>, smem, ready, kOwn)) return e;
    route_fused_kernel<T, K, LG><<<1, kRouteThreads, smem, st>>>(a);
  } else {
    if (cudaError_t e = route_room(route_place_kernel<K>, smem, ready, kBit + 4)) return e;
    route_choose_kernel<T, K, LG><<<blocks, kRouteThreads, 0, st>>>(a);
    if (cudaError_t e = cudaGetLastError()) return e;
    route_place_kernel<K><<<blocks, kRouteThreads, smem, st>>>(a);
  }
  return cudaGetLastError();
}

// Four lanes a row from three eights of experts on, else one.
template <typename T, int K>
cudaError_t launch_route_of(RouteArgs a, int blocks, std::atomic<uint32_t> &ready,
                            cudaStream_t st) {
  const int eights = (a.experts + 7) / 8;
  if (eights < 3) {
    a.per = eights * 8;
    return launch_route_lg<T, K, 0>(a, blocks, ready, st);
  }
  a.per = (eights + 3) / 4 * 8;
  return launch_route_lg<T, K, 2>(a, blocks, ready, st);
}

// The list a lane keeps: the next power of two of top_k.
template <typename T>
cudaError_t launch_route_k(const RouteArgs &a, int blocks, std::atomic<uint32_t> &ready,
                           cudaStream_t st) {
  if (a.k == 1) return launch_route_of<T, 1>(a, blocks, ready, st);
  if (a.k == 2) return launch_route_of<T, 2>(a, blocks, ready, st);
  if (a.k <= 4) return launch_route_of<T, 4>(a, blocks, ready, st);
  if (a.k <= 8) return launch_route_of<T, 8>(a, blocks, ready, st);
  return launch_route_of<T, 16>(a, blocks, ready, st);
}

// ---------------------------------------------------------------------------
// grouped products and the combine
// ---------------------------------------------------------------------------

template <int EPI>
cudaError_t set_grouped_attr() {
  const auto a = cudaFuncAttributeMaxDynamicSharedMemorySize;
  const int smem = GroupedShape::kSmemBytes;
  if (cudaError_t e = cudaFuncSetAttribute(gemm_grouped_kernel<EPI, false>, a, smem)) return e;
  return cudaFuncSetAttribute(gemm_grouped_kernel<EPI, true>, a, smem);
}

template <int EPI>
void launch_grouped_epi(const GroupedMaps &m, const GroupedArgs &a, unsigned grid,
                        cudaStream_t st) {
  const size_t smem = GroupedShape::kSmemBytes;
  if (a.row_src)
    gemm_grouped_kernel<EPI, true>
        <<<grid, kGroupedGatherThreads, smem, st>>>(m.a, m.a128, m.w, m.c, a);
  else
    gemm_grouped_kernel<EPI, false>
        <<<grid, kGroupedThreads, smem, st>>>(m.a, m.a128, m.w, m.c, a);
}

template <typename TY, typename TO>
void launch_combine_of(const CombineArgs &a, bool vec, cudaStream_t st) {
  const int segments = (a.H + 255) / 256;
  const int64_t items = static_cast<int64_t>(a.rows) * segments;
  if (vec && items < (1ll << 31)) {
    const unsigned g = static_cast<unsigned>((items + 7) / 8);
    if (a.k > 4) moe_combine_kernel<TY, TO, 8><<<g, 256, 0, st>>>(a, segments);
    else if (a.k > 2) moe_combine_kernel<TY, TO, 4><<<g, 256, 0, st>>>(a, segments);
    else moe_combine_kernel<TY, TO, 2><<<g, 256, 0, st>>>(a, segments);
  } else {
    moe_combine_any_kernel<TY, TO>
        <<<static_cast<unsigned>((static_cast<int64_t>(a.rows) + 7) / 8), 256, 0, st>>>(a);
  }
}

}  // namespace

cudaError_t launch_rope_table(const double *inv_freq, int n, int64_t max_pos, double scale,
                              float2 *table, cudaStream_t st) {
  const int64_t entries = max_pos * n;
  rope_table_kernel<<<static_cast<unsigned>((entries + 255) / 256), 256, 0, st>>>(
      inv_freq, n, max_pos, scale, table);
  return cudaGetLastError();
}

bool heads_fit(const HeadArgs &a, bool f32) {
  return (f32 ? heads_vec<float>(a) : heads_vec<__nv_bfloat16>(a)) ||
         heads_any_blocks(a) < (1ll << 31);
}

cudaError_t launch_heads(const HeadArgs &a, bool f32, int norm, bool pairs, cudaStream_t st) {
  if (f32) launch_heads_norm<float>(a, norm, pairs, st);
  else launch_heads_norm<__nv_bfloat16>(a, norm, pairs, st);
  return cudaGetLastError();
}

cudaError_t launch_route(const RouteArgs &a, bool f32, int blocks, std::atomic<uint32_t> &ready,
                         cudaStream_t st) {
  return f32 ? launch_route_k<float>(a, blocks, ready, st)
             : launch_route_k<__nv_bfloat16>(a, blocks, ready, st);
}

cudaError_t launch_stage_experts(const void *src, bool bf16, int64_t K, int64_t N, bool gated,
                                 int e0, int count, __nv_bfloat16 *dst, cudaStream_t st) {
  const int cb = static_cast<int>((N + 255) / 256 * 2), kb = static_cast<int>((K + 63) / 64);
  stage_experts_kernel<<<dim3(cb * 4, kb * 2, count), dim3(32, 8), 0, st>>>(
      src, bf16, static_cast<int>(K), static_cast<int>(N), gated, e0, cb, kb, dst);
  return cudaGetLastError();
}

cudaError_t ready_grouped(int *pairs) {
  if (cudaError_t e = set_grouped_attr<kGrpBf16>()) return e;
  if (cudaError_t e = set_grouped_attr<kGrpBf16Gelu8>()) return e;
  if (cudaError_t e = set_grouped_attr<kGrpBf16Erf>()) return e;
  if (cudaError_t e = set_grouped_attr<kGrpF32>()) return e;
  if (cudaError_t e = set_grouped_attr<kGrpBf16SwiGLU>()) return e;
  if (cudaError_t e = set_grouped_attr<kGrpBf16GeGLU>()) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * 74);
  cfg.blockDim = dim3(kGroupedGatherThreads);
  cfg.dynamicSmemBytes = GroupedShape::kSmemBytes;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 2;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaOccupancyMaxActiveClusters(pairs, gemm_grouped_kernel<kGrpBf16, true>, &cfg);
}

cudaError_t launch_grouped(const GroupedMaps &m, int epi, const GroupedArgs &a, unsigned grid,
                           cudaStream_t st) {
  switch (epi) {
    case kGrpBf16: launch_grouped_epi<kGrpBf16>(m, a, grid, st); break;
    case kGrpBf16Gelu8: launch_grouped_epi<kGrpBf16Gelu8>(m, a, grid, st); break;
    case kGrpBf16Erf: launch_grouped_epi<kGrpBf16Erf>(m, a, grid, st); break;
    case kGrpF32: launch_grouped_epi<kGrpF32>(m, a, grid, st); break;
    case kGrpBf16SwiGLU: launch_grouped_epi<kGrpBf16SwiGLU>(m, a, grid, st); break;
    case kGrpBf16GeGLU: launch_grouped_epi<kGrpBf16GeGLU>(m, a, grid, st); break;
  }
  return cudaGetLastError();
}

cudaError_t launch_combine(const CombineArgs &a, bool y_f32, bool out_f32, bool vec,
                           cudaStream_t st) {
  if (y_f32) {
    if (out_f32) launch_combine_of<float, float>(a, vec, st);
    else launch_combine_of<float, __nv_bfloat16>(a, vec, st);
  } else {
    if (out_f32) launch_combine_of<__nv_bfloat16, float>(a, vec, st);
    else launch_combine_of<__nv_bfloat16, __nv_bfloat16>(a, vec, st);
  }
  return cudaGetLastError();
}

}  // namespace nebw
