// The launches of the kernels of rotary and expert layers (layer_kernels.cu),
// for layer_ops.cuh.  They are a translation unit of their own so that the
// driver loads their code when the first of them is called: in one with the
// encoder passes they made the first nebw_open of a process 34 ms instead of
// 20.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>

#include "gemm_grouped.cuh"
#include "heads.cuh"
#include "moe.cuh"

namespace nebw {

cudaError_t launch_rope_table(const double *inv_freq, int n, int64_t max_pos, double scale,
                              float2 *table, cudaStream_t st);

// Whether a launch covers the heads (of fp32 or bf16 elements).
bool heads_fit(const HeadArgs &a, bool f32);
cudaError_t launch_heads(const HeadArgs &a, bool f32, int norm, bool pairs, cudaStream_t st);

// Shared memory of the placing kernels: starts and totals, and the row masks
// and counts of as many tiles of 32 rows as fit beside them (one a warp at
// most).
constexpr int kRouteSmem = 100 * 1024;
inline int route_tiles(int experts) {
  const int fit = (kRouteSmem / (experts * static_cast<int>(sizeof(int))) - 2) / 2;
  return std::min(fit, kRouteWarps);
}
// blocks 0: one block chooses and places.  ready: a bit a kernel, of the device
// that is current.
cudaError_t launch_route(const RouteArgs &a, bool f32, int blocks, std::atomic<uint32_t> &ready,
                         cudaStream_t st);

// `count` experts of src [count, K, N] from number e0 on.
cudaError_t launch_stage_experts(const void *src, bool bf16, int64_t K, int64_t N, bool gated,
                                 int e0, int count, __nv_bfloat16 *dst, cudaStream_t st);

struct GroupedMaps {
  CUtensorMap a, a128, w, c;
};
// The kernels' shared memory on the current device, and how many CTA pairs of
// the grouped product it holds at once (none: the product is refused, the rest
// of the library works).
cudaError_t ready_grouped(int *pairs);
cudaError_t launch_grouped(const GroupedMaps &m, int epi, const GroupedArgs &a, unsigned grid,
                           cudaStream_t st);

cudaError_t launch_combine(const CombineArgs &a, bool y_f32, bool out_f32, bool vec,
                           cudaStream_t st);

}  // namespace nebw
