// The operators of rotary and expert encoder layers, C ABI part of
// include/nebw.h: rotary positions, per-head norms, expert routing, grouped
// products and the combine.  This file is part of the nebw.cu translation
// unit (included at its end): it uses that file's device handle, tensor maps
// and error reporting.  The kernels' launches are in layer_kernels.cu.  None of
// these has a counterpart in the reference.

namespace {

bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Arrays of 4-byte values (or null), which kernels read and write whole.
template <typename... P>
bool words(const P *...p) {
  return (aligned(p, 4) && ...);
}

// Whether two pieces of memory (na, nb bytes) meet.
bool meet(const void *a, int64_t na, const void *b, int64_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return na > 0 && nb > 0 && x < y + nb && y < x + na;
}

// Whether any two rows of two blocks of `rows` rows meet: wa and wb bytes a
// row, sa and sb from one to the next.  Blocks of one stride may interleave
// (Q and K of Q|K|V rows); blocks of two strides that reach into one another
// are taken to be apart.
bool rows_meet(const void *a, int64_t sa, int64_t wa, const void *b, int64_t sb, int64_t wb,
               int64_t rows) {
  if (rows <= 1) return meet(a, wa, b, wb);
  if (sa != sb) return false;
  // row i of b lies d bytes behind row i + by of a, and before the next one
  const int64_t off = static_cast<int64_t>(reinterpret_cast<uintptr_t>(b) -
                                           reinterpret_cast<uintptr_t>(a));
  int64_t by = off / sa, d = off % sa;
  if (d < 0) {
    --by;
    d += sa;
  }
  return (d < wa && std::abs(by) < rows) || (d + wb > sa && std::abs(by + 1) < rows);
}

// Host or this device's memory; *on_device says which.
int where_is(nebw_dev *d, const void *p, bool *on_device) {
  cudaPointerAttributes a;
  NEBW_CUDA(cudaPointerGetAttributes(&a, p));
  *on_device = a.type == cudaMemoryTypeDevice || a.type == cudaMemoryTypeManaged;
  NEBW_REQUIRE(a.type != cudaMemoryTypeDevice || a.device == d->device,
               "the data is on device %d, the handle on device %d", a.device, d->device);
  return NEBW_OK;
}

// The grouped product's kernels, once a handle (when experts are staged).
int ready_grouped(nebw_dev *d) {
  std::lock_guard<std::mutex> lock(d->staged);
  if (d->grouped_ready) return NEBW_OK;
  NEBW_CUDA(nebw::ready_grouped(&d->grouped_pairs));
  d->grouped_ready = true;
  return NEBW_OK;
}

}  // namespace

// ---------------------------------------------------------------------------
// rotary positions and per-head norms
// ---------------------------------------------------------------------------

extern "C" int nebw_rope_freqs(double theta, int32_t rot_dim, const nebw_rope_scaling *s,
                               double *inv_freq, double *scale) {
  NEBW_REQUIRE(inv_freq && scale, "null frequency output");
  NEBW_REQUIRE(rot_dim >= 2 && rot_dim % 2 == 0 && rot_dim <= nebw::kHeadMaxDim,
               "rotary width %d refused: even, 2 .. %d", rot_dim, nebw::kHeadMaxDim);
  NEBW_REQUIRE(theta > 1.0 && std::isfinite(theta), "rotary base %g refused", theta);
  const int n = rot_dim / 2;
  const int kind = s ? s->kind : NEBW_ROPE_PLAIN;
  *scale = 1.0;
  if (kind != NEBW_ROPE_PLAIN) {
    NEBW_REQUIRE(kind == NEBW_ROPE_LINEAR || kind == NEBW_ROPE_NTK || kind == NEBW_ROPE_YARN ||
                     kind == NEBW_ROPE_BANDS,
                 "rotary scaling %d refused", kind);
    NEBW_REQUIRE(s->factor >= 1.0 && std::isfinite(s->factor), "rotary factor %g refused: >= 1",
                 s->factor);
  }
  const bool trained = kind == NEBW_ROPE_YARN || kind == NEBW_ROPE_BANDS;
  double fast = 0.0, slow = 0.0;
  if (trained) {
    NEBW_REQUIRE(s->orig_len > 0, "this rotary scaling needs the trained length");
    fast = s->fast > 0.0 ? s->fast : kind == NEBW_ROPE_YARN ? 32.0 : 4.0;
    slow = s->slow > 0.0 ? s->slow : 1.0;
    NEBW_REQUIRE(fast > slow, "rotary bounds refused: fast %g must be above slow %g", fast, slow);
  }
  constexpr double kTwoPi = 6.283185307179586476925;
  double base = theta;
  if (kind == NEBW_ROPE_NTK) base = n > 1 ? theta * std::pow(s->factor, n / (n - 1.0)) : theta;
  double lo = 0.0, hi = 0.0;
  if (kind == NEBW_ROPE_YARN) {
    // the index whose frequency turns beta times within the trained length:
    // past the last frequency where that still turns more often, bounded by
    // rot_dim - 1 as the definition has it
    const double len = static_cast<double>(s->orig_len);
    lo = std::max(0.0, std::floor(n * std::log(len / (fast * kTwoPi)) / std::log(theta)));
    hi = std::min(rot_dim - 1.0, std::ceil(n * std::log(len / (slow * kTwoPi)) / std::log(theta)));
    if (hi < 0.0) lo = hi - 1.0;  // none turns `slow` times: all are scaled
    *scale = s->attn_scale > 0.0 ? s->attn_scale : 0.1 * std::log(s->factor) + 1.0;
  }
  for (int i = 0; i < n; ++i) {
    const double f = std::pow(base, -static_cast<double>(i) / n);
    double keep = 1.0;  // the share that stays unscaled
    if (kind == NEBW_ROPE_LINEAR) keep = 0.0;
    if (kind == NEBW_ROPE_YARN)
      keep = 1.0 - std::min(1.0, std::max(0.0, (i - lo) / std::max(hi - lo, 1e-3)));
    if (kind == NEBW_ROPE_BANDS)
      keep = std::min(1.0, std::max(0.0, (s->orig_len * f / kTwoPi - slow) / (fast - slow)));
    inv_freq[i] = keep == 1.0 ? f : f * keep + f / s->factor * (1.0 - keep);
  }
  return NEBW_OK;
}

extern "C" int nebw_stage_rope(nebw_dev *d, const double *inv_freq, int32_t n, int64_t max_pos,
                               double scale, uint64_t *handle) {
  if (int rc = use_dev(d)) return rc;
  NEBW_REQUIRE(inv_freq && handle, "null rotary operand");
  NEBW_REQUIRE(n >= 1 && n <= nebw::kHeadMaxDim / 2, "%d rotary frequencies refused: 1 .. %d", n,
               nebw::kHeadMaxDim / 2);
  NEBW_REQUIRE(max_pos >= 1 && max_pos <= (1ll << 28) / n,
               "rotary table of %lld positions refused", static_cast<long long>(max_pos));
  NEBW_REQUIRE(std::isfinite(scale) && scale != 0.0, "rotary scale %g refused", scale);
  for (int i = 0; i < n; ++i)
    NEBW_REQUIRE(std::isfinite(inv_freq[i]), "rotary frequency %d is not finite", i);
  RopeTable t;
  t.n = n;
  t.max_pos = max_pos;
  double *freq = nullptr;
  const size_t entries = static_cast<size_t>(max_pos) * n;
  if (cudaMalloc(&t.table, entries * sizeof(float2)) != cudaSuccess ||
      cudaMalloc(&freq, n * sizeof(double)) != cudaSuccess) {
    cudaGetLastError();
    cudaFree(t.table);
    return set_error(NEBW_ENOMEM, "cudaMalloc for a rotary table [%lld, %d] failed",
                     static_cast<long long>(max_pos), n);
  }
  cudaError_t e =
      cudaMemcpyAsync(freq, inv_freq, n * sizeof(double), cudaMemcpyHostToDevice, d->stream);
  if (e == cudaSuccess) {
    e = nebw::launch_rope_table(freq, n, max_pos, scale, t.table, d->stream);
  }
  if (e == cudaSuccess) e = cudaStreamSynchronize(d->stream);
  cudaFree(freq);
  if (e != cudaSuccess) {
    cudaFree(t.table);
    return set_error(NEBW_ECUDA, "rotary table staging failed: %s", cudaGetErrorString(e));
  }
  const int rc = keep_staged(d, d->ropes, t, handle);
  if (rc) cudaFree(t.table);
  return rc;
}

extern "C" int nebw_packed_positions(nebw_dev *d, const int32_t *off, const int32_t *len,
                                     int32_t B, int32_t max_len, int64_t rows, int32_t *pos,
                                     void *stream) {
  if (int rc = use_dev(d)) return rc;
  NEBW_REQUIRE(B >= 0 && B <= 65535 && max_len >= 0, "positions of %d sequences up to %d refused",
               B, max_len);
  NEBW_REQUIRE(rows >= 0, "rows %lld refused", static_cast<long long>(rows));
  if (B == 0 || max_len == 0) return NEBW_OK;
  NEBW_REQUIRE(off && len && (pos || rows == 0), "null position operand");
  NEBW_REQUIRE(words(off, len, pos), "position operands are not aligned");
  const dim3 grid(static_cast<unsigned>((int64_t{max_len} + 255) / 256), B);
  nebw::row_pos_kernel<<<grid, 256, 0, pick_stream(d, stream)>>>(off, len, max_len, rows, pos,
                                                                 d->d_err);
  NEBW_CUDA(cudaGetLastError());
  return NEBW_OK;
}

extern "C" int nebw_row_positions(nebw_dev *d, const int32_t *off, const int32_t *len, int32_t B,
                                  int32_t max_len, int32_t *pos, void *stream) {
  const int64_t rows = B > 0 && max_len > 0 ? int64_t{B} * max_len : 0;
  return nebw_packed_positions(d, off, len, B, max_len, rows, pos, stream);
}

namespace {

int check_heads(const nebw_heads *h, const char *what, int32_t head_dim, int64_t rows, size_t esz,
                int norm, nebw::HeadSide *side) {
  *side = nebw::HeadSide{};
  if (!h || h->heads == 0) return NEBW_OK;
  NEBW_REQUIRE(h->heads > 0 && h->heads <= 4096, "%d %s heads refused", h->heads, what);
  const int64_t width = static_cast<int64_t>(h->heads) * head_dim;
  if (rows == 0) {  // an empty tensor may have no address
    side->heads = h->heads;
    return NEBW_OK;
  }
  NEBW_REQUIRE(h->x && h->out, "null %s operand", what);
  NEBW_REQUIRE(aligned(h->x, esz) && aligned(h->out, esz), "%s heads are not element-aligned",
               what);
  NEBW_REQUIRE(rows <= 1 || (h->stride >= width && h->out_stride >= width),
               "%s row stride refused: %lld and %lld for %lld elements a row", what,
               static_cast<long long>(h->stride), static_cast<long long>(h->out_stride),
               static_cast<long long>(width));
  NEBW_REQUIRE(h->stride < (1ll << 31) && h->out_stride < (1ll << 31), "%s row stride refused",
               what);
  NEBW_REQUIRE(h->out != h->x || rows <= 1 || h->out_stride == h->stride,
               "%s heads in place need one row stride", what);
  if (norm != NEBW_HEADNORM_NONE) {
    NEBW_REQUIRE(h->gamma, "%s norm without its weight", what);
    NEBW_REQUIRE(norm != NEBW_HEADNORM_LAYER || h->beta, "%s LayerNorm without its bias", what);
    NEBW_REQUIRE(aligned(h->gamma, 4) && aligned(h->beta, 4), "%s norm weights are not aligned",
                 what);
  }
  side->x = h->x;
  side->out = h->out;
  side->stride = h->stride;
  side->out_stride = h->out_stride;
  side->heads = h->heads;
  side->gamma = h->gamma;
  side->beta = h->beta;
  return NEBW_OK;
}

int run_heads(nebw_dev *d, const nebw_heads *q, const nebw_heads *k, int dtype, int64_t rows,
              const int32_t *rows_dev, int32_t head_dim, int norm, float eps, uint64_t rope,
              int layout, const int32_t *pos, void *stream) {
  if (int rc = use_dev(d)) return rc;
  NEBW_REQUIRE(dtype == NEBW_F32 || dtype == NEBW_BF16, "head dtype %d refused", dtype);
  NEBW_REQUIRE(rows >= 0 && rows < (1ll << 31), "rows %lld refused", static_cast<long long>(rows));
  NEBW_REQUIRE(head_dim >= 2 && head_dim % 2 == 0 && head_dim <= nebw::kHeadMaxDim,
               "head_dim %d refused: even, 2 .. %d", head_dim, nebw::kHeadMaxDim);
  NEBW_REQUIRE(norm == NEBW_HEADNORM_NONE || norm == NEBW_HEADNORM_RMS ||
                   norm == NEBW_HEADNORM_LAYER,
               "head norm %d refused", norm);
  NEBW_REQUIRE(norm == NEBW_HEADNORM_NONE || (eps >= 0.0f && std::isfinite(eps)),
               "head norm eps %g refused", static_cast<double>(eps));
  NEBW_REQUIRE(layout == NEBW_ROPE_HALF || layout == NEBW_ROPE_PAIRS, "rotary layout %d refused",
               layout);
  nebw::HeadArgs a{};
  if (rope) {
    const RopeTable *t = find_staged(d, d->ropes, rope);
    NEBW_REQUIRE(t, "unknown rotary handle %llu", static_cast<unsigned long long>(rope));
    NEBW_REQUIRE(2 * t->n <= head_dim, "a rotary width of %d is more than head_dim %d", 2 * t->n,
                 head_dim);
    NEBW_REQUIRE(pos || rows == 0, "rotation without positions");
    NEBW_REQUIRE(words(pos), "positions are not aligned");
    a.n = t->n;
    a.table = t->table;
    a.max_pos = t->max_pos;
    a.pos = pos;
  }
  const size_t esz = dtype == NEBW_F32 ? 4 : 2;
  if (int rc = check_heads(q, "query", head_dim, rows, esz, norm, &a.q)) return rc;
  if (int rc = check_heads(k, "key", head_dim, rows, esz, norm, &a.k)) return rc;
  NEBW_REQUIRE(a.q.heads + a.k.heads > 0, "no heads given");
  NEBW_REQUIRE(words(rows_dev), "the live row count is not aligned");
  const auto apart = [&](const nebw::HeadSide &s, bool out_s, const nebw::HeadSide &t) {
    // s's rows (read or written) and t's written ones
    const int64_t e = static_cast<int64_t>(esz), w = head_dim * e;
    return s.heads == 0 || t.heads == 0 ||
           !rows_meet(out_s ? s.out : s.x, (out_s ? s.out_stride : s.stride) * e, s.heads * w,
                      t.out, t.out_stride * e, t.heads * w, rows);
  };
  if (rows > 0) {
    NEBW_REQUIRE(a.q.x == a.q.out || apart(a.q, false, a.q), "query heads overlap their results");
    NEBW_REQUIRE(a.k.x == a.k.out || apart(a.k, false, a.k), "key heads overlap their results");
    NEBW_REQUIRE(apart(a.q, false, a.k) && apart(a.k, false, a.q) && apart(a.q, true, a.k),
                 "query and key heads overlap");
  }
  if (rows == 0) return NEBW_OK;
  a.rows = rows;
  a.rows_dev = rows_dev;
  a.head_dim = head_dim;
  a.eps = eps;
  a.err = d->d_err;
  const bool f32 = dtype == NEBW_F32;
  NEBW_REQUIRE(nebw::heads_fit(a, f32), "too many heads: %lld rows of %d",
               static_cast<long long>(rows), a.q.heads + a.k.heads);
  NEBW_CUDA(nebw::launch_heads(a, f32, norm, layout == NEBW_ROPE_PAIRS, pick_stream(d, stream)));
  return NEBW_OK;
}

}  // namespace

extern "C" int nebw_rope(nebw_dev *d, const nebw_heads *q, const nebw_heads *k, int dtype,
                         int64_t rows, const int32_t *rows_dev, int32_t head_dim, uint64_t rope,
                         int layout, const int32_t *pos, void *stream) {
  NEBW_REQUIRE(rope != 0, "nebw_rope without a rotary handle");
  return run_heads(d, q, k, dtype, rows, rows_dev, head_dim, NEBW_HEADNORM_NONE, 0.0f, rope, layout,
                   pos, stream);
}

extern "C" int nebw_qk_norm_rope(nebw_dev *d, const nebw_heads *q, const nebw_heads *k, int dtype,
                                 int64_t rows, const int32_t *rows_dev, int32_t head_dim, int norm,
                                 float eps, uint64_t rope, int layout, const int32_t *pos,
                                 void *stream) {
  NEBW_REQUIRE(norm == NEBW_HEADNORM_RMS || norm == NEBW_HEADNORM_LAYER, "head norm %d refused",
               norm);
  return run_heads(d, q, k, dtype, rows, rows_dev, head_dim, norm, eps, rope, layout, pos, stream);
}

// ---------------------------------------------------------------------------
// experts
// ---------------------------------------------------------------------------

namespace {

constexpr int kRouteMostBlocks = 256;  // no sm_100 GPU has more SMs

// One block chooses and places up to about where the two-kernel form takes
// over (measured equal at 190 rows of 64 experts by 8, 128 of 256 by 8, 1024
// of 8 by 2: 6.7 / 9.5 / 6.3 us): that much work of its rows.
bool route_fused(int64_t rows, int64_t experts, int64_t top_k) {
  return rows * (experts + 16 * top_k) <= 40000;
}

// Blocks of the two-kernel form: one an SM at most, which keeps the counts
// that every block sums small (two an SM: 28 us against 27 on 131,071 rows of
// 64 experts by 8, 27 against 20 on 31,000 of 256), of 32 rows at least.
int64_t route_blocks(int64_t rows, int sms) {
  return std::min<int64_t>((rows + 31) / 32, std::min(sms, kRouteMostBlocks));
}

int check_route(int64_t rows, int32_t experts, int32_t top_k) {
  NEBW_REQUIRE(experts >= 1 && experts <= nebw::kRouteMaxExperts, "%d experts refused: 1 .. %d",
               experts, nebw::kRouteMaxExperts);
  NEBW_REQUIRE(top_k >= 1 && top_k <= nebw::kRouteMaxK && top_k <= experts,
               "top_k %d of %d experts refused: 1 .. %d", top_k, experts, nebw::kRouteMaxK);
  NEBW_REQUIRE(rows >= 0 && rows < (1ll << 30) && rows * top_k < (1ll << 30),
               "%lld rows of %d experts refused", static_cast<long long>(rows), top_k);
  return NEBW_OK;
}

}  // namespace

extern "C" int64_t nebw_moe_route_workspace(int64_t rows, int32_t experts, int32_t top_k) {
  if (check_route(rows, experts, top_k)) return -1;
  if (route_fused(rows, experts, top_k)) return 0;
  return int64_t{kRouteMostBlocks} * experts * static_cast<int64_t>(sizeof(int));
}

extern "C" int nebw_moe_route(nebw_dev *d, const void *logits, int dtype, int64_t stride,
                              int64_t rows, const int32_t *rows_dev, int32_t experts,
                              int32_t top_k, int score, int renorm, float scale, int32_t *ids,
                              float *weights, int32_t *group_off, int32_t *row_src,
                              int32_t *row_dst, void *ws, int64_t ws_bytes, void *stream) {
  if (int rc = use_dev(d)) return rc;
  if (int rc = check_route(rows, experts, top_k)) return rc;
  NEBW_REQUIRE(dtype == NEBW_F32 || dtype == NEBW_BF16, "logit dtype %d refused", dtype);
  NEBW_REQUIRE(score == NEBW_ROUTE_SOFTMAX || score == NEBW_ROUTE_SIGMOID, "score %d refused",
               score);
  NEBW_REQUIRE(std::isfinite(scale), "routing scale %g refused", static_cast<double>(scale));
  NEBW_REQUIRE(group_off, "null routing output");
  NEBW_REQUIRE(words(rows_dev, ids, weights, group_off, row_src, row_dst),
               "routing operands are not aligned");
  const cudaStream_t st = pick_stream(d, stream);
  if (rows == 0) {
    NEBW_CUDA(cudaMemsetAsync(group_off, 0, (experts + 1) * sizeof(int), st));
    return NEBW_OK;
  }
  NEBW_REQUIRE(logits && ids && weights && row_src && row_dst, "null routing operand");
  NEBW_REQUIRE(stride >= experts && stride < (1ll << 31),
               "logit row stride %lld refused for %d experts", static_cast<long long>(stride),
               experts);
  const size_t esz = dtype == NEBW_F32 ? 4 : 2;
  NEBW_REQUIRE(aligned(logits, esz) && aligned(ws, 4), "routing operands are not aligned");
  const int64_t need = nebw_moe_route_workspace(rows, experts, top_k);
  NEBW_REQUIRE(ws_bytes >= need && (ws || need == 0),
               "routing workspace of %lld bytes refused: %lld are needed",
               static_cast<long long>(ws_bytes), static_cast<long long>(need));
  // what one block reads or writes must not be what another writes
  const int64_t each = rows * top_k * 4;
  const struct {
    const void *p;
    int64_t bytes;
  } parts[] = {{logits, ((rows - 1) * stride + experts) * static_cast<int64_t>(esz)},
               {ids, each},
               {weights, each},
               {group_off, (experts + 1) * int64_t{4}},
               {row_src, each},
               {row_dst, each},
               {ws, need}};
  for (const auto &x : parts)
    for (const auto *y = &x + 1; y != std::end(parts); ++y)
      NEBW_REQUIRE(!meet(x.p, x.bytes, y->p, y->bytes), "routing operands overlap");
  nebw::RouteArgs a{};
  a.logits = logits;
  a.stride = stride;
  a.rows = static_cast<int>(rows);
  a.rows_dev = rows_dev;
  a.experts = experts;
  a.k = top_k;
  a.sigmoid = score == NEBW_ROUTE_SIGMOID;
  a.renorm = renorm != 0;
  a.scale = scale;
  a.ids = ids;
  a.weights = weights;
  a.group_off = group_off;
  a.row_src = row_src;
  a.row_dst = row_dst;
  a.hist = static_cast<int *>(ws);
  a.vec = experts % 8 == 0 && aligned(logits, 16) && stride * esz % 16 == 0;
  a.tiles = nebw::route_tiles(experts);
  a.whole = (top_k == 4 || top_k == 8 || top_k == 16) && aligned(ids, 16) && aligned(row_dst, 16);
  const bool fused = route_fused(rows, experts, top_k);
  int blocks = fused ? 1 : static_cast<int>(route_blocks(rows, d->sm_count));
  a.block_rows = static_cast<int>(((rows + blocks - 1) / blocks + 31) / 32 * 32);
  blocks = static_cast<int>((rows + a.block_rows - 1) / a.block_rows);
  if (fused) blocks = 0;  // no counts of blocks
  NEBW_CUDA(nebw::launch_route(a, dtype == NEBW_F32, blocks, d->route_ready, st));
  return NEBW_OK;
}

extern "C" int nebw_stage_experts(nebw_dev *d, const void *kn, int dtype, int32_t experts,
                                  int64_t K, int64_t N, int gated, void *stream,
                                  uint64_t *handle) {
  if (int rc = use_dev(d)) return rc;
  NEBW_REQUIRE(kn && handle, "null expert weight operand");
  NEBW_REQUIRE(dtype == NEBW_F32 || dtype == NEBW_BF16, "weight dtype %d refused", dtype);
  NEBW_REQUIRE(experts >= 1 && experts <= nebw::kGroupMaxExperts, "%d experts refused: 1 .. %d",
               experts, nebw::kGroupMaxExperts);
  const int64_t col_blocks = (N + 255) / 256 * 2, k_blocks = (K + 63) / 64;
  NEBW_REQUIRE(K >= 64 && N >= 8 && K % 8 == 0 && N % 8 == 0 && K <= (1 << 20) &&
                   N <= (1 << 20) && experts * col_blocks * k_blocks < (1 << 24),
               "expert weights [%d, K=%lld, N=%lld] refused: K >= 64, K %% 8 == 0, N %% 8 == 0",
               experts, static_cast<long long>(K), static_cast<long long>(N));
  NEBW_REQUIRE(!gated || N % 64 == 0,
               "gated expert weights of N=%lld refused: [up | gate] of a multiple of 32 each",
               static_cast<long long>(N));
  bool on_device = false;
  if (int rc = where_is(d, kn, &on_device)) return rc;
  const cudaStream_t st = pick_stream(d, stream);
  const size_t esz = dtype == NEBW_F32 ? 4 : 2;
  NEBW_REQUIRE(!on_device || aligned(kn, esz), "expert weights are not aligned");
  if (int rc = ready_grouped(d)) return rc;
  const size_t one = static_cast<size_t>(K) * N * esz;
  Experts w;
  w.experts = experts;
  w.K = K;
  w.N = N;
  w.gated = gated != 0;
  void *tmp = nullptr;
  const int64_t blocks = experts * col_blocks * k_blocks;
  if (cudaMalloc(&w.ptr, static_cast<size_t>(blocks) * 128 * 64 * 2) != cudaSuccess ||
      (!on_device && cudaMalloc(&tmp, one) != cudaSuccess)) {
    cudaGetLastError();
    cudaFree(w.ptr);
    return set_error(NEBW_ENOMEM, "cudaMalloc for [%d, %lld, %lld] expert weights failed", experts,
                     static_cast<long long>(N), static_cast<long long>(K));
  }
  cudaError_t e = cudaSuccess;
  if (on_device) {
    e = nebw::launch_stage_experts(kn, dtype == NEBW_BF16, K, N, w.gated, 0, experts, w.ptr, st);
  } else {
    for (int i = 0; i < experts && e == cudaSuccess; ++i) {  // one expert's copy at a time
      e = cudaMemcpyAsync(tmp, static_cast<const char *>(kn) + i * one, one,
                          cudaMemcpyHostToDevice, st);
      if (e != cudaSuccess) break;
      e = nebw::launch_stage_experts(tmp, dtype == NEBW_BF16, K, N, w.gated, i, 1, w.ptr, st);
    }
  }
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  cudaFree(tmp);
  int rc = NEBW_OK;
  if (e != cudaSuccess)
    rc = set_error(NEBW_ECUDA, "expert weight staging failed: %s", cudaGetErrorString(e));
  if (!rc) rc = make_tmap_kmajor(&w.map, w.ptr, blocks * 128, 64, 128);
  if (!rc) rc = keep_staged(d, d->experts, w, handle);
  if (rc) cudaFree(w.ptr);
  return rc;
}

namespace {

int run_grouped(nebw_dev *d, const nebw::GroupedMaps &m, int epi, const nebw::GroupedArgs &a,
                   cudaStream_t st) {
  // the most tiles that the groups can make: every one may end in a part tile
  const int64_t tiles = (a.rows / a.tile_rows + std::min(a.experts, a.rows)) *
                        int64_t{(a.N + nebw::kGroupTileCols - 1) / nebw::kGroupTileCols};
  NEBW_REQUIRE(tiles < (1ll << 30), "grouped product too large");
  NEBW_REQUIRE(d->grouped_pairs > 0, "this GPU holds no CTA pair of the grouped product");
  const unsigned g = 2 * static_cast<unsigned>(std::min<int64_t>(tiles, d->grouped_pairs));
  NEBW_CUDA(nebw::launch_grouped(m, epi, a, g, st));
  return NEBW_OK;
}

}  // namespace

extern "C" int nebw_gemm_grouped(nebw_dev *d, uint64_t weight, const void *A, int64_t a_rows,
                                 const int32_t *row_src, const int32_t *group_off, int64_t rows,
                                 int64_t K, int64_t N, const float *bias, int act, void *C,
                                 int c_dtype, void *stream) {
  if (int rc = use_dev(d)) return rc;
  const Experts *staged = find_staged(d, d->experts, weight);
  NEBW_REQUIRE(staged, "unknown expert weight handle %llu",
               static_cast<unsigned long long>(weight));
  const Experts &w = *staged;
  NEBW_REQUIRE(K == w.K && N == w.N,
               "grouped product [rows, %lld] x [%lld, %lld] does not match the staged experts "
               "[%d, K=%lld, N=%lld]",
               static_cast<long long>(K), static_cast<long long>(K), static_cast<long long>(N),
               w.experts, static_cast<long long>(w.K), static_cast<long long>(w.N));
  NEBW_REQUIRE(rows >= 0 && rows < (1 << 30) && a_rows >= 0 && a_rows < (1 << 30),
               "grouped rows %lld of %lld refused", static_cast<long long>(rows),
               static_cast<long long>(a_rows));
  NEBW_REQUIRE(c_dtype == NEBW_F32 || c_dtype == NEBW_BF16, "output dtype %d refused", c_dtype);
  if (w.gated) {
    NEBW_REQUIRE(act == NEBW_GATE_SILU || act == NEBW_GATE_GELU_ERF, "gate activation %d refused",
                 act);
    NEBW_REQUIRE(c_dtype == NEBW_BF16, "a gated product writes bf16 output");
  } else {
    NEBW_REQUIRE(act == NEBW_ACT_NONE || act == NEBW_ACT_GELU8 || act == NEBW_ACT_GELU_ERF,
                 "activation %d refused", act);
    NEBW_REQUIRE(act == NEBW_ACT_NONE || c_dtype == NEBW_BF16,
                 "an activation epilogue writes bf16 output");
  }
  if (rows == 0) return NEBW_OK;
  NEBW_REQUIRE(A && C && group_off, "null grouped operand");
  NEBW_REQUIRE(a_rows > 0, "grouped rows of an empty A");
  NEBW_REQUIRE(row_src || a_rows >= rows, "A has %lld rows, the groups up to %lld",
               static_cast<long long>(a_rows), static_cast<long long>(rows));
  NEBW_REQUIRE(aligned(A, 16) && aligned(C, 16) && aligned(bias, 16),
               "grouped operands must be 16-byte aligned");
  NEBW_REQUIRE(words(group_off, row_src), "group offsets or row indices are not aligned");
  const int64_t c_bytes = rows * (w.gated ? N / 2 : N) * (c_dtype == NEBW_F32 ? 4 : 2);
  NEBW_REQUIRE(!meet(A, a_rows * K * 2, C, c_bytes),
               "a grouped product's output overlaps its rows");
  nebw::GroupedArgs a{};
  a.off = group_off;
  a.experts = w.experts;
  a.rows = static_cast<int>(rows);
  a.row_src = row_src;
  a.a_rows = static_cast<int>(a_rows);
  a.N = static_cast<int>(N);
  a.K = static_cast<int>(K);
  a.bias = bias;
  a.out = C;
  a.err = d->d_err;
  int epi = nebw::kGrpBf16;
  if (w.gated) epi = act == NEBW_GATE_SILU ? nebw::kGrpBf16SwiGLU : nebw::kGrpBf16GeGLU;
  else if (c_dtype == NEBW_F32) epi = nebw::kGrpF32;
  else if (act == NEBW_ACT_GELU8) epi = nebw::kGrpBf16Gelu8;
  else if (act == NEBW_ACT_GELU_ERF) epi = nebw::kGrpBf16Erf;
  nebw::GroupedMaps m;
  if (int rc = make_tmap_kmajor(&m.a, A, a_rows, K, row_src ? 1 : nebw::kGroupedBox)) return rc;
  if (row_src) m.a128 = m.a;  // not used
  else if (int rc = make_tmap_kmajor(&m.a128, A, a_rows, K, nebw::kGemmBM)) return rc;
  if (int rc = make_tmap_out(&m.c, C, rows, w.gated ? N / 2 : N, c_dtype == NEBW_BF16)) return rc;
  m.w = w.map;
  // small groups: half the rows a tile, two more stages in the ring (15.4
  // against 17.0 us at 64 rows a group, 8 experts, K 768, N 3840 gated; 27.1
  // against 29.6 at 32, 64 experts, K and N 1024); from 128 rows a group on
  // whole tiles read W once (36.9 against 34.7 us there)
  a.tile_rows = rows <= 64 * std::min<int64_t>(w.experts, rows) ? 128 : 256;
  // fp32 output over a long K: half tiles leave room for four parts of K,
  // which halves what is cut off (gemm_grouped_kernel).  Errors of random
  // signs at K 1536 / 2048 / 4096: two parts of whole tiles 7.3e-7 / 1.0e-6 /
  // 2.1e-6, four of half ones 3.5e-7 / 4.7e-7 / 1.0e-6, which fp32 sums keep
  // below 6.1e-7.  It costs 625 us against 413 (65,542 rows, K 4096, N 1024).
  if (c_dtype == NEBW_F32 && K > 1536) a.tile_rows = 128;
  return run_grouped(d, m, epi, a, pick_stream(d, stream));
}

extern "C" int nebw_moe_combine(nebw_dev *d, const void *y, int y_dtype, int64_t y_rows,
                                const int32_t *row_dst, const float *weights, int64_t rows,
                                const int32_t *rows_dev, int32_t top_k, int64_t H,
                                const float *residual, void *out, int out_dtype, void *stream) {
  if (int rc = use_dev(d)) return rc;
  NEBW_REQUIRE(y_dtype == NEBW_F32 || y_dtype == NEBW_BF16, "expert row dtype %d refused", y_dtype);
  NEBW_REQUIRE(out_dtype == NEBW_F32 || out_dtype == NEBW_BF16, "output dtype %d refused",
               out_dtype);
  NEBW_REQUIRE(top_k >= 1 && top_k <= nebw::kRouteMaxK, "top_k %d refused: 1 .. %d", top_k,
               nebw::kRouteMaxK);
  NEBW_REQUIRE(H >= 1 && H <= (1 << 20), "width %lld refused", static_cast<long long>(H));
  NEBW_REQUIRE(rows >= 0 && rows < (1ll << 30) && rows * top_k < (1ll << 30) && y_rows >= 0 &&
                   y_rows < (1ll << 30),
               "%lld rows of %d experts refused", static_cast<long long>(rows), top_k);
  if (rows == 0) return NEBW_OK;
  NEBW_REQUIRE((y || y_rows == 0) && row_dst && weights && out, "null combine operand");
  NEBW_REQUIRE(aligned(y, y_dtype == NEBW_F32 ? 4 : 2) &&
                   aligned(out, out_dtype == NEBW_F32 ? 4 : 2) &&
                   words(row_dst, weights, residual, rows_dev),
               "combine operands are not aligned");
  const int64_t out_bytes = rows * H * (out_dtype == NEBW_F32 ? 4 : 2);
  NEBW_REQUIRE(!meet(y, y_rows * H * (y_dtype == NEBW_F32 ? 4 : 2), out, out_bytes),
               "the combine's output overlaps the experts' rows");
  NEBW_REQUIRE((residual == out && out_dtype == NEBW_F32) ||
                   !meet(residual, residual ? rows * H * 4 : 0, out, out_bytes),
               "the combine's output overlaps its residual");
  nebw::CombineArgs a{};
  a.y = y;
  a.row_dst = row_dst;
  a.weights = weights;
  a.residual = residual;
  a.out = out;
  a.rows = static_cast<int>(rows);
  a.y_rows = static_cast<int>(y_rows);
  a.rows_dev = rows_dev;
  a.k = top_k;
  a.H = static_cast<int>(H);
  a.err = d->d_err;
  const bool vec = H % 8 == 0 && aligned(y, 16) && aligned(out, 16) && aligned(residual, 16);
  NEBW_CUDA(nebw::launch_combine(a, y_dtype == NEBW_F32, out_dtype == NEBW_F32, vec,
                                 pick_stream(d, stream)));
  return NEBW_OK;
}
