// capi_experts.cu -- the extern "C" boundary of 8-bit rows, the router and the
// experts' products (include/lowprec_cuda.h): argument checks, then the launches.
#include <algorithm>
#include <cmath>

#include "experts.cuh"
#include "lp_internal.h"

namespace {

constexpr int64_t kIntMax = 0x7fffffff;
constexpr int64_t kMaxCols = 32768;  // of a row that is normed

#define LP_REQUIRE(cond)              \
  do {                                \
    if (!(cond)) return LP_ERR_SHAPE; \
  } while (0)

// The queued GEMVs of this thread's open batch go first (see capi.cu).
cudaStream_t S(lp_stream_t s) {
  if (lp::batch_open()) lp::batch_flush_keep();
  return static_cast<cudaStream_t>(s);
}

bool bad(const void* p, int64_t len) { return len > 0 && p == nullptr; }
int64_t elem_size(int t) { return t == LP_F32 ? 4 : 2; }

int check_matrix(const lp_matrix* m) {
  if (!m) return LP_ERR_ARG;
  if (m->dtype != LP_F32 && m->dtype != LP_F16 && m->dtype != LP_BF16) return LP_ERR_ARG;
  LP_REQUIRE(m->rows >= 0 && m->rows <= kIntMax && m->cols >= 0 && m->cols <= kIntMax);
  LP_REQUIRE(m->stride >= 0 && m->stride <= kIntMax);
  return bad(m->data, m->rows * m->cols) ? LP_ERR_ARG : LP_OK;
}

int check_rows8(const lp_rows8* r) {
  if (!r) return LP_ERR_ARG;
  if (r->dtype != LP_E4M3 && r->dtype != LP_I8) return LP_ERR_ARG;
  const int g = r->group;
  LP_REQUIRE(g == 32 || (r->dtype == LP_I8 && (g == 64 || g == 128 || g == 256)));
  LP_REQUIRE(r->rows >= 0 && r->rows <= kIntMax && r->cols >= 0 && r->cols <= kIntMax && r->cols % g == 0);
  LP_REQUIRE(r->code_stride >= 0 && r->code_stride <= kIntMax);
  LP_REQUIRE(r->scale_stride >= 0 && r->scale_stride <= kIntMax);
  return bad(r->codes, r->rows * r->cols) || bad(r->scales, r->rows * r->cols) ? LP_ERR_ARG : LP_OK;
}

// Whether rows are read and written 8 elements at a time: 16-byte pieces, codes 8.
bool aligned(const lp_matrix* m) {
  if (!m) return true;
  return ((reinterpret_cast<uintptr_t>(m->data) | static_cast<uintptr_t>(m->stride * elem_size(m->dtype))) & 15) == 0;
}
bool aligned(const lp_rows8* r) {
  if (!r) return true;
  return ((reinterpret_cast<uintptr_t>(r->codes) | static_cast<uintptr_t>(r->code_stride)) & 7) == 0;
}
bool aligned16(const lp_rows8* r) {
  return ((reinterpret_cast<uintptr_t>(r->codes) | static_cast<uintptr_t>(r->code_stride)) & 15) == 0;
}

int check_weights(const lp_expert_weights* w) {
  if (!w) return LP_ERR_ARG;
  if (w->dtype != LP_E2M1 && w->dtype != LP_E4M3) return LP_ERR_ARG;
  if (w->gated != 0 && w->gated != 1) return LP_ERR_ARG;
  LP_REQUIRE(w->experts > 0 && w->rows > 0 && w->cols > 0);
  LP_REQUIRE(w->rows <= kIntMax / 2 && w->cols <= kIntMax / 2 && w->cols % 32 == 0);
  LP_REQUIRE(!w->gated || w->rows % 64 == 0);
  if (w->experts > lp::kRouteExperts) return LP_ERR_UNSUPPORTED;
  // (tiles are found by a 32-bit row of 128 or 64 bytes)
  const lp::experts::Layout l = lp::experts::layout(w->experts, w->rows, w->cols, w->dtype, w->gated);
  return l.tiles > kIntMax / lp::experts::kTileM ? LP_ERR_UNSUPPORTED : LP_OK;
}

struct Span {
  uintptr_t b, e;
};
Span span(const void* p, int64_t n, int64_t size) {
  const uintptr_t b = reinterpret_cast<uintptr_t>(p);
  return {b, b + static_cast<uintptr_t>(p ? n * size : 0)};
}
bool meet(const Span& a, const Span& b) { return a.b < a.e && b.b < b.e && a.b < b.e && b.b < a.e; }

int check_product(const lp_expert_weights* w, bool gated, const lp_rows8* x, const int32_t* offsets,
                  int64_t offsets_len, const int32_t* row_token, int64_t row_token_len) {
  if (const int e = check_weights(w)) return e;
  if (static_cast<bool>(w->gated) != gated) return LP_ERR_ARG;
  if (const int e = check_rows8(x)) return e;
  if (x->dtype != LP_E4M3) return LP_ERR_ARG;
  LP_REQUIRE(x->cols == w->cols && offsets_len == w->experts + 1);
  LP_REQUIRE(row_token_len >= 0 && row_token_len <= kIntMax);
  LP_REQUIRE(row_token || row_token_len == 0 || row_token_len == x->rows);
  if (!w->tiles || !w->scales || !offsets) return LP_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(w->tiles) | reinterpret_cast<uintptr_t>(w->scales)) & 31) return LP_ERR_ARG;
  return aligned16(x) ? LP_OK : LP_ERR_UNSUPPORTED;
}

int64_t product_workspace(const int32_t* row_token, int64_t rows, int64_t cols) {
  return lp::experts::fixed_workspace() + (row_token ? lp::experts::gather_workspace(rows, cols) : 0);
}
int check_workspace(const void* p, int64_t len, int64_t need) {
  LP_REQUIRE(len >= need);
  return !p || reinterpret_cast<uintptr_t>(p) & 15 ? LP_ERR_ARG : LP_OK;
}

}  // namespace

extern "C" {

int lp_quantize_rows(const lp_matrix* x, const lp_rows8* out, lp_stream_t stream) {
  if (const int e = check_matrix(x)) return e;
  if (const int e = check_rows8(out)) return e;
  LP_REQUIRE(out->rows == x->rows && out->cols == x->cols);
  if (x->rows == 0 || x->cols == 0) return LP_OK;
  return lp::launch_quantize_rows(*x, *out, aligned(x) && aligned(out), S(stream));
}

int lp_dequantize_rows(const lp_rows8* rows, const lp_matrix* dst, lp_stream_t stream) {
  if (const int e = check_rows8(rows)) return e;
  if (const int e = check_matrix(dst)) return e;
  LP_REQUIRE(rows->rows == dst->rows && rows->cols == dst->cols);
  if (dst->rows == 0 || dst->cols == 0) return LP_OK;
  return lp::launch_dequantize_rows(*rows, *dst, aligned(rows) && aligned(dst), S(stream));
}

int lp_add_rms_norm(const lp_matrix* x, const lp_matrix* residual, const void* weight, int64_t weight_len,
                    int32_t weight_type, float eps, const lp_matrix* total, const lp_matrix* y, const lp_rows8* q,
                    lp_stream_t stream) {
  if (const int e = check_matrix(x)) return e;
  for (const lp_matrix* m : {residual, total, y}) {
    if (!m) continue;
    if (const int e = check_matrix(m)) return e;
    LP_REQUIRE(m->rows == x->rows && m->cols == x->cols);
  }
  const int stream_type = residual ? residual->dtype : x->dtype;
  if (stream_type != x->dtype && stream_type != LP_F32) return LP_ERR_ARG;
  if (total && total->dtype != stream_type) return LP_ERR_ARG;
  if (q) {
    if (const int e = check_rows8(q)) return e;
    LP_REQUIRE(q->rows == x->rows && q->cols == x->cols);
  }
  if (weight_type != LP_F32 && weight_type != LP_F16 && weight_type != LP_BF16) return LP_ERR_ARG;
  LP_REQUIRE(weight_len == x->cols);
  if (bad(weight, weight_len) || !std::isfinite(eps) || eps < 0.0f) return LP_ERR_ARG;
  if (!total && !y && !q) return LP_ERR_ARG;
  if (x->cols > kMaxCols) return LP_ERR_UNSUPPORTED;
  if (x->rows == 0 || x->cols == 0) return LP_OK;
  const bool vec = x->cols % 8 == 0 && aligned(x) && aligned(residual) && aligned(total) && aligned(y) &&
                   aligned(q) && (reinterpret_cast<uintptr_t>(weight) & 15) == 0;
  return lp::launch_norm(*x, residual, weight, weight_type, eps, total, y, q, vec, S(stream));
}

int lp_experts_workspace(int64_t rows, int64_t cols, int64_t* bytes) {
  LP_REQUIRE(rows >= 0 && rows <= kIntMax && cols >= 0 && cols <= kIntMax);
  if (!bytes) return LP_ERR_ARG;
  *bytes = lp::experts::fixed_workspace() + lp::experts::gather_workspace(rows, cols);
  return LP_OK;
}

int lp_route_experts(const lp_matrix* logits, float* weights, int64_t weights_len, int32_t* experts,
                     int64_t experts_len, int32_t* offsets, int64_t offsets_len, int32_t* row_token,
                     int64_t row_token_len, int32_t* places, int64_t places_len, int64_t k, int32_t renormalize,
                     void* workspace, int64_t workspace_len, lp_stream_t stream) {
  if (const int e = check_matrix(logits)) return e;
  const int64_t t = logits->rows, n = logits->cols;
  LP_REQUIRE(n > 0 && k > 0 && k <= n);
  if (n > lp::kRouteExperts || k > 32) return LP_ERR_UNSUPPORTED;
  LP_REQUIRE(t * k <= kIntMax && offsets_len == n + 1);
  LP_REQUIRE(weights_len == t * k && experts_len == t * k && row_token_len == t * k && places_len == t * k);
  if (bad(weights, t) || bad(experts, t) || bad(row_token, t) || bad(places, t) || !offsets) return LP_ERR_ARG;
  if (renormalize != 0 && renormalize != 1) return LP_ERR_ARG;
  if (const int e = check_workspace(workspace, workspace_len, lp::experts::fixed_workspace())) return e;
  // experts are read again while places are written: nothing that is written may lie on
  // anything else
  const Span s[] = {span(weights, t * k, 4), span(experts, t * k, 4), span(row_token, t * k, 4),
                    span(places, t * k, 4), span(offsets, n + 1, 4),
                    span(workspace, lp::experts::fixed_workspace(), 1),
                    span(logits->data, t ? (t - 1) * logits->stride + n : 0, elem_size(logits->dtype))};
  for (const Span& a : s)
    for (const Span& b : s)
      if (&a < &b && meet(a, b)) return LP_ERR_ARG;
  return lp::launch_route(*logits, weights, experts, offsets, row_token, places, k, renormalize,
                          reinterpret_cast<int32_t*>(static_cast<uint8_t*>(workspace) + lp::experts::kCounterBytes), S(stream));
}

int lp_expert_weights_bytes(const lp_expert_weights* w, int64_t* tile_bytes, int64_t* scale_bytes) {
  if (const int e = check_weights(w)) return e;
  if (!tile_bytes || !scale_bytes) return LP_ERR_ARG;
  const lp::experts::Layout l = lp::experts::layout(w->experts, w->rows, w->cols, w->dtype, w->gated);
  *tile_bytes = l.tiles * l.tile_bytes;
  *scale_bytes = l.tiles * lp::experts::kSfBytes;
  return LP_OK;
}

int lp_expert_weights_pack(const void* codes, int64_t codes_len, const void* scales, int64_t scales_len,
                           int32_t scale_type, const lp_expert_weights* out, lp_stream_t stream) {
  if (const int e = check_weights(out)) return e;
  if (scale_type != LP_F32 && scale_type != LP_E8M0) return LP_ERR_ARG;
  const int64_t n = out->experts * out->rows * out->cols;
  LP_REQUIRE(codes_len == (out->dtype == LP_E2M1 ? n / 2 : n) && scales_len == n / 32);
  if (!codes || !scales || !out->tiles || !out->scales) return LP_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(out->tiles) | reinterpret_cast<uintptr_t>(out->scales)) & 31) return LP_ERR_ARG;
  return lp::launch_pack_experts(codes, scales, scale_type, *out, S(stream));
}

int lp_expert_gemm(const lp_expert_weights* w, const lp_rows8* x, const int32_t* offsets, int64_t offsets_len,
                   const int32_t* row_token, int64_t row_token_len, const lp_matrix* out, void* workspace,
                   int64_t workspace_len, lp_stream_t stream) {
  if (const int e = check_product(w, false, x, offsets, offsets_len, row_token, row_token_len)) return e;
  if (const int e = check_matrix(out)) return e;
  const int64_t rows = row_token ? row_token_len : x->rows;
  LP_REQUIRE(out->rows == rows && out->cols == w->rows);
  if (const int e = check_workspace(workspace, workspace_len, product_workspace(row_token, rows, x->cols))) return e;
  if (rows == 0) return LP_OK;
  LP_REQUIRE(x->rows > 0);
  return lp::launch_experts(*w, *x, offsets, row_token, rows, out, nullptr, workspace, S(stream));
}

int lp_expert_gemm_gated(const lp_expert_weights* w, const lp_rows8* x, const int32_t* offsets,
                         int64_t offsets_len, const int32_t* row_token, int64_t row_token_len, const lp_rows8* out,
                         void* workspace, int64_t workspace_len, lp_stream_t stream) {
  if (const int e = check_product(w, true, x, offsets, offsets_len, row_token, row_token_len)) return e;
  if (const int e = check_rows8(out)) return e;
  if (out->dtype != LP_E4M3) return LP_ERR_ARG;
  const int64_t rows = row_token ? row_token_len : x->rows;
  LP_REQUIRE(out->rows == rows && out->cols == w->rows / 2);
  if (!aligned16(out)) return LP_ERR_UNSUPPORTED;
  if (const int e = check_workspace(workspace, workspace_len, product_workspace(row_token, rows, x->cols))) return e;
  if (rows == 0) return LP_OK;
  LP_REQUIRE(x->rows > 0);
  return lp::launch_experts(*w, *x, offsets, row_token, rows, nullptr, out, workspace, S(stream));
}

int lp_combine_experts(const lp_matrix* rows, const float* weights, int64_t weights_len, const int32_t* places,
                       int64_t places_len, const lp_matrix* residual, const lp_matrix* out, lp_stream_t stream) {
  if (const int e = check_matrix(rows)) return e;
  if (const int e = check_matrix(out)) return e;
  if (residual) {
    if (const int e = check_matrix(residual)) return e;
    LP_REQUIRE(residual->rows == out->rows);
    LP_REQUIRE(residual->cols == out->cols);
    if (residual->dtype != out->dtype) return LP_ERR_ARG;
  }
  const int64_t t = out->rows;
  LP_REQUIRE(rows->cols == out->cols && weights_len == places_len && places_len >= 0 && places_len <= kIntMax);
  if (t == 0 || out->cols == 0) {
    LP_REQUIRE(t > 0 || places_len == 0);
    return LP_OK;
  }
  LP_REQUIRE(places_len % t == 0);
  if (bad(weights, weights_len) || bad(places, places_len)) return LP_ERR_ARG;
  const bool vec = out->cols % 8 == 0 && aligned(rows) && aligned(residual) && aligned(out);
  return lp::launch_combine(*rows, weights, places, places_len / t, residual, *out, vec, S(stream));
}

}  // extern "C"
