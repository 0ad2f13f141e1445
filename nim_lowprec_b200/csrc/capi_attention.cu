// capi_attention.cu -- the extern "C" boundary of the paged cache and its
// attention (include/lowprec_cuda.h): argument checks, then one launch.
#include <algorithm>
#include <cmath>

#include "attn.cuh"
#include "lp_internal.h"

namespace {

constexpr int64_t kIntMax = 0x7fffffff;
constexpr int64_t kCounterBytes = 4096;  // one 4-byte counter per CTA of a launch
constexpr int64_t kSlotRows = 256;       // most rows of a partial result
constexpr int64_t kSlotDim = 128;
// Mean query rows (tokens x group) per request and key head from which the chunk
// kernel is used.  The rows kernel reads the keys again for every 8 rows, the
// chunk kernel's tiles cost the same for 1 row and 128; where requests x key
// heads are few, the repeated reads spread over idle SMs.  4000 cached keys,
// bf16, rows / chunk kernel in us: 16 requests x 8 key heads 16 rows 86 / 94,
// 32 rows 179 / 96; x 32 heads 8 rows 182 / 288, 16 rows 355 / 291, 32 rows
// 699 / 295; one request x 8 heads 32 rows 27 / 41, 64 rows 35 / 42, 128 rows
// 53 / 44 (fp32 over int8: 35 / 40, 48 / 42, 75 / 47).
constexpr int64_t kChunkRows = 24, kChunkRowsFew = 64;
constexpr int64_t kFew = 32;  // requests x key heads

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

// Rows of `width` bytes, `stride` apart (contiguous memory is one row).
struct Span {
  uintptr_t p;
  uint64_t rows, width, stride;
};
Span span(const void* p, int64_t n, int64_t size) {
  return {reinterpret_cast<uintptr_t>(p), n > 0 ? 1u : 0u, static_cast<uint64_t>(n * size), 0};
}
// Whether a byte of `rows` is one of `one`'s, which is contiguous.
bool overlap(const Span& rows, const Span& one) {
  const uintptr_t p = rows.p, b = one.p, e = one.p + one.width;
  if (!rows.rows || !rows.width || !one.rows || e <= p) return false;
  // the last row that begins before one's end
  uint64_t r = rows.rows - 1;
  if (r && rows.stride) r = std::min(r, (e - 1 - p) / rows.stride);
  return p + r * rows.stride + rows.width > b;
}

int64_t elem_size(int t) { return t == LP_F32 ? 4 : t == LP_I8 ? 1 : 2; }

int check_cache(const lp_kv_cache* c) {
  if (!c) return LP_ERR_ARG;
  if (c->dtype != LP_F16 && c->dtype != LP_BF16 && c->dtype != LP_I8) return LP_ERR_ARG;
  LP_REQUIRE(c->pages >= 0 && c->page_size > 0 && c->kv_heads > 0);
  LP_REQUIRE(c->pages <= kIntMax && c->page_size <= kIntMax && c->kv_heads <= 65535);
  LP_REQUIRE(c->head_dim > 0 && c->head_dim % 16 == 0);
  if (c->head_dim > 256) return LP_ERR_UNSUPPORTED;
  if (c->pages == 0) return LP_OK;
  if (!c->k || !c->v) return LP_ERR_ARG;
  if (c->dtype == LP_I8 && (!c->k_scales || !c->v_scales)) return LP_ERR_ARG;
  const int64_t es = elem_size(c->dtype);
  for (int i = 0; i < 3; ++i) {  // not negative, and their kernels' units fit 32 bits
    LP_REQUIRE(c->k_strides[i] >= 0 && c->k_strides[i] * es / 16 <= kIntMax);
    LP_REQUIRE(c->v_strides[i] >= 0 && c->v_strides[i] * es / 16 <= kIntMax);
    if (c->dtype != LP_I8) continue;
    LP_REQUIRE(c->k_scale_strides[i] >= 0 && c->k_scale_strides[i] <= kIntMax);
    LP_REQUIRE(c->v_scale_strides[i] >= 0 && c->v_scale_strides[i] <= kIntMax);
  }
  uint64_t al = reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v);
  for (int i = 0; i < 3; ++i)
    al |= static_cast<uint64_t>(c->k_strides[i] * es) | static_cast<uint64_t>(c->v_strides[i] * es);
  return al & 15 ? LP_ERR_UNSUPPORTED : LP_OK;
}

int check_rows(const lp_rows* r, int64_t heads) {
  if (!r) return LP_ERR_ARG;
  if (r->dtype != LP_F32 && r->dtype != LP_F16 && r->dtype != LP_BF16) return LP_ERR_ARG;
  LP_REQUIRE(r->tokens >= 0 && r->tokens <= kIntMax && r->heads == heads);
  LP_REQUIRE(r->token_stride >= 0 && r->token_stride <= kIntMax);
  LP_REQUIRE(r->head_stride >= 0 && r->head_stride <= kIntMax);
  return bad(r->data, r->tokens) ? LP_ERR_ARG : LP_OK;
}

bool aligned16(const lp_rows& r) {
  const int64_t es = elem_size(r.dtype);
  return ((reinterpret_cast<uintptr_t>(r.data) | static_cast<uint64_t>(r.token_stride * es) |
           static_cast<uint64_t>(r.head_stride * es)) & 15) == 0;
}

int check_kv_rows(const lp_kv_cache* c, const lp_rows* k, const lp_rows* v, const int64_t* slots,
                  int64_t slots_len) {
  if (const int e = check_cache(c)) return e;
  if (const int e = check_rows(k, c->kv_heads)) return e;
  if (const int e = check_rows(v, c->kv_heads)) return e;
  if (k->dtype != v->dtype) return LP_ERR_ARG;
  LP_REQUIRE(k->tokens == v->tokens && slots_len == k->tokens);
  return bad(slots, slots_len) ? LP_ERR_ARG : LP_OK;
}

lp::attn::Pool pool(const void* data, const float* scales, const int64_t* s, const int64_t* ss) {
  return {static_cast<const uint8_t*>(data), scales, s[0], s[1], s[2], ss[0], ss[1], ss[2]};
}

int64_t workspace_bytes() {
  return kCounterBytes + lp::device_info().sm_count * 2ll * kSlotRows * (kSlotDim + 2) * 4;
}

}  // namespace

extern "C" {

int lp_assign_pages(const int32_t* ctx_lens, int64_t ctx_lens_len, const int32_t* new_lens,
                    int64_t new_lens_len, int64_t page_size, const int32_t* free_pages,
                    int64_t free_pages_len, const int32_t* free_head, int32_t* block_tables,
                    int64_t table_width, int64_t table_stride, int32_t* q_start,
                    int64_t q_start_len, int32_t* seq_lens, int64_t seq_lens_len, int64_t* slots,
                    int64_t slots_len, int32_t* positions, int64_t positions_len,
                    int32_t* free_head_out, lp_stream_t stream) {
  const int64_t n = ctx_lens_len;
  LP_REQUIRE(n >= 0 && n <= kIntMax / 2 && new_lens_len == n && seq_lens_len == n);
  LP_REQUIRE(q_start_len == n + 1 && page_size > 0 && page_size <= kIntMax);
  LP_REQUIRE(free_pages_len >= 0 && free_pages_len <= kIntMax);
  LP_REQUIRE(table_width >= 0 && table_width <= kIntMax && table_stride >= table_width);
  LP_REQUIRE(slots_len >= 0 && slots_len <= kIntMax);
  LP_REQUIRE(positions == nullptr || positions_len == slots_len);
  if (bad(ctx_lens, n) || bad(new_lens, n) || bad(seq_lens, n) || !q_start) return LP_ERR_ARG;
  if (bad(free_pages, free_pages_len) || bad(block_tables, n * table_width)) return LP_ERR_ARG;
  if (bad(slots, slots_len) || !free_head || !free_head_out) return LP_ERR_ARG;
  // Every block reads all the lengths, and tokens read the free list, while others write
  // their results: nothing that is written may lie on anything else.
  const Span in[] = {span(ctx_lens, n, 4), span(new_lens, n, 4), span(free_pages, free_pages_len, 4),
                     span(free_head, 1, 4)};
  const Span out[] = {span(q_start, n + 1, 4), span(seq_lens, n, 4), span(slots, slots_len, 8),
                      span(positions, positions ? slots_len : 0, 4), span(free_head_out, 1, 4)};
  const Span table{reinterpret_cast<uintptr_t>(block_tables), static_cast<uint64_t>(n),
                   static_cast<uint64_t>(table_width) * 4, static_cast<uint64_t>(table_stride) * 4};
  for (const Span& i : in)
    if (overlap(table, i)) return LP_ERR_ARG;
  for (const Span& o : out) {
    if (overlap(table, o)) return LP_ERR_ARG;
    for (const Span& i : in)
      if (overlap(i, o)) return LP_ERR_ARG;
    for (const Span& x : out)
      if (&x != &o && overlap(x, o)) return LP_ERR_ARG;
  }
  return lp::launch_assign_pages(ctx_lens, new_lens, n, page_size, free_pages, free_pages_len,
                                 free_head, block_tables, table_stride, table_width, q_start,
                                 seq_lens, slots, slots_len, positions, free_head_out, S(stream));
}

int lp_store_kv(const lp_kv_cache* cache, const lp_rows* k, const lp_rows* v,
                const int64_t* slots, int64_t slots_len, lp_stream_t stream) {
  if (const int e = check_kv_rows(cache, k, v, slots, slots_len)) return e;
  if (k->tokens == 0) return LP_OK;
  return lp::launch_store_kv(*cache, *k, *v, slots, aligned16(*k) && aligned16(*v), S(stream));
}

int lp_load_kv(const lp_kv_cache* cache, const int64_t* slots, int64_t slots_len,
               const lp_rows* k, const lp_rows* v, lp_stream_t stream) {
  if (const int e = check_kv_rows(cache, k, v, slots, slots_len)) return e;
  if (k->tokens == 0) return LP_OK;
  return lp::launch_load_kv(*cache, slots, *k, *v, aligned16(*k) && aligned16(*v), S(stream));
}

int lp_paged_attention_workspace(int64_t* bytes) {
  if (!bytes) return LP_ERR_ARG;
  *bytes = workspace_bytes();
  return LP_OK;
}

int lp_paged_attention(const lp_kv_cache* cache, const int32_t* block_tables, int64_t table_width,
                       int64_t table_stride, const int32_t* q_start, int64_t q_start_len,
                       const int32_t* seq_lens, int64_t seq_lens_len, const lp_rows* q,
                       const lp_rows* out, float scale, int64_t window, int64_t sinks, float* lse,
                       int64_t lse_len, void* workspace, int64_t workspace_len,
                       lp_stream_t stream) {
  if (const int e = check_cache(cache)) return e;
  if (!q || !out) return LP_ERR_ARG;
  if (const int e = check_rows(q, q->heads)) return e;
  if (const int e = check_rows(out, q->heads)) return e;
  if (q->dtype != out->dtype) return LP_ERR_ARG;
  const int64_t n = seq_lens_len;
  LP_REQUIRE(q->heads > 0 && q->heads <= 65535 && q->heads % cache->kv_heads == 0);
  LP_REQUIRE(out->tokens == q->tokens && q->tokens * q->heads <= kIntMax / 2);
  LP_REQUIRE(n >= 0 && n <= kIntMax / 2 && q_start_len == n + 1);
  LP_REQUIRE(table_width >= 0 && table_width <= kIntMax && table_stride >= table_width);
  LP_REQUIRE(window >= 0 && sinks >= 0);
  LP_REQUIRE(lse == nullptr || lse_len == q->tokens * q->heads);
  if (!std::isfinite(scale)) return LP_ERR_ARG;
  if (bad(block_tables, n * table_width) || !q_start || bad(seq_lens, n)) return LP_ERR_ARG;
  if (cache->head_dim != 64 && cache->head_dim != 96 && cache->head_dim != 128)
    return LP_ERR_UNSUPPORTED;
  if (q->tokens == 0 || n == 0) return LP_OK;
  LP_REQUIRE(workspace_len >= workspace_bytes());
  if (!workspace || reinterpret_cast<uintptr_t>(workspace) & 15) return LP_ERR_ARG;

  lp::attn::Args a;
  a.q = q->data;
  a.out = out->data;
  a.lse = lse;
  a.q_type = q->dtype;
  a.q_vec = aligned16(*q) && aligned16(*out);
  a.q_token = q->token_stride;
  a.q_head = q->head_stride;
  a.o_token = out->token_stride;
  a.o_head = out->head_stride;
  a.k = pool(cache->k, cache->k_scales, cache->k_strides, cache->k_scale_strides);
  a.v = pool(cache->v, cache->v_scales, cache->v_strides, cache->v_scale_strides);
  a.table = block_tables;
  a.qstart = q_start;
  a.seqlens = seq_lens;
  a.table_stride = table_stride;
  a.table_width = static_cast<int>(table_width);
  a.pages = static_cast<int>(cache->pages);
  a.page_size = static_cast<int>(cache->page_size);
  a.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (cache->page_size == int64_t{1} << i) a.page_shift = i;
  a.requests = static_cast<int>(n);
  a.tokens = static_cast<int>(q->tokens);
  a.heads = static_cast<int>(q->heads);
  a.kv_heads = static_cast<int>(cache->kv_heads);
  a.group = a.heads / a.kv_heads;
  a.window = static_cast<int>(std::min(window, kIntMax / 2));
  a.sinks = static_cast<int>(std::min(sinks, kIntMax / 2));
  a.scale_log2 = scale * 1.4426950408889634f;
  a.counters = static_cast<uint32_t*>(workspace);
  a.partials = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kCounterBytes);
  const int64_t rows = n * cache->kv_heads < kFew ? kChunkRowsFew : kChunkRows;
  const bool chunk = q->tokens * a.group >= rows * n;
  return chunk ? lp::launch_attn_chunk(a, cache->dtype, cache->head_dim, S(stream))
               : lp::launch_attn_rows(a, cache->dtype, cache->head_dim, S(stream));
}

}  // extern "C"
