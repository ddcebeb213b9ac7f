// C ABI of rotary positions, the 8-bit cache and attention over it: argument checks and launches.
#include "capi_checks.h"

using namespace tfm;

namespace {

constexpr int64_t kMaxStride = (int64_t)1 << 40;
constexpr double kLog2e = 1.4426950408889634074;

void need_heads(int32_t heads) { need(heads > 0 && heads <= kMaxHeads, "heads must be in [1, 1024]"); }

// Rows of heads with strides, and the bytes that they span.
Span rows_span(const void* p, int64_t rows, int32_t heads, int32_t dim, int64_t row_stride, int64_t head_stride,
               const char* name) {
  if (row_stride < 0 || head_stride < 0 || row_stride > kMaxStride || head_stride > kMaxStride)
    fail(TFM_E_INVALID, std::string(name) + ": strides must be in [0, 2^40]");
  need_ptr(p, name);
  return Span{p, (size_t)((rows - 1) * row_stride + (heads - 1) * head_stride + dim) * 2};
}

void need_rotation(const tfm_rotation* r, int32_t head_dim) {
  need(r->pairs > 0 && 2 * (int64_t)r->pairs <= head_dim, "pairs must be in [1, head_dim / 2]");
  need(r->scale == r->scale && r->scale - r->scale == 0.0f, "rotation scale must be finite");
  need_ptr(r->frequencies, "frequencies");
}

struct CacheSpans {
  Span k, v, ks, vs, table, lengths, starts;
};

// Checks a cache and its batch; the kernels' arguments.
KvBatchArgs need_batch(const tfm_kv_cache* c, const tfm_kv_batch* b, int64_t rows, CacheSpans* spans) {
  need_ptr(c, "cache");
  need_ptr(b, "batch");
  need(c->pages > 0, "the cache has no pages");
  if (c->pages > INT32_MAX) fail(TFM_E_UNSUPPORTED, "more than 2^31 - 1 pages are not built");
  need(c->kv_heads > 0 && c->kv_heads <= kMaxHeads, "kv_heads must be in [1, 1024]");
  int shift = 4;
  while (shift < 8 && (1 << shift) != c->page_tokens) ++shift;
  if ((1 << shift) != c->page_tokens) fail(TFM_E_UNSUPPORTED, "page_tokens must be 16, 32, 64, 128 or 256");
  if (c->head_dim != 64 && c->head_dim != 128) fail(TFM_E_UNSUPPORTED, "only head_dim 64 and 128 are built");
  need(b->sequences >= 0 && b->sequences <= kMaxRows, "sequences out of range");
  need(b->table_width > 0, "table_width must be positive");
  if (((int64_t)b->table_width << shift) > (1 << 30)) fail(TFM_E_UNSUPPORTED, "tables of more than 2^30 tokens are not built");
  need(b->max_rows >= 0 && b->max_rows <= kMaxRows, "max_rows out of range");
  need(b->starts || (int64_t)b->sequences * b->max_rows == rows, "without starts rows must be sequences * max_rows");
  KvBatchArgs a{c->k,           c->v,      c->k_scales, c->v_scales, (int)c->pages,  c->kv_heads,    shift,
                b->table,       b->lengths, b->starts,  b->sequences, b->table_width,
                (int)std::min<int64_t>(b->max_rows, rows), (int)rows};
  if (rows == 0 || b->sequences == 0) return a;
  need_ptr(c->k, "k codes");
  need_ptr(c->v, "v codes");
  need_ptr(c->k_scales, "k_scales");
  need_ptr(c->v_scales, "v_scales");
  need_align16(c->k, "k codes");
  need_align16(c->v, "v codes");
  need_ptr(b->table, "table");
  need_ptr(b->lengths, "lengths");
  const size_t places = (size_t)c->pages * (size_t)c->kv_heads, n = (size_t)b->sequences;
  const size_t codes = (places << shift) * (size_t)c->head_dim;
  *spans = CacheSpans{{c->k, codes},
                      {c->v, codes},
                      {c->k_scales, places * 4},
                      {c->v_scales, places * 4},
                      {b->table, n * (size_t)b->table_width * 4},
                      {b->lengths, n * 4},
                      {b->starts, (n + 1) * 4}};
  return a;
}

int group_of(int32_t heads, const KvBatchArgs& b) {
  need_heads(heads);
  need(heads % b.kv_heads == 0, "heads must be a multiple of kv_heads");
  const int group = heads / b.kv_heads;
  if ((int64_t)b.rows * group > (1 << 30)) fail(TFM_E_UNSUPPORTED, "rows * heads / kv_heads past 2^30 is not built");
  return group;
}

AttentionPlan plan_of(int64_t rows, int32_t heads, int32_t window, int32_t head_dim, const KvBatchArgs& b) {
  int64_t capacity = (int64_t)b.table_width << b.page_shift;
  if (window > 0) capacity = std::min<int64_t>(capacity, (int64_t)window + b.max_rows);
  return attention_plan(rows, group_of(heads, b), b.kv_heads, head_dim, b.sequences, b.max_rows, capacity);
}

struct AttentionWs {
  float* out;
  float2* ml;
  int4* cut;
  int* cut_entry;
  size_t bytes;
};
AttentionWs carve_attention(const AttentionPlan& p, int kv_heads, int head_dim, void* base) {
  AttentionWs w{};
  if (!p.split) return w;
  Carver c(base);
  // Tiles are cut only where they are fewer than the target, into at most that many parts.
  const size_t slots = (size_t)p.target * (size_t)kv_heads * (size_t)p.columns;
  w.out = c.take<float>(slots * (size_t)head_dim);
  w.ml = c.take<float2>(slots);
  w.cut = c.take<int4>((size_t)p.target + 1);
  w.cut_entry = c.take<int>((size_t)p.target);
  w.bytes = align_up(c.offset, 256);
  return w;
}

}  // namespace

extern "C" {

int tfm_rotary(const void* x, int64_t rows, int32_t heads, int32_t head_dim, int64_t row_stride, int64_t head_stride,
               const void* positions, int32_t position_bits, const tfm_rotation* rotation, int32_t dtype, void* out,
               int64_t out_row_stride, int64_t out_head_stride, void* stream) {
  return guarded([&] {
    need_rows(rows);
    need_heads(heads);
    need(head_dim > 0, "head_dim must be positive");
    if (head_dim > kRotaryMaxDim) fail(TFM_E_UNSUPPORTED, "head_dim past 1024 is not built");
    need_storage(dtype);
    need(position_bits == 32 || position_bits == 64, "position_bits must be 32 or 64");
    need_ptr(rotation, "rotation");
    if (rows == 0) return;
    need_rotation(rotation, head_dim);
    need_ptr(positions, "positions");
    const Span in = rows_span(x, rows, heads, head_dim, row_stride, head_stride, "x");
    const Span o = rows_span(out, rows, heads, head_dim, out_row_stride, out_head_stride, "out");
    const int64_t rs = rows > 1 ? out_row_stride : kMaxStride, hs = heads > 1 ? out_head_stride : head_dim;
    const int64_t rs2 = rows > 1 ? out_row_stride : head_dim, hs2 = heads > 1 ? out_head_stride : kMaxStride;
    need((hs >= head_dim && rs >= (heads - 1) * hs + head_dim) || (rs2 >= head_dim && hs2 >= (rows - 1) * rs2 + head_dim),
         "rows of out overlap");
    const bool same = x == out && (rows == 1 || row_stride == out_row_stride) && (heads == 1 || head_stride == out_head_stride);
    need(same || !meet(o, in), "out overlaps an x that it is not");
    need_apart({o}, {{positions, (size_t)rows * (size_t)(position_bits / 8)}, {rotation->frequencies, (size_t)rotation->pairs * 8}},
               "out must not overlap positions or frequencies");
    const RotaryArgs a{static_cast<const uint16_t*>(x), static_cast<uint16_t*>(out), row_stride, head_stride, out_row_stride,
                       out_head_stride, positions, position_bits == 64, rotation->frequencies, rotation->scale, (int)rows,
                       heads, rotation->pairs, same ? 0 : head_dim - 2 * rotation->pairs, rotation->interleaved != 0};
    launch_rotary(dtype == TFM_DTYPE_F16, a, static_cast<hipStream_t>(stream));
  });
}

int tfm_cache_append(const void* k, int64_t k_row_stride, int64_t k_head_stride, const void* v, int64_t v_row_stride,
                     int64_t v_head_stride, int64_t rows, const tfm_rotation* rotation, int32_t dtype,
                     const tfm_kv_cache* cache, const tfm_kv_batch* batch, void* stream) {
  return guarded([&] {
    need_rows(rows);
    need_storage(dtype);
    CacheSpans at{};
    KvAppendArgs a{};
    a.b = need_batch(cache, batch, rows, &at);
    if (rows == 0 || batch->sequences == 0 || batch->max_rows == 0) return;
    Span frequencies{nullptr, 0};
    if (rotation) {
      need_rotation(rotation, cache->head_dim);
      if (rotation->pairs % 8) fail(TFM_E_UNSUPPORTED, "pairs must be a multiple of 8 here (tfm_rotary takes any)");
      frequencies = Span{rotation->frequencies, (size_t)rotation->pairs * 8};
      a.frequencies = rotation->frequencies;
      a.pairs = rotation->pairs;
      a.scale = rotation->scale;
      a.interleaved = rotation->interleaved != 0;
    }
    const Span ks = rows_span(k, rows, cache->kv_heads, cache->head_dim, k_row_stride, k_head_stride, "k");
    const Span vs = rows_span(v, rows, cache->kv_heads, cache->head_dim, v_row_stride, v_head_stride, "v");
    need_apart({at.k, at.v, at.ks, at.vs}, {ks, vs, frequencies, at.table, at.lengths, at.starts},
               "the cache's arrays must not overlap an input or each other");
    a.k = static_cast<const uint16_t*>(k);
    a.v = static_cast<const uint16_t*>(v);
    a.k_row = k_row_stride, a.k_head = k_head_stride, a.v_row = v_row_stride, a.v_head = v_head_stride;
    const int64_t slots = (a.b.max_rows + cache->page_tokens - 2) / cache->page_tokens + 1;
    if (slots * batch->sequences > (1 << 22)) fail(TFM_E_UNSUPPORTED, "sequences * pages of max_rows past 2^22 are not built");
    launch_cache_append(dtype == TFM_DTYPE_F16, cache->head_dim, a, static_cast<hipStream_t>(stream));
  });
}

int tfm_cache_read(const tfm_kv_cache* cache, const tfm_kv_batch* batch, int32_t dtype, void* k, void* v, void* stream) {
  return guarded([&] {
    need(dtype == TFM_DTYPE_BF16 || dtype == TFM_DTYPE_F16 || dtype == TFM_DTYPE_F32, "unknown dtype");
    need_ptr(batch, "batch");
    need(!batch->starts, "starts must be null");
    const int64_t rows = batch->sequences > 0 && batch->max_rows > 0 ? (int64_t)batch->sequences * batch->max_rows : 0;
    need_rows(rows);
    CacheSpans at{};
    const KvBatchArgs a = need_batch(cache, batch, rows, &at);
    if (rows == 0) return;
    need_ptr(k, "k");
    need_ptr(v, "v");
    need_align16(k, "k");
    need_align16(v, "v");
    const size_t bytes = (size_t)rows * (size_t)cache->kv_heads * (size_t)cache->head_dim * size_of(dtype);
    if (rows * cache->kv_heads > ((int64_t)1 << 28)) fail(TFM_E_UNSUPPORTED, "rows * kv_heads past 2^28 is not built");
    need_apart({{k, bytes}, {v, bytes}}, {at.k, at.v, at.ks, at.vs, at.table, at.lengths},
               "k and v must not overlap the cache, the batch or each other");
    launch_cache_read(dtype, cache->head_dim, a, k, v, static_cast<hipStream_t>(stream));
  });
}

size_t tfm_cache_attention_workspace_bytes(int64_t rows, int32_t heads, int32_t window, const tfm_kv_cache* cache,
                                           const tfm_kv_batch* batch) {
  size_t bytes = 0;
  guarded([&] {
    need_rows(rows);
    CacheSpans at{};
    const KvBatchArgs b = need_batch(cache, batch, rows, &at);
    if (rows == 0 || b.sequences == 0 || b.max_rows == 0) return;
    bytes = carve_attention(plan_of(rows, heads, window, cache->head_dim, b), b.kv_heads, cache->head_dim, nullptr).bytes;
  });
  return bytes;  // 0 for arguments that the call refuses
}

int tfm_cache_attention(const void* q, int64_t row_stride, int64_t head_stride, int64_t rows, int32_t heads,
                        const tfm_kv_cache* cache, const tfm_kv_batch* batch, float scale, int32_t causal, int32_t window,
                        int32_t dtype, void* out, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded([&] {
    need_rows(rows);
    need_storage(dtype);
    need(window >= 0, "window must not be negative");
    need(causal || window == 0, "a window needs causal");
    CacheSpans at{};
    AttentionArgs a{};
    a.scale = (float)(scale * kLog2e);
    need(a.scale - a.scale == 0.0f, "scale must be finite, times log2(e) too");
    a.b = need_batch(cache, batch, rows, &at);
    a.group = group_of(heads, a.b);
    if (rows == 0 || batch->sequences == 0 || batch->max_rows == 0) return;
    const Span in = rows_span(q, rows, heads, cache->head_dim, row_stride, head_stride, "q");
    need_ptr(out, "out");
    if (reinterpret_cast<uintptr_t>(out) & 7) fail(TFM_E_INVALID, "out must be 8-byte aligned");
    const AttentionPlan plan = plan_of(rows, heads, window, cache->head_dim, a.b);
    if ((int64_t)plan.items * a.b.kv_heads >= (1 << 24)) fail(TFM_E_UNSUPPORTED, "more than 2^24 tiles of (row, head) are not built");
    const AttentionWs ws = carve_attention(plan, a.b.kv_heads, cache->head_dim, workspace);
    if (ws.bytes) need_ws(workspace, workspace_bytes, ws.bytes);
    const Span o{out, (size_t)rows * (size_t)heads * (size_t)cache->head_dim * 2};
    need_apart({o, {ws.bytes ? workspace : nullptr, ws.bytes}},
               {in, at.k, at.v, at.ks, at.vs, at.table, at.lengths, at.starts},
               "out and workspace must not overlap an input or each other");
    a.q = static_cast<const uint16_t*>(q);
    a.out = static_cast<uint16_t*>(out);
    a.q_row = row_stride;
    a.q_head = head_stride;
    a.heads = heads;
    a.causal = causal != 0;
    a.window = window;
    a.min_chunk = plan.min_chunk;
    a.target = plan.target;
    a.part_out = ws.out;
    a.part_ml = ws.ml;
    a.cut = ws.cut;
    a.cut_entry = ws.cut_entry;
    launch_cache_attention(dtype == TFM_DTYPE_F16, cache->head_dim, plan, a, static_cast<hipStream_t>(stream));
  });
}

}  // extern "C"
