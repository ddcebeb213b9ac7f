// C ABI of the operators around the block: argument checks and launches.
#include <initializer_list>

#include "tfm_internal.h"

using namespace tfm;

namespace {

void need_rows(int64_t rows) { need(rows >= 0 && rows <= kMaxRows, "rows out of range"); }

void need_storage(int32_t dtype) {
  need(dtype == TFM_DTYPE_BF16 || dtype == TFM_DTYPE_F16, "unknown dtype");
}

void need_eps(float eps, const char* name) {
  if (!(eps >= 0.0f) || eps > 3.4e38f) fail(TFM_E_INVALID, std::string(name) + " must be a non-negative number");
}

// The bytes of one buffer; null or empty ones share memory with nothing.
struct Span {
  const void* at;
  size_t bytes;
};
bool meet(const Span& a, const Span& b) {
  const uintptr_t p = reinterpret_cast<uintptr_t>(a.at), q = reinterpret_cast<uintptr_t>(b.at);
  return p && q && (p > q ? p - q < b.bytes : q - p < a.bytes) && a.bytes && b.bytes;
}

// No output shares memory with an input or another output.
void need_apart(std::initializer_list<Span> outs, std::initializer_list<Span> ins, const char* message) {
  for (const Span* o = outs.begin(); o != outs.end(); ++o) {
    for (const Span& in : ins) need(!meet(*o, in), message);
    for (const Span* other = outs.begin(); other != o; ++other) need(!meet(*o, *other), message);
  }
}

size_t size_of(int32_t dtype) { return dtype == TFM_DTYPE_F32 ? 4 : 2; }

constexpr int kProductMaxK = 131056;  // 128 * 128 * K < 2^31

void need_product(int64_t rows, int32_t n_out, int32_t k_in) {
  need_rows(rows);
  need(n_out > 0 && k_in > 0, "n_out and k_in must be positive");
  if (n_out > (1 << 28)) fail(TFM_E_UNSUPPORTED, "n_out past 2^28 is not built");
  if (k_in % 16 != 0) fail(TFM_E_UNSUPPORTED, "k_in must be a multiple of 16");
  if (k_in > kProductMaxK) fail(TFM_E_UNSUPPORTED, "k_in past 131056 could overflow the 32-bit sum");
}

struct LinearWs {
  int8_t* codes;
  float* scales;
  size_t bytes;
};
LinearWs carve_linear(int64_t rows, int32_t k_in, void* base) {
  Carver c(base);
  LinearWs w{};
  w.codes = c.take<int8_t>((size_t)rows * (size_t)k_in);
  w.scales = c.take<float>((size_t)rows);
  w.bytes = align_up(c.offset, 256);
  return w;
}

}  // namespace

extern "C" {

int tfm_norm_residual(const tfm_norm_step* step, int64_t rows, int32_t width, int32_t dtype, void* stream) {
  return guarded([&] {
    need_ptr(step, "step");
    need_rows(rows);
    need(width > 0, "width must be positive");
    if (width > kNormMaxWidth) fail(TFM_E_UNSUPPORTED, "width past 32768 is not built");
    need_storage(dtype);
    need(step->gate_kind >= TFM_GATE_NONE && step->gate_kind <= TFM_GATE_FULL, "unknown gate kind");
    if (step->post_weight) need_eps(step->post_eps, "post_eps");
    if (step->pre_weight) need_eps(step->pre_eps, "pre_eps");
    need(step->residual_multiplier == step->residual_multiplier, "residual_multiplier is not a number");
    if (rows == 0) return;  // empty tensors may have null pointers
    need(step->h || step->x || step->codes, "no output asked for");
    need(step->pre_weight || (!step->x && !step->codes), "x and codes need pre_weight");
    need((step->codes == nullptr) == (step->scales == nullptr), "codes and scales go together");
    need_ptr(step->y, "y");
    if (step->gate_kind != TFM_GATE_NONE) need_ptr(step->gate, "gate");
    const size_t n = (size_t)rows, w = (size_t)width, bytes = n * w * 2;
    const int32_t gk = step->gate_kind;
    const Span y{step->y, bytes}, residual{step->residual, bytes};
    const Span gate{gk == TFM_GATE_NONE ? nullptr : step->gate,
                    gk == TFM_GATE_FULL ? bytes : gk == TFM_GATE_TOKEN ? n * 4 : w * 2};
    const Span post{step->post_weight, w * 2}, pre{step->pre_weight, w * 2};
    const Span h{step->h, bytes}, x{step->x, bytes};
    // Each lane has read its own elements of y, residual and a full gate (or a single row's) before it writes
    // h; weights and the other gates are read by every row.
    const bool full = gk == TFM_GATE_FULL || (gk == TFM_GATE_CHANNEL && rows == 1);
    const Span none{nullptr, 0};
    for (const Span& in : {y, residual, full ? gate : none}) {
      need(h.at == in.at || !meet(h, in), "h overlaps an input that it is not");
      need(!meet(x, in), "x must not alias y, residual or gate");
    }
    need(!meet(x, h), "x must not alias h");
    for (const Span& in : {post, pre, full ? none : gate})
      need(!meet(h, in) && !meet(x, in), "h and x must not overlap a weight or a gate that rows share");
    need_apart({{step->codes, n * w}, {step->scales, n * 4}}, {y, residual, gate, post, pre, h, x},
               "codes and scales must not overlap an input or another output");
    launch_norm_residual(dtype == TFM_DTYPE_F16, *step, (int)rows, width, static_cast<hipStream_t>(stream));
  });
}

int tfm_quantize_rows(const void* x, int64_t rows, int32_t width, int32_t dtype, int8_t* codes, float* scales,
                      void* stream) {
  return guarded([&] {
    need_rows(rows);
    need(width > 0, "width must be positive");
    if (width > kQuantizeMaxWidth) fail(TFM_E_UNSUPPORTED, "width past 131072 is not built");
    need_storage(dtype);
    if (rows == 0) return;
    need_ptr(x, "x");
    need_ptr(codes, "codes");
    need_ptr(scales, "scales");
    const size_t n = (size_t)rows, w = (size_t)width;
    need_apart({{codes, n * w}, {scales, n * 4}}, {{x, n * w * 2}}, "codes and scales must not overlap x or each other");
    launch_quantize_rows(dtype == TFM_DTYPE_F16, static_cast<const uint16_t*>(x), (int)rows, width, codes, scales,
                         static_cast<hipStream_t>(stream));
  });
}

int tfm_int8_qmm(const int8_t* x, const float* x_scales, int64_t rows, const int8_t* w, const float* w_scales,
                 const void* bias, int32_t n_out, int32_t k_in, int32_t dtype, void* out, void* stream) {
  return guarded([&] {
    need_product(rows, n_out, k_in);
    need(dtype == TFM_DTYPE_BF16 || dtype == TFM_DTYPE_F16 || dtype == TFM_DTYPE_F32, "unknown dtype");
    if (rows == 0) return;
    need_ptr(x, "x");
    need_ptr(x_scales, "x_scales");
    need_ptr(w, "w");
    need_ptr(w_scales, "w_scales");
    need_ptr(out, "out");
    need_align16(x, "x");
    need_align16(w, "w");
    const size_t m = (size_t)rows, n = (size_t)n_out, k = (size_t)k_in;
    need_apart({{out, m * n * size_of(dtype)}},
               {{x, m * k}, {x_scales, m * 4}, {w, n * k}, {w_scales, n * 4}, {bias, n * size_of(dtype)}},
               "out must not overlap an input");
    launch_int8_qmm(dtype, x, x_scales, rows, w, w_scales, bias, n_out, k_in, out, static_cast<hipStream_t>(stream));
  });
}

size_t tfm_int8_linear_workspace_bytes(int64_t rows, int32_t k_in) {
  if (rows < 0 || rows > kMaxRows || k_in <= 0 || int8_linear_few(rows, k_in)) return 0;
  return carve_linear(rows, k_in, nullptr).bytes;
}

int tfm_int8_linear(const void* x, int64_t rows, const int8_t* w, const float* w_scales, const void* bias,
                    int32_t n_out, int32_t k_in, int32_t dtype, void* out, void* workspace, size_t workspace_bytes,
                    void* stream) {
  return guarded([&] {
    need_product(rows, n_out, k_in);
    need_storage(dtype);
    if (rows == 0) return;
    need_ptr(x, "x");
    need_ptr(w, "w");
    need_ptr(w_scales, "w_scales");
    need_ptr(out, "out");
    need_align16(w, "w");
    hipStream_t s = static_cast<hipStream_t>(stream);
    const size_t m = (size_t)rows, n = (size_t)n_out, k = (size_t)k_in;
    const Span in{x, m * k * 2}, wq{w, n * k}, wscale{w_scales, n * 4}, b{bias, n * 2}, o{out, m * n * 2};
    if (int8_linear_few(rows, k_in)) {
      need_apart({o}, {in, wq, wscale, b}, "out must not overlap an input");
      launch_int8_linear_few(dtype == TFM_DTYPE_F16, static_cast<const uint16_t*>(x), rows, w, w_scales, bias, n_out,
                             k_in, out, s);
      return;
    }
    const LinearWs ws = carve_linear(rows, k_in, workspace);
    need_ws(workspace, workspace_bytes, ws.bytes);
    need_apart({o, {workspace, ws.bytes}}, {in, wq, wscale, b}, "out and workspace must not overlap an input or each other");
    launch_quantize_rows(dtype == TFM_DTYPE_F16, static_cast<const uint16_t*>(x), (int)rows, k_in, ws.codes, ws.scales,
                         s);
    launch_int8_qmm(dtype, ws.codes, ws.scales, rows, w, w_scales, bias, n_out, k_in, out, s);
  });
}

int tfm_token_logprobs(const void* logits, int64_t rows, int32_t vocab, int64_t row_stride, int32_t dtype,
                       const void* tokens, int32_t token_bits, int32_t top, float scale, float* logprobs,
                       float* entropy, int32_t* top_ids, float* top_logprobs, void* stream) {
  return guarded([&] {
    need_rows(rows);
    need(vocab > 0, "vocab must be positive");
    if (vocab > (1 << 24)) fail(TFM_E_UNSUPPORTED, "vocab past 2^24 is not built");
    need(row_stride >= vocab, "row_stride < vocab");
    need(dtype == TFM_DTYPE_BF16 || dtype == TFM_DTYPE_F16 || dtype == TFM_DTYPE_F32, "unknown dtype");
    need(top >= 0 && top <= vocab, "need 0 <= top <= vocab");
    if (top > 64) fail(TFM_E_UNSUPPORTED, "more than 64 alternatives are not built");
    // Below 1e-35 logits whose difference passes the largest number would still count beside each other.
    need(scale >= 1e-35f && scale <= 1e30f, "scale must be in [1e-35, 1e30]");
    if (rows == 0) return;  // empty tensors may have null pointers
    need((tokens == nullptr) == (logprobs == nullptr), "tokens and logprobs go together");
    need(!tokens || token_bits == 32 || token_bits == 64, "token_bits must be 32 or 64");
    need(logprobs || entropy || top > 0, "no output asked for");
    need_ptr(logits, "logits");
    if (top > 0) {
      need_ptr(top_ids, "top_ids");
      need_ptr(top_logprobs, "top_logprobs");
    }
    const size_t n = (size_t)rows, size = size_of(dtype), k = n * (size_t)top;
    need_apart({{logprobs, n * 4}, {entropy, n * 4}, {top_ids, k * 4}, {top_logprobs, k * 4}},
               {{logits, ((n - 1) * (size_t)row_stride + (size_t)vocab) * size}, {tokens, n * (size_t)(token_bits / 8)}},
               "outputs must not overlap an input or each other");
    const LogprobsArgs a{logits, row_stride,       (int)rows, vocab,   top,     scale,
                         tokens, token_bits == 64, logprobs,  entropy, top_ids, top_logprobs};
    launch_token_logprobs(dtype, a, static_cast<hipStream_t>(stream));
  });
}

}  // extern "C"
