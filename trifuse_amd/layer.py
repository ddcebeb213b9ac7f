"""The operators of a decoder layer around its MoE block, over the HIP library.

What stands between two blocks and behind the last one (tfm_norm_residual,
tfm_quantize_rows, tfm_int8_qmm, tfm_int8_linear, tfm_token_logprobs, tfm_rotary and
the tfm_cache_* calls of include/trifuse_moe.h, which has the exact definitions):

* ``rms_norm`` and ``norm_residual``: the norm in front of a block, and in one
  pass the norm behind it, its gate, the scaled residual and the next block's
  norm, which can come out as 8-bit codes;
* ``quantize_rows``, ``int8_qmm`` and ``int8_linear``: rows to 8-bit codes with
  a scale each, and products of such rows with weights of the same form (a
  scale for each token and for each channel), beside the group-wise
  ``moe.native_affine_qmm``;
* ``token_logprobs``: log probabilities of given tokens, entropy and the most
  likely alternatives, from the output head's logits;
* ``rotary``, ``KVCache``, ``cache_append``, ``cache_read`` and ``cache_attention``:
  from the fused projection's queries, keys and values to the output projection's
  input, over a paged cache of 8-bit codes with a scale for each page and head.

Tensors are torch tensors of one HIP device; work is enqueued on that device's
current stream. There is no CPU fallback and no backward. Every sum, norm and
softmax statistic is held in fp32 (8-bit products in int32) and each output is
rounded once; ``cache_attention`` multiplies with softmax weights as halves.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib

# A small call is bound by its host time: arguments are checked and outputs
# allocated in native code (csrc/layer_binding.cpp), and the current device and
# stream are asked for as numbers (0.1 us each; a torch.cuda.Stream object takes
# 2 to 3). One row: norm_residual about 5 us a call, int8_linear about 4 (4.7 to 5.5 and
# 3.6 to 4.5, by the host), against 8.8 and 7.8 with both in Python.
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_native = None


def _enqueue(name: str, x: torch.Tensor, *args):
    """The native operator on x's device and that device's current stream."""
    global _native
    if _native is None:
        _native = _lib.load_layer()
    op = getattr(_native, name)
    index = x.get_device()
    if index < 0:  # refused there
        return op(0, x, *args)
    if index == _current_device():
        return op(_raw_stream(index), x, *args)
    with torch.cuda.device(index):
        return op(_raw_stream(index), x, *args)


# ---------------------------------------------------------------------------
# Norms and residuals
# ---------------------------------------------------------------------------

def norm_residual(y: torch.Tensor, residual: Optional[torch.Tensor] = None, *,
                  post_weight: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                  residual_multiplier: float = 1.0, pre_weight: Optional[torch.Tensor] = None, eps: float = 1e-5,
                  post_eps: Optional[float] = None, quantize: bool = False, out: Optional[torch.Tensor] = None):
    """h = residual + residual_multiplier * gate * post(y), and the next block's input x = pre(h).

    y [..., H] bf16 or f16; residual like y (None: zero). post(y) is the RMSNorm
    of y with post_weight [H] (None: y itself) and post_eps (None: eps). gate:
    None, [H] or y's shape in y's dtype, or one fp32 value a row (y's leading
    shape, or that with a 1). Returns h without pre_weight; (h, x) with
    pre_weight [H]; (h, codes, scales) with quantize, codes int8 in y's shape
    and scales fp32 in its leading shape. x is normed from h before its
    rounding. out receives h and may be y, residual or a gate in y's shape; it shares no
    other memory with an input."""
    return _enqueue("norm_residual", y, residual, post_weight, gate, residual_multiplier, pre_weight, eps, post_eps,
                    quantize, out)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float, quantize: bool = False):
    """x * rsqrt(mean(x^2) + eps) * weight over the last axis, rounded once; with
    quantize, its 8-bit codes and scales (as quantize_rows)."""
    return _enqueue("rms_norm", x, weight, eps, quantize)


# ---------------------------------------------------------------------------
# Products in 8-bit integers
# ---------------------------------------------------------------------------

def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """8-bit codes of each row of x [..., K] (tokens, or a weight matrix's channels) and their fp32 scales
    [...]: codes * scales is x to half a step of max|row| / 127."""
    return _enqueue("quantize_rows", x)


def int8_qmm(codes: torch.Tensor, scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor,
             bias: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """(codes . w^T) * scales * w_scales + bias in `dtype` (bf16, f16 or fp32): codes int8 [..., K] with scales
    fp32 [...] (quantize_rows, norm_residual), w int8 [N, K] with w_scales fp32 [N], bias [N] in `dtype`. K is a
    multiple of 16."""
    return _enqueue("int8_qmm", codes, scales, w, w_scales, bias, dtype)


def int8_linear(x: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor,
                bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x . (w * w_scales)^T + bias in x's dtype, with x [..., K] rounded to 8-bit codes and a scale a row in the
    call: int8_qmm(*quantize_rows(x), ...)."""
    return _enqueue("int8_linear", x, w, w_scales, bias)


# ---------------------------------------------------------------------------
# Log probabilities
# ---------------------------------------------------------------------------

def token_logprobs(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, top: int = 0, scale: float = 1.0):
    """(logprobs, entropy, top_ids, top_logprobs) of softmax(scale * logits) over the last axis.

    logits [..., V] bf16, f16 or fp32: contiguous, or 2-D with unit stride in a
    row (a padded vocabulary's logits[:, :V]). tokens int32 or int64 in the
    leading shape: logprobs, fp32 in that shape, NaN for a token outside
    [0, V) (None without tokens). entropy is fp32 in the leading shape, in nats.
    top_ids (int32) and top_logprobs (fp32) [..., top] are the `top` largest
    logits, largest first, ties to the lower id. Masked logits are -inf; a row
    of nothing else has entropy 0 and log probabilities -inf. scale: 1e-35 to 1e30."""
    return _enqueue("token_logprobs", logits, tokens, top, scale)


# ---------------------------------------------------------------------------
# Rotary positions and attention over an 8-bit cache
# ---------------------------------------------------------------------------

def rotary_frequencies(pairs: int, base: float = 10000.0, *, stretch: float = 1.0, method: str = "linear",
                       context: Optional[int] = None, slow: float = 1.0, fast: float = 32.0,
                       device=None) -> Tuple[torch.Tensor, float]:
    """(frequencies fp64 [pairs], scale) for ``rotary``: base ** (-i / pairs) radians a position, and for a context
    ``stretch`` times as long as the one that a model was trained on

    * "linear": every frequency divided by stretch; scale 1;
    * "base": base multiplied by stretch ** (pairs / (pairs - 1)), which keeps the fastest pair and slows the
      slowest to 1 / stretch; scale 1;
    * "bands": a pair that turns at least ``fast`` times over the trained ``context`` keeps its frequency, one
      that turns at most ``slow`` times has it divided by stretch, between them the two are mixed, linearly in the
      turns; scale 0.1 ln(stretch) + 1. A model trained with another mixture (linear in the pair's number, say)
      needs frequencies of its own."""
    if pairs < 1:
        raise ValueError("pairs must be positive")
    if not (base > 0 and stretch >= 1 and math.isfinite(base) and math.isfinite(stretch)):
        raise ValueError("base must be positive and stretch at least 1")
    if method not in ("linear", "base", "bands"):
        raise ValueError(f"unknown method {method!r}")
    if method == "base":
        base = base * stretch ** (pairs / max(pairs - 1, 1))
    f = float(base) ** (-torch.arange(pairs, dtype=torch.float64) / pairs)
    scale = 1.0
    if method == "linear":
        f = f / stretch
    elif method == "bands":
        if not context or context < 1 or not fast > slow:
            raise ValueError("bands need the trained context and fast > slow")
        kept = ((f * (context / (2 * math.pi)) - slow) / (fast - slow)).clamp(0, 1)
        f = f * (kept + (1 - kept) / stretch)
        scale = 0.1 * math.log(stretch) + 1.0
    return f.to(device), scale


def rotary(x: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor, *, interleaved: bool = False,
           scale: float = 1.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Pairs of a head's channels turned by position * frequency: (x1 c - x2 s, x2 c + x1 s) with c = scale * cos and
    s = scale * sin, angles in 64 bits, rounded once.

    x [rows, heads, head_dim] bf16 or f16, any strides of rows and heads (a view into a fused projection);
    positions int32 or int64 [rows]; frequencies fp64 [pairs] (``rotary_frequencies``), 2 * pairs <= head_dim: pair i
    is channels (i, pairs + i), or (2i, 2i + 1) with interleaved, and channels behind the pairs are copied. out may
    be x itself; a new one is contiguous."""
    return _enqueue("rotary", x, positions, frequencies, interleaved, scale, out)


class KVCache(NamedTuple):
    """A pool of pages of keys and values: int8 codes [pages, kv_heads, page_tokens, head_dim] and fp32 scales
    [pages, kv_heads] of each (value = code * scale). page_tokens: 16, 32, 64, 128 or 256; head_dim: 64 or 128.
    Pages need no clearing: the first token of a page starts its scale anew."""
    k: torch.Tensor
    v: torch.Tensor
    k_scales: torch.Tensor
    v_scales: torch.Tensor

    @classmethod
    def empty(cls, pages: int, kv_heads: int, page_tokens: int, head_dim: int, device="cuda") -> "KVCache":
        codes = (pages, kv_heads, page_tokens, head_dim)
        return cls(*(torch.zeros(codes, dtype=torch.int8, device=device) for _ in "kv"),
                   *(torch.zeros(codes[:2], dtype=torch.float32, device=device) for _ in "kv"))


def cache_append(k: torch.Tensor, v: torch.Tensor, cache: KVCache, table: torch.Tensor, lengths: torch.Tensor, *,
                 starts: Optional[torch.Tensor] = None, max_rows: Optional[int] = None,
                 frequencies: Optional[torch.Tensor] = None, interleaved: bool = False,
                 rotary_scale: float = 1.0) -> None:
    """Writes a step's keys and values [rows, kv_heads, head_dim] (bf16 or f16, any strides of rows and heads) into
    the cache, keys turned to their positions first where frequencies (as ``rotary``, pairs a multiple of 8) are given.

    Sequence b has lengths[b] tokens (int32) with this step's, token t in page table[b, t // page_tokens] (int32
    [sequences, width]). Its rows are starts[b] : starts[b + 1] (int32 [sequences + 1], max_rows at least the most of
    one sequence; None: all rows), the last of its tokens; without starts every sequence has the same number.
    A page and head takes the larger of its scale and max|x| / 127 of its new tokens; codes that it
    held are rounded to a larger scale. An infinity or a NaN makes the page NaN. Pages are not shared between
    sequences that write to them in one call. A token past its table row's end is not written."""
    _enqueue("cache_append", k, v, *cache, table, lengths, starts, max_rows, frequencies, interleaved, rotary_scale)


def cache_read(cache: KVCache, table: torch.Tensor, lengths: torch.Tensor, rows: int,
               dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """(k, v) [sequences * rows, kv_heads, head_dim] in `dtype` (bf16, f16 or fp32): the last `rows` tokens of every
    sequence as the values that their codes stand for, to be kept elsewhere. Tokens before the first, and past the
    table row's end, are zero."""
    return _enqueue("cache_read", cache.k, *cache[1:], table, lengths, rows, dtype)


def cache_attention(q: torch.Tensor, cache: KVCache, table: torch.Tensor, lengths: torch.Tensor, *,
                    starts: Optional[torch.Tensor] = None, max_rows: Optional[int] = None,
                    scale: Optional[float] = None, causal: bool = True, window: int = 0,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale * q . k) v over the cached tokens that each row sees, in q's dtype and shape.

    q [rows, heads, head_dim] bf16 or f16, any strides of rows and heads, heads a multiple of the cache's; table,
    lengths, starts and max_rows as in ``cache_append``, behind which it goes: row i of n of sequence b is at position
    lengths[b] - n + i, and sees tokens up to its own (causal) or all of its sequence, with window > 0 (causal) the
    last `window` of them. A row that sees none is zero; rows behind the last sequence are not written. scale: None
    is head_dim ** -0.5. Softmax weights are halves: 2^-11 of themselves, and a token more than 23 below a row's top
    score (in nats) has none. Pass max_rows with starts where it is known: it picks the kernel, as the table's width does
    (a table about as wide as the longest sequence is served best)."""
    return _enqueue("cache_attention", q, *cache, table, lengths, starts, max_rows, scale, causal, window, out)
