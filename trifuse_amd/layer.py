"""The operators of a decoder layer around its MoE block, over the HIP library.

What stands between two blocks and behind the last one (tfm_norm_residual,
tfm_quantize_rows, tfm_int8_qmm, tfm_int8_linear and tfm_token_logprobs of
include/trifuse_moe.h, which has the exact definitions):

* ``rms_norm`` and ``norm_residual``: the norm in front of a block, and in one
  pass the norm behind it, its gate, the scaled residual and the next block's
  norm, which can come out as 8-bit codes;
* ``quantize_rows``, ``int8_qmm`` and ``int8_linear``: rows to 8-bit codes with
  a scale each, and products of such rows with weights of the same form (a
  scale for each token and for each channel), beside the group-wise
  ``moe.native_affine_qmm``;
* ``token_logprobs``: log probabilities of given tokens, entropy and the most
  likely alternatives, from the output head's logits.

Tensors are torch tensors of one HIP device; work is enqueued on that device's
current stream. There is no CPU fallback and no backward. Every sum, norm and
softmax is held in fp32 (products in int32) and each output is rounded once.
"""
from __future__ import annotations

from typing import Optional, Tuple

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
