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

import ctypes
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import (TFM_DTYPE_BF16, TFM_DTYPE_F16, TFM_DTYPE_F32, TFM_GATE_CHANNEL, TFM_GATE_FULL, TFM_GATE_NONE,
                   TFM_GATE_TOKEN, NormStep, call)
from .moe import _dev, _dtype_code, _ptr

_FLOATS = {torch.bfloat16: TFM_DTYPE_BF16, torch.float16: TFM_DTYPE_F16, torch.float32: TFM_DTYPE_F32}


# The current stream's handle without a torch.cuda.Stream object around it
# (0.1 against 2 to 3 us of host time a call, of 10 in all).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(device: torch.device, name: str, *args) -> None:
    """An entry point on `device` and its current stream (the last argument)."""
    if device.index == torch.cuda.current_device():
        call(name, *args, _raw_stream(device.index))
    else:
        with torch.cuda.device(device):
            call(name, *args, _raw_stream(device.index))


def _on(t: torch.Tensor, name: str, device: torch.device) -> None:
    if t.device != device or not t.is_contiguous():
        _dev(t, name)
        raise ValueError(f"{name} is on {t.device}, not on {device}")


def _rows(x: torch.Tensor, name: str) -> Tuple[int, int]:
    """(rows, width) of x [..., width]."""
    if x.ndim < 1 or x.shape[-1] == 0:
        raise ValueError(f"{name} must be [..., width] with a positive width")
    width = x.shape[-1]
    return x.numel() // width, width


def _vector(t: Optional[torch.Tensor], name: str, n: int, dtype: torch.dtype, device: torch.device) -> None:
    if t is None:
        return
    _on(t, name, device)
    if t.dtype != dtype or t.ndim != 1 or t.shape[0] != n:
        raise ValueError(f"{name} must be {dtype} [{n}]")


def _codes(shape: torch.Size, device: torch.device) -> Tuple[torch.Tensor, torch.Tensor]:
    return (torch.empty(shape, dtype=torch.int8, device=device),
            torch.empty(shape[:-1], dtype=torch.float32, device=device))


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
    rounding. out receives h and may be y or residual."""
    dt = _dtype_code(y, "y")
    _dev(y, "y")
    rows, width = _rows(y, "y")
    dev = y.device
    if residual is not None:
        _on(residual, "residual", dev)
        if residual.shape != y.shape or residual.dtype != y.dtype:
            raise ValueError("residual geometry/dtype differs")
    _vector(post_weight, "post_weight", width, y.dtype, dev)
    _vector(pre_weight, "pre_weight", width, y.dtype, dev)
    kind = TFM_GATE_NONE
    if gate is not None:
        _on(gate, "gate", dev)
        if gate.dtype == y.dtype and gate.shape == (width,):
            kind = TFM_GATE_CHANNEL
        elif gate.dtype == y.dtype and gate.shape == y.shape:
            kind = TFM_GATE_FULL
        elif gate.dtype == torch.float32 and gate.shape in (y.shape[:-1], (*y.shape[:-1], 1)):
            kind = TFM_GATE_TOKEN
        else:
            raise ValueError("gate must be [H] or y's shape in y's dtype, or fp32 with one value a row")
    if quantize and pre_weight is None:
        raise ValueError("quantize needs pre_weight")
    if out is None:
        out = torch.empty_like(y)
    else:
        _on(out, "out", dev)
        if out.shape != y.shape or out.dtype != y.dtype:
            raise ValueError("out geometry/dtype differs")
    x = codes = scales = None
    if quantize:
        codes, scales = _codes(y.shape, dev)
    elif pre_weight is not None:
        x = torch.empty_like(y)
    step = NormStep(y.data_ptr(), _ptr(residual), _ptr(post_weight), _ptr(gate), _ptr(pre_weight), out.data_ptr(),
                    _ptr(x), _ptr(codes), _ptr(scales), kind, residual_multiplier,
                    eps if post_eps is None else post_eps, eps)
    _call(dev, "tfm_norm_residual", ctypes.byref(step), rows, width, dt)
    if quantize:
        return out, codes, scales
    return out if x is None else (out, x)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float, quantize: bool = False):
    """x * rsqrt(mean(x^2) + eps) * weight over the last axis, rounded once; with
    quantize, its 8-bit codes and scales (as quantize_rows)."""
    dt = _dtype_code(x, "x")
    _dev(x, "x")
    rows, width = _rows(x, "x")
    _vector(weight, "weight", width, x.dtype, x.device)
    y = codes = scales = None
    if quantize:
        codes, scales = _codes(x.shape, x.device)
    else:
        y = torch.empty_like(x)
    step = NormStep(x.data_ptr(), None, None, None, weight.data_ptr(), None, _ptr(y), _ptr(codes), _ptr(scales),
                    TFM_GATE_NONE, 1.0, 0.0, eps)
    _call(x.device, "tfm_norm_residual", ctypes.byref(step), rows, width, dt)
    return (codes, scales) if quantize else y


# ---------------------------------------------------------------------------
# Products in 8-bit integers
# ---------------------------------------------------------------------------

def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """8-bit codes of each row of x [..., K] (tokens, or a weight matrix's channels) and their fp32 scales
    [...]: codes * scales is x to half a step of max|row| / 127."""
    dt = _dtype_code(x, "x")
    _dev(x, "x")
    rows, width = _rows(x, "x")
    codes, scales = _codes(x.shape, x.device)
    _call(x.device, "tfm_quantize_rows", x.data_ptr(), rows, width, dt, codes.data_ptr(), scales.data_ptr())
    return codes, scales


def _int8_weight(w: torch.Tensor, w_scales: torch.Tensor, bias: Optional[torch.Tensor], width: int,
                 dtype: torch.dtype, device: torch.device) -> int:
    _on(w, "w", device)
    if w.dtype != torch.int8 or w.ndim != 2 or w.shape[1] != width or w.shape[0] == 0:
        raise ValueError(f"w must be int8 [n_out, {width}]")
    _vector(w_scales, "w_scales", w.shape[0], torch.float32, device)
    _vector(bias, "bias", w.shape[0], dtype, device)
    return w.shape[0]


def int8_qmm(codes: torch.Tensor, scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor,
             bias: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """(codes . w^T) * scales * w_scales + bias in `dtype` (bf16, f16 or fp32): codes int8 [..., K] with scales
    fp32 [...] (quantize_rows, norm_residual), w int8 [N, K] with w_scales fp32 [N], bias [N] in `dtype`. K is a
    multiple of 16."""
    if dtype not in _FLOATS:
        raise ValueError(f"unknown output dtype {dtype}")
    _dev(codes, "codes")
    if codes.dtype != torch.int8:
        raise ValueError("codes must be int8")
    rows, width = _rows(codes, "codes")
    _on(scales, "scales", codes.device)
    if scales.dtype != torch.float32 or scales.shape != codes.shape[:-1]:
        raise ValueError("scales must be fp32 with one value a row of codes")
    n = _int8_weight(w, w_scales, bias, width, dtype, codes.device)
    out = torch.empty((*codes.shape[:-1], n), dtype=dtype, device=codes.device)
    _call(codes.device, "tfm_int8_qmm", codes.data_ptr(), scales.data_ptr(), rows, w.data_ptr(), w_scales.data_ptr(),
          _ptr(bias), n, width, _FLOATS[dtype], out.data_ptr())
    return out


def int8_linear(x: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor,
                bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x . (w * w_scales)^T + bias in x's dtype, with x [..., K] rounded to 8-bit codes and a scale a row in the
    call: int8_qmm(*quantize_rows(x), ...)."""
    dt = _dtype_code(x, "x")
    _dev(x, "x")
    rows, width = _rows(x, "x")
    n = _int8_weight(w, w_scales, bias, width, x.dtype, x.device)
    out = torch.empty((*x.shape[:-1], n), dtype=x.dtype, device=x.device)
    need = _lib.load().tfm_int8_linear_workspace_bytes(rows, width)
    ws = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    _call(x.device, "tfm_int8_linear", x.data_ptr(), rows, w.data_ptr(), w_scales.data_ptr(), _ptr(bias), n, width, dt,
          out.data_ptr(), _ptr(ws), need)
    return out


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
    of nothing else has entropy 0 and log probabilities -inf."""
    code = _FLOATS.get(logits.dtype)
    if code is None:
        raise NotImplementedError(f"logits: only bf16, f16 and fp32 are built (got {logits.dtype})")
    if not logits.is_cuda:
        raise ValueError("logits must be a GPU tensor (the MoE path has no CPU fallback)")
    rows, vocab = _rows(logits, "logits")
    stride = vocab
    if not logits.is_contiguous():
        if logits.ndim != 2 or (logits.stride(1) != 1 and vocab > 1):
            raise ValueError("logits must be contiguous, or 2-D with contiguous rows")
        stride = logits.stride(0) if rows > 1 else vocab
    if type(top) is not int or not 0 <= top <= vocab:
        raise ValueError("Invalid top-k")
    dev, lead = logits.device, logits.shape[:-1]
    entropy = torch.empty(lead, dtype=torch.float32, device=dev)
    ids = torch.empty((*lead, top), dtype=torch.int32, device=dev)
    best = torch.empty_like(ids, dtype=torch.float32)
    logprobs = None
    if tokens is not None:
        _on(tokens, "tokens", dev)
        if tokens.dtype not in (torch.int32, torch.int64) or tokens.shape != lead:
            raise ValueError("tokens must be int32 or int64 with one value a row of logits")
        logprobs = torch.empty_like(entropy)
    _call(dev, "tfm_token_logprobs", logits.data_ptr(), rows, vocab, stride, code, _ptr(tokens),
          64 if tokens is not None and tokens.dtype == torch.int64 else 32, top, scale, _ptr(logprobs),
          entropy.data_ptr(), ids.data_ptr(), best.data_ptr())
    return logprobs, entropy, ids, best
