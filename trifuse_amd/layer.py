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
from typing import NoReturn, Optional, Tuple

import torch

from . import _lib
from ._lib import (TFM_DTYPE_BF16, TFM_DTYPE_F16, TFM_DTYPE_F32, TFM_GATE_CHANNEL, TFM_GATE_FULL, TFM_GATE_NONE,
                   TFM_GATE_TOKEN, NormStep)
from .moe import _DTYPES, _dev, _dtype_code

_FLOATS = {torch.bfloat16: TFM_DTYPE_BF16, torch.float16: TFM_DTYPE_F16, torch.float32: TFM_DTYPE_F32}

# A small call is bound by its host time, so the checks below read each
# attribute once and say what is wrong on a path of their own, and the current
# device and stream are asked for as numbers (0.1 us each; a torch.cuda.Stream
# object takes 2 to 3).
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(device: torch.device, name: str, *args) -> None:
    """An entry point on `device` and its current stream (the last argument)."""
    index = device.index
    if index == _current_device():
        _lib.call(name, *args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            _lib.call(name, *args, _raw_stream(index))


def _rows(x: torch.Tensor, name: str, code: Optional[int], floats: bool = True) -> Tuple[int, int, torch.device]:
    """(rows, width, device) of x [..., width], contiguous on a GPU and, with floats, of a built dtype."""
    if floats and code is None:
        _dtype_code(x, name)
    if not x.is_cuda or not x.is_contiguous():
        _dev(x, name)
    width = x.shape[-1] if x.ndim else 0
    if not width:
        raise ValueError(f"{name} must be [..., width] with a positive width")
    return x.numel() // width, width, x.device


def _refuse(t: torch.Tensor, name: str, device: torch.device, what: str) -> NoReturn:
    _dev(t, name)
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    raise ValueError(f"{name} must be {what}")


def _vector(t: torch.Tensor, name: str, n: int, dtype: torch.dtype, device: torch.device) -> int:
    """Address of t [n]."""
    if t.dtype is not dtype or t.numel() != n or t.ndim != 1 or not t.is_contiguous() or t.device != device:
        _refuse(t, name, device, f"{dtype} [{n}]")
    return t.data_ptr()


def _like(t: torch.Tensor, name: str, y: torch.Tensor, device: torch.device) -> int:
    """Address of t, of y's shape and dtype."""
    if t.dtype is not y.dtype or t.shape != y.shape or not t.is_contiguous() or t.device != device:
        _refuse(t, name, device, "of the same geometry and dtype")
    return t.data_ptr()


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
    dt = _DTYPES.get(y.dtype)
    rows, width, dev = _rows(y, "y", dt)
    r = None if residual is None else _like(residual, "residual", y, dev)
    post = None if post_weight is None else _vector(post_weight, "post_weight", width, y.dtype, dev)
    pre = None if pre_weight is None else _vector(pre_weight, "pre_weight", width, y.dtype, dev)
    kind, g = TFM_GATE_NONE, None
    if gate is not None:
        kind, g = _gate_of(gate, y, width, dev)
    if out is None:
        out = torch.empty_like(y)
        h = out.data_ptr()
    else:
        h = _like(out, "out", y, dev)
    x = codes = scales = xp = cp = sp = None
    if quantize:
        if pre is None:
            raise ValueError("quantize needs pre_weight")
        codes, scales = _codes(y.shape, dev)
        cp, sp = codes.data_ptr(), scales.data_ptr()
    elif pre is not None:
        x = torch.empty_like(y)
        xp = x.data_ptr()
    step = NormStep(y.data_ptr(), r, post, g, pre, h, xp, cp, sp, kind, residual_multiplier,
                    eps if post_eps is None else post_eps, eps)
    _call(dev, "tfm_norm_residual", ctypes.byref(step), rows, width, dt)
    if quantize:
        return out, codes, scales
    return out if x is None else (out, x)


def _gate_of(gate: torch.Tensor, y: torch.Tensor, width: int, device: torch.device) -> Tuple[int, int]:
    """(TFM_GATE_*, address)."""
    if not gate.is_contiguous() or gate.device != device:
        _refuse(gate, "gate", device, "contiguous")
    if gate.dtype is y.dtype and gate.ndim == 1 and gate.numel() == width:
        return TFM_GATE_CHANNEL, gate.data_ptr()
    if gate.dtype is y.dtype and gate.shape == y.shape:
        return TFM_GATE_FULL, gate.data_ptr()
    if gate.dtype is torch.float32 and gate.shape in (y.shape[:-1], (*y.shape[:-1], 1)):
        return TFM_GATE_TOKEN, gate.data_ptr()
    raise ValueError("gate must be [H] or y's shape in y's dtype, or fp32 with one value a row")


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float, quantize: bool = False):
    """x * rsqrt(mean(x^2) + eps) * weight over the last axis, rounded once; with
    quantize, its 8-bit codes and scales (as quantize_rows)."""
    dt = _DTYPES.get(x.dtype)
    rows, width, dev = _rows(x, "x", dt)
    w = _vector(weight, "weight", width, x.dtype, dev)
    if quantize:
        codes, scales = _codes(x.shape, dev)
        step = NormStep(x.data_ptr(), None, None, None, w, None, None, codes.data_ptr(), scales.data_ptr(),
                        TFM_GATE_NONE, 1.0, 0.0, eps)
    else:
        y = torch.empty_like(x)
        step = NormStep(x.data_ptr(), None, None, None, w, None, y.data_ptr(), None, None, TFM_GATE_NONE, 1.0, 0.0, eps)
    _call(dev, "tfm_norm_residual", ctypes.byref(step), rows, width, dt)
    return (codes, scales) if quantize else y


# ---------------------------------------------------------------------------
# Products in 8-bit integers
# ---------------------------------------------------------------------------

def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """8-bit codes of each row of x [..., K] (tokens, or a weight matrix's channels) and their fp32 scales
    [...]: codes * scales is x to half a step of max|row| / 127."""
    dt = _DTYPES.get(x.dtype)
    rows, width, dev = _rows(x, "x", dt)
    codes, scales = _codes(x.shape, dev)
    _call(dev, "tfm_quantize_rows", x.data_ptr(), rows, width, dt, codes.data_ptr(), scales.data_ptr())
    return codes, scales


def _weight(w: torch.Tensor, width: int, device: torch.device) -> int:
    """Channels of w [n_out, width]."""
    if (w.dtype is not torch.int8 or w.ndim != 2 or w.shape[1] != width or not w.is_contiguous() or w.device != device
            or not w.shape[0]):
        _refuse(w, "w", device, f"int8 [n_out, {width}]")
    return w.shape[0]


def int8_qmm(codes: torch.Tensor, scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor,
             bias: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """(codes . w^T) * scales * w_scales + bias in `dtype` (bf16, f16 or fp32): codes int8 [..., K] with scales
    fp32 [...] (quantize_rows, norm_residual), w int8 [N, K] with w_scales fp32 [N], bias [N] in `dtype`. K is a
    multiple of 16."""
    if dtype not in _FLOATS:
        raise ValueError(f"unknown output dtype {dtype}")
    rows, width, dev = _rows(codes, "codes", None, floats=False)
    if codes.dtype is not torch.int8:
        raise ValueError("codes must be int8")
    if (scales.dtype is not torch.float32 or scales.shape != codes.shape[:-1] or not scales.is_contiguous()
            or scales.device != dev):
        _refuse(scales, "scales", dev, "fp32 with one value a row of codes")
    n = _weight(w, width, dev)
    ws = _vector(w_scales, "w_scales", n, torch.float32, dev)
    b = None if bias is None else _vector(bias, "bias", n, dtype, dev)
    out = torch.empty((*codes.shape[:-1], n), dtype=dtype, device=dev)
    _call(dev, "tfm_int8_qmm", codes.data_ptr(), scales.data_ptr(), rows, w.data_ptr(), ws, b, n, width,
          _FLOATS[dtype], out.data_ptr())
    return out


def int8_linear(x: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor,
                bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x . (w * w_scales)^T + bias in x's dtype, with x [..., K] rounded to 8-bit codes and a scale a row in the
    call: int8_qmm(*quantize_rows(x), ...)."""
    dt = _DTYPES.get(x.dtype)
    rows, width, dev = _rows(x, "x", dt)
    n = _weight(w, width, dev)
    scales = _vector(w_scales, "w_scales", n, torch.float32, dev)
    b = None if bias is None else _vector(bias, "bias", n, x.dtype, dev)
    out = torch.empty((*x.shape[:-1], n), dtype=x.dtype, device=dev)
    need = _lib.load().tfm_int8_linear_workspace_bytes(rows, width)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _call(dev, "tfm_int8_linear", x.data_ptr(), rows, w.data_ptr(), scales, b, n, width, dt, out.data_ptr(),
          ws.data_ptr() if need else None, need)
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
    vocab = logits.shape[-1] if logits.ndim else 0
    if not vocab:
        raise ValueError("logits must be [..., vocab] with a positive vocab")
    rows = logits.numel() // vocab
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
    logprobs, at, bits, to = None, None, 64, None
    if tokens is not None:
        bits = 64 if tokens.dtype is torch.int64 else 32
        if (bits == 32 and tokens.dtype is not torch.int32) or tokens.shape != lead or not tokens.is_contiguous() \
                or tokens.device != dev:
            _refuse(tokens, "tokens", dev, "int32 or int64 with one value a row of logits")
        logprobs = torch.empty_like(entropy)
        at, to = tokens.data_ptr(), logprobs.data_ptr()
    _call(dev, "tfm_token_logprobs", logits.data_ptr(), rows, vocab, stride, code, at, bits, top, scale, to,
          entropy.data_ptr(), ids.data_ptr(), best.data_ptr())
    return logprobs, entropy, ids, best
