"""The entry points around the block on the host (no GPU): refusals before any device work, and the host
mirror's checks."""
import ctypes

import pytest

from trifuse_amd import _lib

P = 4096  # a non-null pointer that is never dereferenced
BF16, F16, F32 = _lib.TFM_DTYPE_BF16, _lib.TFM_DTYPE_F16, _lib.TFM_DTYPE_F32


def check(status, code, msg):
    assert status == code, _lib.load().tfm_last_error()
    if code:
        assert msg in _lib.load().tfm_last_error().decode()


def step(**kw):
    a = dict(y=P, residual=None, post_weight=None, gate=None, pre_weight=None, h=P, x=None, codes=None, scales=None,
             gate_kind=_lib.TFM_GATE_NONE, residual_multiplier=1.0, post_eps=1e-5, pre_eps=1e-5)
    a.update(kw)
    return _lib.NormStep(**a)


@pytest.mark.parametrize("kw,rows,width,dtype,code,msg", [
    (dict(), -1, 64, BF16, 1, "rows"),
    (dict(), 1 << 22, 64, BF16, 1, "rows"),
    (dict(), 1, 0, BF16, 1, "width"),
    (dict(), 1, 32769, BF16, 2, "width"),
    (dict(), 1, 64, F32, 1, "dtype"),
    (dict(gate_kind=4), 1, 64, BF16, 1, "gate kind"),
    (dict(gate_kind=1), 1, 64, BF16, 1, "gate is null"),
    (dict(post_weight=P, post_eps=-1.0), 1, 64, BF16, 1, "post_eps"),
    (dict(pre_weight=P, pre_eps=float("nan")), 1, 64, BF16, 1, "pre_eps"),
    (dict(residual_multiplier=float("nan")), 1, 64, BF16, 1, "residual_multiplier"),
    (dict(h=None), 1, 64, BF16, 1, "no output"),
    (dict(x=P + 4096), 1, 64, BF16, 1, "pre_weight"),
    (dict(pre_weight=P, codes=P), 1, 64, BF16, 1, "codes and scales"),
    (dict(pre_weight=P, scales=P), 1, 64, BF16, 1, "codes and scales"),
    (dict(y=None), 1, 64, BF16, 1, "y is null"),
    (dict(pre_weight=P, x=P), 1, 64, BF16, 1, "alias"),
    (dict(h=P + 64), 1, 64, BF16, 1, "overlaps"),
    (dict(h=P - 2), 1, 64, BF16, 1, "overlaps"),
    (dict(y=P + 65536, residual=P + 100), 1, 64, BF16, 1, "overlaps"),
    (dict(y=P + 65536, gate=P + 1024, gate_kind=3), 9, 64, BF16, 1, "overlaps"),
    (dict(pre_weight=P, h=P + 65536, x=P + 65540), 1, 64, BF16, 1, "alias h"),
    (dict(pre_weight=P, h=P + 65536, x=P + 126), 1, 64, BF16, 1, "alias y"),
    (dict(y=None), 0, 64, BF16, 0, ""),
])
def test_norm_residual_rejects(kw, rows, width, dtype, code, msg):
    s = step(**kw)
    check(_lib.load().tfm_norm_residual(ctypes.byref(s), rows, width, dtype, None), code, msg)


def test_norm_residual_needs_a_step():
    check(_lib.load().tfm_norm_residual(None, 1, 64, BF16, None), 1, "step")


@pytest.mark.parametrize("x,rows,width,dtype,codes,scales,code,msg", [
    (P, -1, 64, BF16, P, P, 1, "rows"),
    (P, 1, 0, BF16, P, P, 1, "width"),
    (P, 1, 131073, BF16, P, P, 2, "width"),
    (P, 1, 64, F32, P, P, 1, "dtype"),
    (None, 1, 64, F16, P, P, 1, "x is null"),
    (P, 1, 64, F16, None, P, 1, "codes"),
    (P, 1, 64, F16, P, None, 1, "scales"),
    (None, 0, 64, F16, None, None, 0, ""),
])
def test_quantize_rows_rejects(x, rows, width, dtype, codes, scales, code, msg):
    check(_lib.load().tfm_quantize_rows(x, rows, width, dtype, codes, scales, None), code, msg)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(rows=-1), 1, "rows"),
    (dict(n=0), 1, "n_out"),
    (dict(n=(1 << 28) + 1), 2, "n_out"),
    (dict(k=0), 1, "k_in"),
    (dict(k=24), 2, "multiple of 16"),
    (dict(k=131072), 2, "overflow"),
    (dict(dtype=7), 1, "dtype"),
    (dict(x=None), 1, "x is null"),
    (dict(xs=None), 1, "x_scales"),
    (dict(w=None), 1, "w is null"),
    (dict(ws=None), 1, "w_scales"),
    (dict(out=None), 1, "out"),
    (dict(x=P + 8), 1, "x must be 16-byte aligned"),
    (dict(w=P + 1), 1, "w must be 16-byte aligned"),
    (dict(rows=0, x=None, out=None), 0, ""),
])
def test_int8_qmm_rejects(kw, code, msg):
    a = dict(x=P, xs=P, rows=2, w=P, ws=P, bias=None, n=64, k=64, dtype=F32, out=P)
    a.update(kw)
    check(_lib.load().tfm_int8_qmm(a["x"], a["xs"], a["rows"], a["w"], a["ws"], a["bias"], a["n"], a["k"], a["dtype"],
                                   a["out"], None), code, msg)


def test_int8_linear_rejects():
    lib = _lib.load()
    need = lib.tfm_int8_linear_workspace_bytes(500, 256)
    assert need >= 500 * 256 + 500 * 4 and lib.tfm_int8_linear_workspace_bytes(-1, 256) == 0
    assert lib.tfm_int8_linear_workspace_bytes(1, 256) == 0
    check(lib.tfm_int8_linear(P, 500, P, P, None, 64, 256, F32, P, P, need, None), 1, "dtype")
    check(lib.tfm_int8_linear(P, 500, P, P, None, 64, 256, BF16, P, P, need - 1, None), 3, "too small")
    check(lib.tfm_int8_linear(P, 500, P, P, None, 64, 256, BF16, P, P + 16, need, None), 3, "aligned")
    check(lib.tfm_int8_linear(P, 500, P, P, None, 64, 256, BF16, P, None, need, None), 3, "null")
    check(lib.tfm_int8_linear(None, 500, P, P, None, 64, 256, BF16, P, P, need, None), 1, "x is null")
    check(lib.tfm_int8_linear(P, 500, P, P, None, 64, 250, BF16, P, P, need, None), 2, "multiple of 16")
    check(lib.tfm_int8_linear(None, 0, None, None, None, 64, 256, BF16, None, None, 0, None), 0, "")


@pytest.mark.parametrize("kw,code,msg", [
    (dict(rows=-1), 1, "rows"),
    (dict(vocab=0), 1, "vocab"),
    (dict(vocab=(1 << 24) + 1, stride=1 << 25), 2, "vocab"),
    (dict(stride=99), 1, "row_stride"),
    (dict(dtype=3), 1, "dtype"),
    (dict(top=-1), 1, "top"),
    (dict(top=101), 1, "top"),
    (dict(vocab=1000, stride=1000, top=65), 2, "64 alternatives"),
    (dict(scale=0.0), 1, "scale"),
    (dict(scale=-1.0), 1, "scale"),
    (dict(scale=float("inf")), 1, "scale"),
    (dict(scale=float("nan")), 1, "scale"),
    (dict(tokens=None), 1, "tokens and logprobs"),
    (dict(logprobs=None), 1, "tokens and logprobs"),
    (dict(bits=16), 1, "token_bits"),
    (dict(tokens=None, logprobs=None, entropy=None, top=0), 1, "no output"),
    (dict(logits=None), 1, "logits"),
    (dict(ids=None), 1, "top_ids"),
    (dict(best=None), 1, "top_logprobs"),
    (dict(rows=0, logits=None), 0, ""),
])
def test_token_logprobs_rejects(kw, code, msg):
    a = dict(logits=P, rows=2, vocab=100, stride=100, dtype=BF16, tokens=P, bits=64, top=4, scale=1.0, logprobs=P,
             entropy=P, ids=P, best=P)
    a.update(kw)
    check(_lib.load().tfm_token_logprobs(a["logits"], a["rows"], a["vocab"], a["stride"], a["dtype"], a["tokens"],
                                         a["bits"], a["top"], a["scale"], a["logprobs"], a["entropy"], a["ids"],
                                         a["best"], None), code, msg)


def test_host_mirror_refuses_cpu_tensors_and_other_types():
    import torch

    from trifuse_amd import layer

    x = torch.zeros((3, 64), dtype=torch.bfloat16)
    w = torch.zeros((8, 64), dtype=torch.int8)
    s = torch.ones(8)
    for f in (lambda: layer.rms_norm(x, x[0], 1e-5), lambda: layer.norm_residual(x, x), lambda: layer.quantize_rows(x),
              lambda: layer.int8_linear(x, w, s), lambda: layer.int8_qmm(w, s, w, s), lambda: layer.token_logprobs(x)):
        with pytest.raises(ValueError, match="GPU tensor"):
            f()
    for f in (lambda: layer.norm_residual(x.double()), lambda: layer.quantize_rows(x.float()),
              lambda: layer.int8_linear(x.float(), w, s), lambda: layer.token_logprobs(x.double())):
        with pytest.raises(NotImplementedError):
            f()


def test_native_host_side_refuses_what_is_no_tensor():
    import torch

    from trifuse_amd import _lib as lib

    native = lib.load_layer()
    assert lib.load_layer() is native
    x = torch.zeros((3, 64), dtype=torch.bfloat16)
    for f in (lambda: native.quantize_rows(0, None), lambda: native.quantize_rows(0), lambda: native.quantize_rows(0, 1.5),
              lambda: native.rms_norm(0, [x], None, 1e-5, False)):
        with pytest.raises(TypeError):
            f()
    with pytest.raises(lib.TfmUnsupported):
        lib.raise_status(lib.TFM_E_UNSUPPORTED)
    with pytest.raises(lib.TfmError):
        lib.raise_status(lib.TFM_E_INVALID)


@pytest.mark.parametrize("kw", [
    dict(post_weight=P), dict(post_weight=P + 64), dict(pre_weight=P + 9 * 128 - 2), dict(pre_weight=P - 126),
    dict(gate=P + 128, gate_kind=_lib.TFM_GATE_CHANNEL), dict(gate=P, gate_kind=_lib.TFM_GATE_TOKEN),
    dict(gate=P - 32, gate_kind=_lib.TFM_GATE_TOKEN),
    dict(h=None, x=P, pre_weight=P + 1024), dict(h=None, x=P, pre_weight=P - 2),
    dict(h=None, x=P, pre_weight=P + 65536, gate=P + 4, gate_kind=_lib.TFM_GATE_TOKEN),
    dict(pre_weight=P + 65536, codes=P, scales=P + 70000), dict(pre_weight=P + 65536, codes=P + 70000, scales=P + 8),
    dict(pre_weight=P + 65536, y=P + 20000, codes=P + 20000 + 1151, scales=P + 70000),
    dict(pre_weight=P + 65536, codes=P + 65536 + 127, scales=P + 70000),
    dict(pre_weight=P + 65536, codes=P + 70000, scales=P + 65536 - 35),
    dict(pre_weight=P + 65536, codes=P + 70000, scales=P + 70575),
    dict(pre_weight=P + 65536, gate=P + 80000, gate_kind=_lib.TFM_GATE_TOKEN, codes=P + 80035, scales=P + 70000),
])
def test_norm_residual_refuses_outputs_over_weights_gates_and_each_other(kw):
    """9 rows of 64 elements: 1152 bytes, weights 128, a gate or scale for each row 36, codes 576."""
    s = step(**{**dict(y=P + 4096 * 9, h=P), **kw})
    check(_lib.load().tfm_norm_residual(ctypes.byref(s), 9, 64, BF16, None), 1, "overlap")


@pytest.mark.parametrize("codes,scales", [(P, P + 8192), (P + 1151, P + 8192), (P - 575, P + 8192), (P + 8192, P + 4),
                                          (P + 8192, P + 8192 + 572), (P + 8192, P + 8192 - 32)])
def test_quantize_rows_refuses_overlaps(codes, scales):
    check(_lib.load().tfm_quantize_rows(P, 9, 64, BF16, codes, scales, None), 1, "overlap")


@pytest.mark.parametrize("out,bias", [(P, None), (P + 1024, None), (P + 4096, None), (P + 4096 + 35, None),
                                      (P + 8192 + 640, None), (P + 12288, None), (P + 16384 - 717, P + 16384)])
def test_products_refuse_an_output_over_an_input(out, bias):
    """9 rows of 128 codes at P, scales at P + 4096, 20 channels of 128 at P + 8192, their scales at P + 12288."""
    check(_lib.load().tfm_int8_qmm(P, P + 4096, 9, P + 8192, P + 12288, bias, 20, 128, F32, out, None), 1, "overlap")


def test_int8_linear_refuses_overlaps():
    lib, w, ws, far = _lib.load(), 1 << 24, 1 << 25, 1 << 26
    need = lib.tfm_int8_linear_workspace_bytes(500, 256)
    for rows, out, work in ((2, P + 512, None), (2, w + 10, None), (2, ws + 4, None), (500, P, far), (500, w, far),
                            (500, far, P), (500, far, w - 256), (500, far, ws), (500, far + 300, far)):
        check(lib.tfm_int8_linear(P, rows, w, ws, None, 64, 256, BF16, out, work, need if work else 0, None), 1, "overlap")


@pytest.mark.parametrize("kw", [dict(logprobs=P), dict(entropy=P + 2 * 400 + 199), dict(ids=P + 3 * 400 - 1 - 200),
                                dict(best=P + 5000 - 47), dict(entropy=P + 10000 + 8), dict(best=P + 30000 + 44)])
def test_token_logprobs_refuses_overlaps(kw):
    """3 rows of 100 logits, 200 apart, at P; 3 tokens at P + 5000."""
    a = dict(logprobs=P + 10000, entropy=P + 20000, ids=P + 30000, best=P + 40000)
    a.update(kw)
    check(_lib.load().tfm_token_logprobs(P, 3, 100, 200, BF16, P + 5000, 64, 4, 1.0, a["logprobs"], a["entropy"],
                                         a["ids"], a["best"], None), 1, "overlap")


@pytest.mark.parametrize("scale", [9e-36, 1.1e30])
def test_token_logprobs_refuses_scales_past_its_bounds(scale):
    check(_lib.load().tfm_token_logprobs(P, 3, 100, 100, BF16, None, 64, 0, scale, None, P + 8192, None, None, None), 1,
          "scale must be in")
