"""Rotary positions, the 8-bit cache and attention over it on the host (no GPU): refusals before any device work, the
mirror's checks, and the frequencies of stretched contexts."""
import ctypes
import math

import pytest
import torch

from trifuse_amd import _lib, layer

P = 1 << 40  # a non-null, aligned pointer that is never dereferenced; others stand far from it
STEP = 1 << 32
BF16, F16, F32 = _lib.TFM_DTYPE_BF16, _lib.TFM_DTYPE_F16, _lib.TFM_DTYPE_F32


def check(status, code, msg):
    assert status == code, _lib.load().tfm_last_error()
    if code:
        assert msg in _lib.load().tfm_last_error().decode()


def rotation(**kw):
    return _lib.Rotation(**{**dict(frequencies=P, pairs=32, interleaved=0, scale=1.0), **kw})


def cache(**kw):
    a = dict(k=P + STEP, v=P + 2 * STEP, k_scales=P + 3 * STEP, v_scales=P + 4 * STEP, pages=8, kv_heads=2, page_tokens=16,
             head_dim=64)
    return _lib.KvCache(**{**a, **kw})


def batch(**kw):
    a = dict(table=P + 5 * STEP, lengths=P + 6 * STEP, starts=P + 7 * STEP, sequences=3, table_width=2, max_rows=4)
    return _lib.KvBatch(**{**a, **kw})


CACHES = [
    (dict(pages=0), {}, 1, "no pages"),
    (dict(pages=1 << 31), {}, 2, "pages"),
    (dict(kv_heads=0), {}, 1, "kv_heads"),
    (dict(kv_heads=1025), {}, 1, "kv_heads"),
    (dict(page_tokens=8), {}, 2, "page_tokens"),
    (dict(page_tokens=48), {}, 2, "page_tokens"),
    (dict(page_tokens=512), {}, 2, "page_tokens"),
    (dict(head_dim=96), {}, 2, "head_dim"),
    (dict(k=None), {}, 1, "k codes is null"),
    (dict(v=None), {}, 1, "v codes is null"),
    (dict(k_scales=None), {}, 1, "k_scales is null"),
    (dict(v_scales=None), {}, 1, "v_scales is null"),
    (dict(k=P + STEP + 8), {}, 1, "16-byte"),
    ({}, dict(sequences=-1), 1, "sequences"),
    ({}, dict(table_width=0), 1, "table_width"),
    (dict(page_tokens=256), dict(table_width=(1 << 22) + 1), 2, "2^30"),
    ({}, dict(max_rows=-1), 1, "max_rows"),
    ({}, dict(table=None), 1, "table is null"),
    ({}, dict(lengths=None), 1, "lengths is null"),
]


def append(c=None, b=None, r=None, k=P, v=P + 8 * STEP, rows=12, stride=128, head=64, dtype=BF16):
    c, b = c or cache(), b or batch()
    return _lib.load().tfm_cache_append(k, stride, head, v, stride, head, rows, ctypes.byref(r) if r else None, dtype,
                                        ctypes.byref(c), ctypes.byref(b), None)


def read(c=None, b=None, dtype=BF16, k=P, v=P + 8 * STEP):
    c, b = c or cache(), b or batch(starts=None)
    return _lib.load().tfm_cache_read(ctypes.byref(c), ctypes.byref(b), dtype, k, v, None)


def attention(c=None, b=None, q=P, rows=12, heads=6, stride=384, head=64, scale=0.125, causal=1, window=0, dtype=BF16,
              out=P + 9 * STEP, ws=P + 10 * STEP, ws_bytes=1 << 30):
    c, b = c or cache(), b or batch()
    return _lib.load().tfm_cache_attention(q, stride, head, rows, heads, ctypes.byref(c), ctypes.byref(b), scale, causal,
                                           window, dtype, out, ws, ws_bytes, None)


@pytest.mark.parametrize("ck,bk,code,msg", CACHES)
def test_cache_and_batch_rejects(ck, bk, code, msg):
    check(append(cache(**ck), batch(**bk)), code, msg)
    check(attention(cache(**ck), batch(**bk)), code, msg)
    if not {"sequences", "max_rows"} & set(bk):  # no rows to read then
        check(read(cache(**ck), batch(**{**bk, "starts": None})), code, msg)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(rows=-1), 1, "rows"),
    (dict(rows=1 << 22), 1, "rows"),
    (dict(heads=0), 1, "heads"),
    (dict(heads=1025), 1, "heads"),
    (dict(dim=0), 1, "head_dim"),
    (dict(dim=1026), 2, "head_dim"),
    (dict(dtype=F32), 1, "dtype"),
    (dict(bits=16), 1, "position_bits"),
    (dict(r=None), 1, "rotation is null"),
    (dict(r=dict(pairs=0)), 1, "pairs"),
    (dict(r=dict(pairs=33)), 1, "pairs"),
    (dict(r=dict(scale=math.inf)), 1, "finite"),
    (dict(r=dict(frequencies=None)), 1, "frequencies"),
    (dict(x=None), 1, "x is null"),
    (dict(positions=None), 1, "positions is null"),
    (dict(out=None), 1, "out is null"),
    (dict(stride=-1), 1, "strides"),
    (dict(ostride=255), 1, "overlap"),
    (dict(ohead=63), 1, "overlap"),
    (dict(out=P + 2), 1, "overlaps"),
    (dict(out=P, ostride=512), 1, "overlaps"),
    (dict(positions=P + STEP), 1, "positions"),
    (dict(rows=0, x=None, out=None, positions=None), 0, ""),
])
def test_rotary_rejects(kw, code, msg):
    a = dict(x=P, rows=5, heads=4, dim=64, stride=256, head=64, positions=P + 2 * STEP, bits=64, r={}, dtype=BF16, out=P + STEP,
             ostride=256, ohead=64)
    a.update(kw)
    r = None if a["r"] is None else ctypes.byref(rotation(**{"frequencies": P + 3 * STEP, **a["r"]}))
    check(_lib.load().tfm_rotary(a["x"], a["rows"], a["heads"], a["dim"], a["stride"], a["head"], a["positions"], a["bits"], r,
                                 a["dtype"], a["out"], a["ostride"], a["ohead"], None), code, msg)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(rows=-1), 1, "rows"),
    (dict(dtype=F32), 1, "dtype"),
    (dict(k=None), 1, "k is null"),
    (dict(v=None), 1, "v is null"),
    (dict(stride=-2), 1, "strides"),
    (dict(r=rotation(pairs=12)), 2, "multiple of 8"),
    (dict(r=rotation(pairs=40)), 1, "pairs"),
    (dict(b=batch(starts=None), rows=11), 1, "sequences * max_rows"),
    (dict(k=P + STEP), 1, "overlap"),
    (dict(v=P + 4 * STEP), 1, "overlap"),
    (dict(c=cache(v=P + STEP + 64)), 1, "overlap"),
    (dict(b=batch(sequences=1 << 21, max_rows=100), rows=100), 2, "2^22"),
    (dict(rows=0, k=None, v=None), 0, ""),
    (dict(b=batch(max_rows=0)), 0, ""),
    (dict(b=batch(sequences=0)), 0, ""),
])
def test_append_rejects(kw, code, msg):
    check(append(**kw), code, msg)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(dtype=3), 1, "dtype"),
    (dict(b=batch()), 1, "starts"),
    (dict(k=None), 1, "k is null"),
    (dict(v=P + 8), 1, "16-byte"),
    (dict(k=P + STEP), 1, "overlap"),
    (dict(v=P + 16), 1, "overlap"),
    (dict(b=batch(starts=None, sequences=1 << 21, max_rows=2)), 1, "rows"),
    (dict(b=batch(starts=None, sequences=0), k=None), 0, ""),
])
def test_read_rejects(kw, code, msg):
    check(read(**kw), code, msg)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(rows=-1), 1, "rows"),
    (dict(dtype=F32), 1, "dtype"),
    (dict(heads=5), 1, "multiple"),
    (dict(heads=0), 1, "heads"),
    (dict(heads=1026), 1, "heads"),
    (dict(window=-1), 1, "window"),
    (dict(window=3, causal=0), 1, "causal"),
    (dict(scale=math.nan), 1, "scale"),
    (dict(scale=math.inf), 1, "scale"),
    (dict(scale=3e38), 1, "scale"),  # past fp32 in the exponent's base
    (dict(c=cache(kv_heads=1), rows=(1 << 22) - 1, heads=1024, b=batch(max_rows=(1 << 22) - 1)), 2, "2^30"),
    (dict(q=None), 1, "q is null"),
    (dict(out=None), 1, "out is null"),
    (dict(out=P + 9 * STEP + 2), 1, "aligned"),
    (dict(out=P), 1, "overlap"),
    (dict(out=P + STEP), 1, "overlap"),
    (dict(head=-64), 1, "strides"),
    (dict(rows=0, q=None, out=None, ws=None, ws_bytes=0), 0, ""),
    (dict(b=batch(sequences=0), q=None), 0, ""),
    (dict(b=batch(table_width=100), ws=None), 3, "workspace"),
    (dict(b=batch(table_width=100), ws=P + 10 * STEP + 64), 3, "aligned"),
    (dict(b=batch(table_width=100), ws_bytes=100), 3, "too small"),
    (dict(b=batch(table_width=100), ws=P + 9 * STEP), 1, "overlap"),
])
def test_attention_rejects(kw, code, msg):
    check(attention(**kw), code, msg)


def test_workspace_bytes():
    need = lambda c, b, rows=12, heads=6, window=0: _lib.load().tfm_cache_attention_workspace_bytes(  # noqa: E731
        rows, heads, window, ctypes.byref(c), ctypes.byref(b))
    assert need(cache(), batch()) == 0  # one workgroup reads so few tokens
    assert need(cache(), batch(table_width=4096)) > 0
    assert need(cache(), batch(table_width=4096), window=64) == 0
    assert need(cache(), batch(table_width=4096), rows=0) == 0
    assert need(cache(head_dim=80), batch(table_width=4096)) == 0  # refused by the call itself


def _tensors():
    c = layer.KVCache.empty(4, 2, 16, 64, device="cpu")
    return c, torch.zeros((2, 2), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)


def test_mirror_has_no_cpu_fallback():
    c, table, lengths = _tensors()
    x = torch.zeros((2, 2, 64), dtype=torch.bfloat16)
    f, scale = layer.rotary_frequencies(32)
    for call in (lambda: layer.rotary(x, torch.zeros(2, dtype=torch.int64), f),
                 lambda: layer.cache_append(x, x, c, table, lengths),
                 lambda: layer.cache_read(c, table, lengths, 1),
                 lambda: layer.cache_attention(x, c, table, lengths)):
        with pytest.raises(ValueError, match="GPU tensor"):
            call()


def test_cache_layout():
    c = layer.KVCache.empty(5, 3, 32, 128, device="cpu")
    assert c.k.shape == c.v.shape == (5, 3, 32, 128) and c.k.dtype == torch.int8
    assert c.k_scales.shape == c.v_scales.shape == (5, 3) and c.v_scales.dtype == torch.float32


def test_frequencies():
    f, scale = layer.rotary_frequencies(64)
    assert f.dtype == torch.float64 and scale == 1.0
    want = [10000.0 ** (-i / 64) for i in range(64)]
    assert all(abs(a - b) <= 2 ** -50 * b for a, b in zip(f.tolist(), want))
    g, scale = layer.rotary_frequencies(64, stretch=4.0)
    assert torch.equal(g, f / 4) and scale == 1.0
    g, scale = layer.rotary_frequencies(64, stretch=4.0, method="base")
    assert scale == 1.0 and g[0] == 1.0 and abs(float(g[-1] / f[-1]) - 0.25) < 1e-12
    g, scale = layer.rotary_frequencies(64, stretch=4.0, method="bands", context=4096)
    turns = f * 4096 / (2 * math.pi)
    assert scale == 0.1 * math.log(4.0) + 1.0
    assert torch.equal(g[turns >= 32], f[turns >= 32]) and torch.equal(g[turns <= 1], f[turns <= 1] / 4)
    between = (turns > 1) & (turns < 32)
    assert between.any() and bool(((g < f) & (g > f / 4))[between].all())
    one, scale = layer.rotary_frequencies(1, stretch=2.0, method="base")
    assert one.tolist() == [1.0]
    assert torch.equal(layer.rotary_frequencies(64, stretch=1.0, method="bands", context=4096)[0], f)


@pytest.mark.parametrize("kw", [dict(pairs=0), dict(pairs=4, base=0.0), dict(pairs=4, stretch=0.5), dict(pairs=4, method="other"),
                                dict(pairs=4, method="bands"), dict(pairs=4, method="bands", context=4096, slow=8.0, fast=8.0)])
def test_frequencies_reject(kw):
    with pytest.raises(ValueError):
        layer.rotary_frequencies(**kw)
