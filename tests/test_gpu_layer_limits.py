"""The operators around the block at the edges of what they accept: aliases, scales, allocation, long rows of codes."""
import math

import pytest
import torch

from tests.test_gpu_layer import (BF16, EPS, F, F16, F32, _layer_pass, _layer_state, check_logprobs, close, codes_of,
                                  logprobs64, norm64, product64, rand, scales_of, step64)
from trifuse_amd import layer
from trifuse_amd._lib import TfmError, TfmUnsupported

pytestmark = pytest.mark.gpu


def test_norm_residual_over_its_gate(gpu):
    """h written over a gate of y's shape gives the same bits, one row and its [H] form too."""
    for shape in ((5, 512), (5, 515), (1, 512), (512,), (9000,)):
        y, r, g, w = rand(shape, 1), rand(shape, 2), rand(shape, 3), rand(shape[-1:], 4, 0.1, mean=1.0)
        h, x = layer.norm_residual(y, r, gate=g, pre_weight=w, eps=EPS)
        into = g.clone()
        h2, x2 = layer.norm_residual(y, r, gate=into, pre_weight=w, eps=EPS, out=into)
        assert h2.data_ptr() == into.data_ptr() and torch.equal(h2, h) and torch.equal(x2, x)


def test_norm_residual_gated_by_its_own_row(gpu):
    """A single row's [H] gate is the row itself, and h is written over both."""
    for width in (512, 9000):
        y, w = rand((1, width), 1), rand((width,), 2, 0.1, mean=1.0)
        h, x = layer.norm_residual(y, gate=y[0].clone(), pre_weight=w, eps=EPS)
        h2, x2 = layer.norm_residual(y, gate=y[0], pre_weight=w, eps=EPS, out=y)
        assert torch.equal(h2, h) and torch.equal(x2, x)


def test_norm_residual_refuses_out_over_shared_inputs(gpu):
    buf = rand((9, 64), 1)
    y, gates = rand((4, 64), 2), torch.ones(260, device="cuda")
    cases = [dict(post_weight=buf[3]), dict(pre_weight=buf[5]), dict(gate=buf[2]),
             dict(post_weight=buf.view(-1)[6 * 64 - 1:7 * 64 - 1])]
    before = buf.clone()
    for kw in cases:
        with pytest.raises(TfmError, match="overlap"):
            layer.norm_residual(y, out=buf[2:6], **kw)
    with pytest.raises(TfmError, match="overlap"):
        layer.norm_residual(y, gate=gates[100:104], out=gates[:128].view(BF16).view(4, 64))
    assert torch.equal(buf, before) and (gates == 1).all()
    assert torch.equal(layer.norm_residual(y, post_weight=buf[6], out=buf[2:6]), layer.norm_residual(y, post_weight=before[6]))
    assert gates.dtype == F32


# -- scales ------------------------------------------------------------------------

def check_sure(logits, tokens, top, scale):
    """check_logprobs' bounds (rel and its use are explained there) with the entropy as -sum p lp: where lp is under
    2^-53, p = e^lp is 1 in 64 bits too, so that xlogy(p, p) there drops the sure token's own term, R of the
    R (1 + |ln R|) that the entropy is."""
    logp, entropy, ids, best = layer.token_logprobs(logits, tokens, top=top, scale=scale)
    rp, _, rids, rbest = logprobs64(logits, tokens, top, scale)
    lp = logprobs64(logits, None, logits.shape[-1], scale)[3]  # of every token
    re = -torch.where(lp.exp() > 0, lp.exp() * lp, 0.0).sum(-1)
    rel = (logits.shape[-1] / 256 + 340) * 2.0 ** -24

    def near(got, ref, extra=0.0):
        got = got.double().cpu()
        assert torch.equal(got.isnan(), ref.isnan())
        off = (got - ref).abs()
        ok = (got == ref) | (off <= ref.abs().clamp(max=1.0) * rel * 2 + ref.abs() * 2.0 ** -22 + extra)
        assert ok.all(), f"worst {off[~ok].max()}"

    assert torch.equal(ids.cpu().long(), rids)
    near(best, rbest)
    near(logp, rp)
    near(entropy, re, extra=re * rel * 2 + rel * 2 * re.clamp(max=1.0))


@pytest.mark.parametrize("scale", [1e-35, 1e-30, 1e-20, 1e-3, 100.0, 1e4, 1e30])
@pytest.mark.parametrize("vocab", [16, 700, 9001, 40000])
def test_token_logprobs_at_any_scale(gpu, scale, vocab):
    """Logits of a few units of 1 / scale, in places that different threads read, beside masked ones."""
    rows = []
    for sigma in (0.3, 3.0, 40.0):
        g = torch.Generator().manual_seed(vocab)
        row = torch.randn(vocab, generator=g, dtype=torch.float64) * sigma / scale
        rows += [row, torch.where(torch.arange(vocab) % 16 < 8, 0.0, -2.0 / scale),
                 torch.where(torch.rand(vocab, generator=g) < 0.5, -math.inf, row)]
    logits = torch.stack(rows).float().cuda()
    tokens = torch.arange(len(rows), device="cuda") * (vocab // 10)
    check_sure(logits, tokens, 5, torch.tensor(scale, dtype=F32).double().item())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_token_logprobs_of_the_largest_differences(gpu, dtype):
    """Differences past the largest number: probability 0, and a finite log probability where it is one."""
    big = torch.finfo(dtype).max
    logits = torch.full((3, 600), -big, dtype=dtype, device="cuda")
    logits[:, 7] = big
    logits[1, 300], logits[2] = big, torch.where(torch.arange(600, device="cuda") % 2 == 0, big, -big)
    tokens = torch.tensor([8, 9, 11], device="cuda")
    for scale in (1e-35, 1e-10, 0.25):
        scale = torch.tensor(scale, dtype=F32).double().item()
        check_logprobs(logits, tokens, 3, scale)
        assert torch.isfinite(layer.token_logprobs(logits, tokens, scale=scale)[0]).all()
    assert (layer.token_logprobs(logits, tokens)[0] == -math.inf).all()


# -- allocation --------------------------------------------------------------------

def ones(shape, dtype):
    return torch.ones(shape, dtype=dtype, device="cuda")


def test_an_output_that_does_not_fit_is_out_of_memory(gpu):
    """As torch's own allocations raise it, so that a caller can retry with fewer rows; the next call works."""
    n = 1 << 20  # an output of 2^40 elements
    x, w, s = ones((n, 16), BF16), ones((n, 16), torch.int8), ones((n,), F32)
    with pytest.raises(torch.OutOfMemoryError):
        layer.int8_linear(x, w, s)
    with pytest.raises(torch.OutOfMemoryError):
        layer.int8_qmm(w, s, w, s)
    assert (layer.int8_qmm(w[:5], s[:5], w[:3], s[:3], dtype=F32) == 16).all()


def test_limits_come_before_the_output(gpu):
    """Sizes that no product takes are refused as such, whatever their output would need."""
    n = 1 << 20
    for rows, k, error, message in ((n, 24, TfmUnsupported, "multiple of 16"), (1 << 22, 16, TfmError, "rows")):
        x, w, s = ones((rows, k), BF16), ones((n, k), torch.int8), ones((max(n, rows),), F32)
        with pytest.raises(error, match=message):
            layer.int8_linear(x, w, s[:n])
        with pytest.raises(error, match=message):
            layer.int8_qmm(ones((rows, k), torch.int8), s[:rows], w, s[:n])


# -- products ----------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_a_row_has_the_same_bits_in_every_batch(gpu, dtype):
    """8190 channels: few rows, 64 x 64, 128 x 128, 256 x 192 (fp32: another) and 256 x 256 tiles, in this order."""
    k, n = 272, 8190
    codes, w, scales, ws = codes_of((2047, k), 1), codes_of((n, k), 2), scales_of(2047, 3), scales_of(n, 4)
    bias = rand((n,), 5, 1.0, dtype)
    whole = layer.int8_qmm(codes, scales, w, ws, bias=bias, dtype=dtype)
    for rows in (1, 9, 16, 40, 300, 1100):
        for at in (0, 2047 - rows):
            part = layer.int8_qmm(codes[at:at + rows], scales[at:at + rows], w, ws, bias=bias, dtype=dtype)
            assert torch.equal(part, whole[at:at + rows]), (rows, at)


@pytest.mark.parametrize("rows,k,n", [(8, 7104, 640), (8, 7120, 640), (8, 8192, 640), (4, 14336, 515), (2, 32768, 96),
                                      (1, 57216, 70), (1, 57280, 70), (16, 3520, 130), (16, 3536, 130), (3, 131056, 33)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_int8_linear_of_few_long_rows(gpu, rows, k, n, dtype):
    """Rows on both sides of what the few-row kernel's shared memory holds: quantize_rows and int8_qmm, bit for bit,
    and int8_qmm against 64 bits."""
    x, w, ws, bias = rand((rows, k), 1, 1.0, dtype), codes_of((n, k), 2), scales_of(n, 4), rand((n,), 5, 1.0, dtype)
    codes, scales = layer.quantize_rows(x)
    out = layer.int8_qmm(codes, scales, w, ws, bias=bias, dtype=dtype)
    close(out, *product64(codes, scales, w, ws, bias), dtype)
    assert torch.equal(layer.int8_linear(x, w, ws, bias=bias), out)


# -- together ----------------------------------------------------------------------

@pytest.mark.parametrize("rows", [1, 5, 70, 300])
def test_each_step_of_a_pass(gpu, rows):
    """Each step of a layer's pass against 64 bits on the step's own inputs, to one rounding of each output."""
    s = _layer_state(rows, 512, 3001)

    def codes_close(codes, scales, x64, ex):
        step, worst = scales.double()[:, None], ex.amax(-1, keepdim=True)
        assert ((codes.double() * step - x64).abs() <= step * (0.5 + 2.0 ** -15) + ex + worst).all()

    h, codes, scales = layer.norm_residual(s["y"], s["h"], post_weight=s["w1"], gate=s["gate"], residual_multiplier=0.22,
                                           pre_weight=s["w2"], eps=EPS, quantize=True)
    h64, eh, x64, ex = step64(s["y"], s["h"], s["w1"], s["gate"], 0.22, s["w2"])
    close(h, h64, eh, BF16)
    codes_close(codes, scales, x64, ex)
    mid = layer.int8_qmm(codes, scales, s["p"], s["ps"], dtype=BF16)
    close(mid, *product64(codes, scales, s["p"], s["ps"], None), BF16)
    last = layer.norm_residual(mid, h, residual_multiplier=0.22)
    h64, eh, _, _ = step64(mid, h, None, None, 0.22, None)
    close(last, h64, eh, BF16)
    codes, scales = layer.rms_norm(last, s["w3"], EPS, quantize=True)
    x64 = norm64(last.double(), s["w3"].double())
    codes_close(codes, scales, x64, F * x64.abs())
    logits = layer.int8_qmm(codes, scales, s["head"], s["hs"], dtype=F32)
    close(logits, *product64(codes, scales, s["head"], s["hs"], None), F32)
    check_logprobs(logits, s["tokens"], 5, 0.5)
    whole = _layer_pass(s)
    assert torch.equal(whole[0], last) and torch.equal(whole[1], logits)
