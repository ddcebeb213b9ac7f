"""The operators around the block at the edges of what they accept: aliases, scales, allocation, long rows of codes."""
import math

import pytest
import torch

from tests.test_gpu_layer import BF16, EPS, F32, check_logprobs, logprobs64, rand
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
