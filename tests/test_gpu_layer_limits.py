"""The operators around the block at the edges of what they accept: aliases, scales, allocation, long rows of codes."""
import pytest
import torch

from tests.test_gpu_layer import BF16, EPS, F32, rand
from trifuse_amd import layer
from trifuse_amd._lib import TfmError

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
