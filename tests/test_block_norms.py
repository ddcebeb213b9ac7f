"""The host side of the block between its norms (no GPU)."""
import contextlib
import threading
import time

import pytest
import torch

from trifuse_amd import layer
from trifuse_amd import moe as tmoe


class OnDevice(torch.Tensor):
    """A CPU tensor that says it is on GPU 1."""

    def get_device(self):
        return 1


@pytest.mark.parametrize("current", [0, 1])
def test_forward_norms_runs_on_its_tensors_device(monkeypatch, current):
    """The norms and the block between them are enqueued with h's device as the current one, which is put back."""
    device = [current]
    seen = []

    @contextlib.contextmanager
    def use(index):
        before, device[0] = device[0], int(index)
        yield
        device[0] = before

    monkeypatch.setattr(torch.cuda, "current_device", lambda: device[0])
    monkeypatch.setattr(torch.cuda, "device", use)
    monkeypatch.setattr(tmoe, "_dev", lambda t, name: None)
    monkeypatch.setattr(tmoe, "_stream", lambda: 100 + device[0])
    monkeypatch.setattr(tmoe, "call", lambda name, *args: name == "tfm_plan_create" or seen.append((name, args[-1])))
    blk = tmoe.MoEBlock(64, 64, 4, 2)
    monkeypatch.setattr(blk, "_weights", lambda w, router: tmoe.MoeWeights())
    monkeypatch.setattr(blk, "workspace", lambda tokens, where: torch.empty(256, dtype=torch.uint8))
    monkeypatch.setattr(layer, "rms_norm", lambda x, w, eps: seen.append(("norm", 100 + device[0])) or x)
    monkeypatch.setattr(layer, "norm_residual", lambda y, h, **kw: seen.append(("residual", 100 + device[0])) or h)
    h = torch.zeros((3, 64), dtype=torch.bfloat16).as_subclass(OnDevice)
    out = blk.forward_norms(h, None, torch.ones(64, dtype=torch.bfloat16), 1e-5)
    assert out.shape == h.shape and device[0] == current
    assert seen == [("norm", 101), ("tfm_moe_forward", 101), ("residual", 101)]


def test_two_threads_make_one_second_plan(monkeypatch):
    """Calls that need the plan without the multiplier at once share one: none is left without an owner."""
    made, both = [], threading.Barrier(2)

    def create(name, geometry, handle):
        made.append(name)
        if len(made) > 1:  # the block's own plan is made alone
            time.sleep(0.2)
        handle._obj.value = len(made)

    monkeypatch.setattr(tmoe, "call", create)
    blk = tmoe.MoEBlock(64, 64, 4, 2, residual_multiplier=0.5)
    got = []

    def use():
        both.wait(timeout=10)
        got.append(blk._unit_plan().value)

    threads = [threading.Thread(target=use) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    blk._plan = blk._unit = None  # no plans of the library's: nothing to destroy
    assert made == ["tfm_plan_create"] * 2 and got == [2, 2]
