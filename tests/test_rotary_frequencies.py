"""Frequencies of stretched contexts against their formulas, a pair at a time (no GPU)."""
import math

import pytest

from trifuse_amd import layer


@pytest.mark.parametrize("pairs,base,stretch", [(2, 10000.0, 2.0), (32, 10000.0, 8.0), (64, 500000.0, 32.0), (64, 10000.0, 1.0)])
def test_base(pairs, base, stretch):
    f, scale = layer.rotary_frequencies(pairs, base, stretch=stretch, method="base")
    assert scale == 1.0
    for i, got in enumerate(f.tolist()):
        # base ** (-i / pairs) times stretch ** (-i / (pairs - 1)): two powers of at most 30 in the exponent, 64 bits
        want = math.exp(-i / pairs * math.log(base) - i / (pairs - 1) * math.log(stretch))
        assert abs(got - want) <= 2.0 ** -45 * want


@pytest.mark.parametrize("pairs,base,stretch,context,slow,fast", [
    (64, 10000.0, 4.0, 4096, 1.0, 32.0), (32, 10000.0, 16.0, 8192, 1.0, 32.0), (64, 500000.0, 8.0, 8192, 2.0, 64.0),
    (16, 10000.0, 40.0, 4096, 0.5, 3.0)])
def test_bands(pairs, base, stretch, context, slow, fast):
    """The mixed range is linear in the turns that a pair makes over the trained context."""
    f, scale = layer.rotary_frequencies(pairs, base, stretch=stretch, method="bands", context=context, slow=slow, fast=fast)
    assert scale == 0.1 * math.log(stretch) + 1.0
    mixed = 0
    for i, got in enumerate(f.tolist()):
        plain = math.exp(-i / pairs * math.log(base))
        turns = plain * context / (2 * math.pi)
        kept = 1.0 if turns >= fast else 0.0 if turns <= slow else (turns - slow) / (fast - slow)
        mixed += 0.0 < kept < 1.0
        want = plain * kept + plain / stretch * (1 - kept)
        # `kept` is off by a few steps of 64 bits of turns / (fast - slow), which is below 2 where it counts
        assert abs(got - want) <= 2.0 ** -44 * plain
    assert mixed >= 2
