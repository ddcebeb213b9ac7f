"""Attention over the 8-bit cache where its definition is easiest to lose: windows as long as an int, rows that
look at many tokens a little."""
import math

import pytest
import torch

from tests.test_gpu_attention import FORMS, attend64, compare, half_step, make, queries, run

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


# -- windows -------------------------------------------------------------------------

@pytest.mark.parametrize("rows,width,spare", FORMS)
def test_windows_as_long_as_an_int(gpu, rows, width, spare):
    """A window longer than every sequence hides nothing, also from sequences with rows before their first token."""
    lengths = [max(1, rows // 2), 0, rows + 20, min(5, rows)]
    cache, table = make(gpu, lengths, 1, 16, 64, seed=90)
    q, starts = queries(4 * rows, 2, 64, BF16, gpu, seed=90), [i * rows for i in range(5)]
    want, bound = attend64(q, cache, table, lengths, starts, 0.125, True, 0)
    all_of_it = run(q, cache, table, lengths, starts, gpu, width, spare)
    compare(all_of_it, want, bound)
    for window in (2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - rows, 2 ** 30):
        assert torch.equal(run(q, cache, table, lengths, starts, gpu, width, spare, window=window), all_of_it)


# -- many tokens that a row looks at a little ------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,width,spare", FORMS)
def test_one_token_far_above_the_others(gpu, dtype, rows, width, spare):
    """The first token takes nearly all of the weight and has the value zero, so that the output is what the others bring:
    with n of them, each e^-gap of the first, n e^-gap / (1 + n e^-gap) of their value."""
    page, length, dim = 16, 390 if spare else 700, 64
    cache, table = make(gpu, [length], 1, page, dim, seed=91)
    first = table[0, 0].item()
    cache.k.zero_()
    cache.k[first, 0, 0, 0] = 127
    codes = (torch.arange(dim) * 5 % 255 - 127).to(torch.int8).to(gpu)
    cache.v[:] = codes
    cache.v[first, 0, 0] = 0
    cache.k_scales.fill_(1.0)
    q = torch.zeros((rows, 2, dim), dtype=dtype, device=gpu)
    q[..., 0] = 1.0
    for gap in (9.0, 14.0, 16.0, 17.0, 17.4, 20.0):
        scale = torch.tensor(gap / 127, dtype=torch.float32).item()
        w = math.exp(-scale * 127)
        share = (length - 1) * w / (1 + (length - 1) * w)
        unit = 1 / (64 * share)  # a value scale that brings outputs near 1
        cache.v_scales.fill_(unit)
        unit = cache.v_scales[0, 0].item()
        want = (codes.cpu().double() * unit * share).expand(rows, 2, dim)
        # The first's weight is at least 2^8 as a half, each other's w times that: each is off by half a step, 2^-11 of
        # itself, or 2^-25 where it is subnormal. An exponent is at most 64 in size: five roundings of 2^-19
        # in front of 2^x, times ln 2, for each of the two, and the fp32 sums below 2^-17 (64 additions in a row).
        relative = max(2.0 ** -11, 2.0 ** -25 / (w * 2 ** 8)) + 2.0 ** -11 + 7 * 2.0 ** -19 + 2.0 ** -17
        got = run(q, cache, table, [length], [0, rows], gpu, width, spare, causal=False, scale=scale)
        compare(got, want, want.abs() * (1.01 * relative + half_step(dtype)))


@pytest.mark.parametrize("rows,width,spare", FORMS)
@pytest.mark.parametrize("spread", [2.0 ** -6, 2.0 ** 5, 2.0 ** 12, 2.0 ** 20])
def test_far_above_in_a_page_of_another_scale(gpu, rows, width, spare, spread):
    """The same with the others' values in a scale `spread` times smaller than the first's page has."""
    page, length, dim = 16, 390 if spare else 700, 64
    cache, table = make(gpu, [length], 1, page, dim, seed=92)
    first, n = table[0, 0].item(), length - page
    cache.k.zero_()
    cache.k[first, 0, :, 0] = 127
    codes = (torch.arange(dim) * 5 % 255 - 127).to(torch.int8).to(gpu)
    cache.v[:] = codes
    cache.v[first] = 0
    cache.k_scales.fill_(1.0)
    cache.v_scales.fill_(1.0)
    cache.v_scales[first] = spread
    q = torch.zeros((rows, 2, dim), dtype=BF16, device=gpu)
    q[..., 0] = 1.0
    for gap in (2.0, 7.0, 12.0):
        scale = torch.tensor(gap / 127, dtype=torch.float32).item()
        w = math.exp(-scale * 127)
        share = n * w / (page + n * w)
        want = (codes.cpu().double() * share).expand(rows, 2, dim)
        # As above; a weight that enters the product is w / spread of the first's, and off by 2^-33 of that where it is
        # a subnormal half: n of them, times codes up to 127, over the sum of weights, (16 + n w) / spread.
        lost = n * 127 * 2.0 ** -33 * spread / (page + n * w)
        relative = 2.0 ** -10 + 7 * 2.0 ** -19 + 2.0 ** -17
        got = run(q, cache, table, [length], [0, rows], gpu, width, spare, causal=False, scale=scale)
        compare(got, want, want.abs() * (1.01 * relative + half_step(BF16)) + lost)
