"""Attention over the 8-bit cache, and appending to it, where the definition is easiest to lose: windows as long as an
int, rows that look at many tokens a little, huge scores, lengths past the table, thousands of sequences, more parts
than the joining kernel holds at once."""
import math

import pytest
import torch

from tests.test_gpu_attention import FORMS, append_steps, attend64, compare, half_step, make, queries, run, same_cache, starts_of
from trifuse_amd import layer

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def i32(values, gpu):
    return torch.tensor(values, dtype=torch.int32, device=gpu)


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


# -- scores of any size ------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,width,spare", FORMS)
def test_the_largest_of_huge_scores_is_the_row(gpu, dtype, rows, width, spare):
    """Scores so large that a step of fp32 is many binades of a weight: the token that stands above all others takes the row,
    and nothing overflows."""
    page, length, dim = 16, 390 if spare else 700, 64
    cache, table = make(gpu, [length], 1, page, dim, seed=98)
    cache.k_scales.fill_(1.0)
    g = torch.Generator().manual_seed(98)
    for top in (0, 37, length // 2, length - 1):
        # Channel 0 alone makes the score: 127 for one token, at most 60 for the others; other channels only change sums.
        cache.k[..., 0] = torch.randint(-127, 61, cache.k.shape[:3], generator=g).to(torch.int8).to(gpu)
        at = table[0, top // page].item()
        cache.k[at, 0, top % page, 0] = 127
        q = torch.zeros((rows, 2, dim), dtype=dtype, device=gpu)
        q[..., 0] = 1.0
        q[..., 1:] = (torch.randn((rows, 2, dim - 1), generator=g) * 2.0 ** -8).to(dtype).to(gpu)
        want = (cache.v[at, 0, top % page].cpu().double() * cache.v_scales[at, 0].cpu().double()).expand(rows, 2, dim)
        for size in (2.0 ** 10, 2.0 ** 20, 2.0 ** 23, 2.0 ** 24, 2.0 ** 25, 2.0 ** 26, 2.0 ** 28, 2.0 ** 31, 2.0 ** 40, 2.0 ** 80):
            # The others' sums: 63 channels of at most 4 x 2^-8 x 127, a standard deviation of 2^-8 x 40 x 8: below 20 of the 67
            # between 127 and 60, so that they are over 300 below at the smallest size. The output is one value, code times
            # scale: its weight is the same in both sums and falls out, which leaves an inverse, a division and a few products.
            got = run(q, cache, table, [length], [0, rows], gpu, width, spare, causal=False, scale=size / 127)
            compare(got, want, want.abs() * (half_step(dtype) + 2.0 ** -19))


# -- lengths past the table ------------------------------------------------------------

def held_to(rows, lengths, room):
    """[(rows, length)] of the same batch with the rows that have a place: row i of n is at position length - n + i."""
    return [(max(0, min(n, room - (length - n))), min(length, room)) for n, length in zip(rows, lengths)]


@pytest.mark.parametrize("page,kv_heads,dim,pairs", [(16, 2, 64, 0), (16, 5, 128, 64), (64, 1, 128, 0), (256, 2, 64, 16)])
def test_rows_past_the_table_are_not_written(gpu, page, kv_heads, dim, pairs):
    """A token behind the table's last place is nowhere: it is not written, and those before it stay."""
    room = 3 * page
    rows, lengths = [1, 30, 20, 5, 4, 7], [room + 1, room + 20, 1000 + room, 2 ** 31 - 1, 40, 2 ** 30 + 3]
    cache, table = make(gpu, [room] * 6, kv_heads, page, dim, seed=93)
    g = torch.Generator().manual_seed(93)
    k, v = (torch.randn((sum(rows) + 2, kv_heads, dim), generator=g).to(BF16) * 3 for _ in "kv")
    kw = dict(frequencies=layer.rotary_frequencies(pairs, device=gpu)[0]) if pairs else {}
    other = layer.KVCache(*(t.clone() for t in cache))
    want = [t.cpu().clone() for t in cache]
    for _ in range(2):  # as replays of one step do
        layer.cache_append(k.to(gpu), v.to(gpu), cache, table.to(gpu), i32(lengths, gpu), starts=i32(starts_of(rows), gpu),
                           max_rows=30, **kw)
    for b, (n, length) in enumerate(held_to(rows, lengths, room)):
        start = starts_of(rows)[b]
        mine = [t[start:start + n] for t in (k, v)]
        for _ in range(2):
            append_steps(want, *mine, table[b:b + 1], [length], [0, n])
            if n:
                layer.cache_append(*(t.to(gpu) for t in mine), other, table[b:b + 1].to(gpu), i32([length], gpu), **kw)
    same_cache(cache, [t.cpu() for t in other])
    if not pairs:
        same_cache(cache, want)
    back = layer.cache_read(cache, table.to(gpu), i32(lengths, gpu), 25, torch.float32)
    for got, codes, scales in ((back[0], cache.k, cache.k_scales), (back[1], cache.v, cache.v_scales)):
        values = (codes.float() * scales[:, :, None, None]).cpu()
        got = got.cpu().view(6, 25, kv_heads, dim)
        for b, length in enumerate(lengths):
            for i in range(25):
                t = length - 25 + i
                assert torch.equal(got[b, i], values[table[b, t // page], :, t % page]) if t < room else not got[b, i].any()


@pytest.mark.parametrize("causal,window", [(True, 0), (True, 33), (True, 2 ** 31 - 1), (False, 0)])
@pytest.mark.parametrize("rows,width,spare", FORMS)
def test_rows_past_the_table_stay_at_their_positions(gpu, rows, width, spare, causal, window):
    """They see the tokens that there are, from where they stand."""
    page, room = 16, 64 if spare else 160
    lengths = [room + 1, room + rows // 2, room + 30, room + 1000]
    cache, table = make(gpu, [room] * 4, 2, page, 64, seed=94)
    q, starts = queries(4 * rows, 4, 64, F16, gpu, seed=94), [i * rows for i in range(5)]
    longer = torch.nn.functional.pad(table, (0, -(-max(lengths) // page) - table.shape[1]), value=-1)
    want, bound = attend64(q, cache, longer, lengths, starts, 0.125, causal, min(window, 10 ** 6))
    compare(run(q, cache, table, lengths, starts, gpu, 0, spare, causal=causal, window=window), want, bound)
    if width:  # the same with room for the tokens, but no pages: other kernels
        compare(run(q, cache, table, lengths, starts, gpu, width, spare, causal=causal, window=window), want, bound)
    far = [2 ** 31 - 1, 2 ** 30 + 7, 2 ** 31 - 20, 2 ** 30]
    got = run(q, cache, table, far, starts, gpu, 0, spare, causal=causal, window=window)
    if 0 < window < 2 ** 20:
        assert not got.any()
    else:  # all there are: the last position is 2^31 - 2, from where a window of 2^31 - 1 begins at token 0
        want, bound = attend64(q, cache, longer, [room + 1000] * 4, starts, 0.125, causal, 0)
        compare(got, want, bound)


def test_append_leaves_what_is_not_its_own(gpu):
    """Rows at negative positions, pages that are none, lengths past the table, rows behind the last sequence; starts that
    no batch has."""
    page, dim = 16, 64
    cache, table = make(gpu, [40, 40, 40], 1, page, dim, seed=9)
    table[1, 1] = -1
    table[1, 2] = cache.k.shape[0]
    lengths, rows = [3, 40, 1000], [10, 40, 20]
    g = torch.Generator().manual_seed(97)
    k, v = (torch.randn((75, 1, dim), generator=g).to(F16) for _ in "kv")
    want = [t.cpu().clone() for t in cache]
    layer.cache_append(k.to(gpu), v.to(gpu), cache, table.to(gpu), i32(lengths, gpu), starts=i32(starts_of(rows), gpu),
                       max_rows=40)
    append_steps(want, k, v, table[:2], lengths[:2], [0, 10, 50])
    same_cache(cache, want)
    layer.cache_append(k.to(gpu), v.to(gpu), cache, table.to(gpu), i32([-3, 40, 40], gpu), starts=i32([70, -5, 1 << 30, 3], gpu),
                       max_rows=40)
    torch.cuda.synchronize()


# -- thousands of sequences ------------------------------------------------------------------

@pytest.mark.parametrize("dtype,sequences,rows,heads,kv_heads,dim,even,width", [
    (BF16, 3000, 1, 2, 2, 64, True, 0), (BF16, 3000, 1, 2, 2, 64, False, 0), (F16, 9000, 1, 4, 1, 64, False, 0),
    (F16, 9000, 1, 4, 1, 64, False, 4000), (BF16, 2000, 2, 2, 1, 128, False, 4000), (BF16, 2300, 2, 2, 1, 128, False, 4000),
    (F16, 1500, 5, 4, 1, 64, True, 0),  # 16 and 32 columns a workgroup
    (BF16, 5000, 3, 16, 1, 128, False, 0), (BF16, 70, 130, 1, 1, 64, False, 0), (F16, 200, 40, 12, 1, 64, True, 0),
    (BF16, 257, 9, 24, 4, 128, False, 0)])
def test_thousands_of_sequences(gpu, dtype, sequences, rows, heads, kv_heads, dim, even, width):
    """Each gets what it gets in a batch of its own: short ones of many lengths, some with neither rows nor tokens."""
    g = torch.Generator().manual_seed(sequences)
    n = [rows] * sequences if even else [0 if i % 7 == 3 else 1 + (5 * i) % rows for i in range(sequences)]
    lengths = [0 if i % 11 == 5 else (13 * i) % 45 + m for i, m in enumerate(n)]
    cache, table = make(gpu, [48] * 40, kv_heads, 16, dim, seed=sequences)
    table = table[torch.randint(0, 40, (sequences,), generator=g)]
    room = -(-max(lengths) // 16)  # the same pages again where a sequence is longer
    table = table.repeat(1, -(-room // table.shape[1]))[:, :room].contiguous()
    q, starts = queries(sum(n), heads, dim, dtype, gpu, seed=sequences), starts_of(n)
    wide = torch.nn.functional.pad(table, (0, max(0, width // 16 - room)), value=-1).to(gpu)
    out = torch.full((sum(n) + (0 if even else 3), heads, dim), 7.0, dtype=dtype, device=gpu)  # rows behind the last sequence
    layer.cache_attention(torch.cat([q, q[:out.shape[0] - sum(n)]]), cache, wide, i32(lengths, gpu), out=out,
                          **(dict() if even else dict(starts=i32(starts, gpu), max_rows=rows)))
    assert bool((out[sum(n):] == 7.0).all())
    some = sorted({0, 1, 63, 64, 65, sequences - 1, *torch.randint(0, sequences, (40,), generator=g).tolist()} & set(range(sequences)))
    for b in some:
        if n[b]:
            mine = slice(starts[b], starts[b + 1])
            compare(out[mine], *attend64(q[mine], cache, table[b:b + 1], [lengths[b]], [0, n[b]], dim ** -0.5, True, 0))
    if rows * heads // kv_heads > 32:  # the rest may take another kernel in small batches
        return
    for b0 in range(0, sequences, 50):
        b1 = min(b0 + 50, sequences)
        mine = slice(starts[b0], starts[b1])
        small = layer.cache_attention(q[mine], cache, table[b0:b1].to(gpu), i32(lengths[b0:b1], gpu),
                                      starts=i32([s - starts[b0] for s in starts[b0:b1 + 1]], gpu), max_rows=rows)
        assert torch.equal(out[mine], small)


def test_starts_that_no_large_batch_has(gpu):
    """Whatever starts say, nothing leaves the arrays and every workgroup ends."""
    cache, table = make(gpu, [40], 2, 16, 64, seed=96)
    q, g = queries(5000, 2, 64, BF16, gpu, seed=96), torch.Generator().manual_seed(96)
    for n, group in ((5000, 1), (300, 1), (300, 17)):
        rows = q[:, :1].expand(-1, 2 * group, -1)
        for starts in (torch.randint(-(2 ** 31), 2 ** 31 - 1, (n + 1,), generator=g), torch.randint(-9, 5009, (n + 1,), generator=g),
                       torch.arange(n, -1, -1), torch.full((n + 1,), 2 ** 31 - 1), torch.zeros(n + 1)):
            layer.cache_attention(rows, cache, table.expand(n, -1).contiguous().to(gpu), i32([40] * n, gpu),
                                  starts=starts.to(torch.int32).to(gpu), max_rows=7)
            torch.cuda.synchronize()


# -- more parts than the joining kernel holds at once ---------------------------------------

@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,slope,others", [(1, 0.0, 0), (16, 0.0, 0), (1, 3.0, 0), (16, -3.0, 0), (8, 0.0, 79), (8, 3.0, 79)])
def test_each_of_many_parts_counts(gpu, dtype, rows, slope, others):
    """70000 tokens of one key head, in over 500 parts, alone and among short sequences (a column then has fewer threads in
    the join). Channel c is zero but in its own 64th of the tokens, so that it is missing, or doubled, where those are."""
    page, length, dim = 256, 70000, 64
    cache, table = make(gpu, [length], 1, page, dim, seed=95)
    at, t = table[0].long(), torch.arange(table.shape[1] * page)
    # Scores 0, or rising or falling along the tokens by `slope` in all, a step every 276 of them.
    k, v = torch.zeros((len(t), dim), dtype=torch.int8), torch.zeros((len(t), dim), dtype=torch.int8)
    step = (t // 276).clamp_max(253) - 127
    k[:, 0] = step.to(torch.int8) if slope else 0
    mine = t * dim // length
    inside = t < length
    v[t[inside], mine[inside]] = (60 + mine[inside]).to(torch.int8)
    cache.k[at, 0], cache.v[at, 0] = k.view(-1, page, dim).to(gpu), v.view(-1, page, dim).to(gpu)
    cache.k_scales.fill_(0.5)
    cache.v_scales.fill_(1.0)
    q = torch.zeros((rows * (1 + others), 2, dim), dtype=dtype, device=gpu)
    q[..., 0] = 1.0
    scale = torch.tensor(slope / 127, dtype=torch.float32).item()
    w = torch.softmax(step[:length].double() * 0.5 * scale, 0)
    want = (w @ v[:length].double()).expand(rows, 2, dim)
    # Half a step of a half for each weight, in both sums; an exponent below 16 with five roundings of 2^-21, times ln 2,
    # in both; at most 1024 additions in fp32 in a row (a part's tokens, and the parts); the output's rounding.
    bound = want.abs() * (2.0 ** -10 + 7 * 2.0 ** -21 + 2.0 ** -13 + half_step(dtype))
    assert bool((want > 20 * bound).all())  # a channel that is missing, doubled or another's is seen
    short = torch.full((others, table.shape[1]), -1, dtype=torch.int32)
    short[:, 0] = table[0, 0]  # its first five tokens, which are alike
    got = run(q, cache, torch.cat([table, short]), [length] + [5] * others, [i * rows for i in range(2 + others)], gpu,
              causal=False, scale=scale)
    compare(got[:rows], want, bound)
    alike = v[0].double().expand(rows * others, 2, dim)
    compare(got[rows:], alike, alike * (2.0 ** -10 + half_step(dtype)))
    drop = torch.ones(length, dtype=torch.float64)
    drop[256 * 128:257 * 128] = 0  # what the loss of one part alone would do
    assert bool((((w * drop) @ v[:length].double() - want[0, 0]).abs() > 2 * bound[0, 0]).any())
