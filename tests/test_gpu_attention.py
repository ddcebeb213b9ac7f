"""Rotary positions, the 8-bit cache and attention over it against plain implementations in 64 bits.

Tolerances are sums of the roundings that the definitions allow: half a step of the output's type, half a step of a half
for each softmax weight, and the fp32 sums (each test says which)."""
import math

import pytest
import torch

from trifuse_amd import layer

pytestmark = pytest.mark.gpu

DT = [torch.bfloat16, torch.float16]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# -- references ----------------------------------------------------------------

def turn64(x, positions, f, interleaved, scale):
    """x [rows, heads, D] in 64 bits, pairs turned."""
    n = f.numel()
    y = x.double().clone()
    a = positions.double()[:, None, None] * f
    c, s = scale * torch.cos(a), scale * torch.sin(a)
    i = slice(0, 2 * n, 2) if interleaved else slice(0, n)
    j = slice(1, 2 * n, 2) if interleaved else slice(n, 2 * n)
    u, v = x.double()[..., i], x.double()[..., j]
    y[..., i], y[..., j] = u * c - v * s, v * c + u * s
    return y


def sequences_of(starts, lengths, table, page):
    """[(first row, rows, length)] as the library holds them to the arrays."""
    return [(a, b - a, min(n, table.shape[1] * page)) for a, b, n in zip(starts, starts[1:], lengths)]


def attend64(q, cache, table, lengths, starts, scale, causal, window):
    """(out, bound): the definition in 64 bits on the CPU, and how far a result may be from it."""
    ck, cv, sk, sv = (t.cpu().double() for t in cache)
    pages, kv_heads, page, dim = cache.k.shape
    q = q.cpu()
    rows, heads = q.shape[:2]
    group = heads // kv_heads
    out, bound = torch.zeros(rows, heads, dim, dtype=torch.float64), torch.zeros(rows, heads, dim, dtype=torch.float64)
    for b, (start, n, length) in enumerate(sequences_of(starts, lengths, table, page)):
        ids = table[b].tolist()
        there = torch.tensor([0 <= ids[t // page] < pages for t in range(length)], dtype=torch.bool)
        at = torch.tensor([ids[t // page] if there[t] else 0 for t in range(length)], dtype=torch.long)
        off = torch.arange(length) % page
        for h in range(heads):
            g = h // group
            k, v = ck[at, g, off] * sk[at, g][:, None], cv[at, g, off] * sv[at, g][:, None]
            t, p = torch.arange(length), torch.arange(length - n, length)[:, None]
            sees = there.expand(n, length)
            if causal:
                sees = sees & (t <= p)
            if window:
                sees = sees & (t > p - window)
            some = sees.any(1)
            if not some.any():
                continue
            sees, row, to = sees[some], q[start:start + n, h].double()[some], torch.arange(start, start + n)[some]
            w = torch.softmax((row @ k.t() * scale).masked_fill(~sees, -math.inf), 1)
            out[to, h] = w @ v
            # fp32 sums of a score (D products, of codes plus 128, and the exponent's arithmetic) as a relative error of
            # its weight, twice for the quotient; half a step of a half for each weight, in both sums; weights
            # below 2^-14 of the first to half their smallest step, 2^-25: 127 codes of the largest scale in one
            # sum, up to 16 times its scale's in the other; the output's own rounding.
            lifted = k.abs() + 128 * sk[at, g][:, None]
            most = (row.abs() @ lifted.t()).masked_fill(~sees, 0).amax(1) * abs(scale)
            score, count = (dim + 16) * 2.0 ** -24 * (most + 8), sees.sum(1)
            largest = sv[at, g].expand_as(sees).masked_fill(~sees, 0).amax(1)
            bound[to, h] = (w @ v.abs()) * (2 * score + 2.0 ** -11 + 2.0 ** -20 + count * 2.0 ** -21)[:, None] \
                + (count * 2.0 ** -25 * 127 * largest)[:, None] + half_step(q.dtype) * out[to, h].abs()
    return out, bound


def make(gpu, lengths, kv_heads, page, dim, seed, spare=3, value_scale=1.0):
    """A cache with random codes for sequences of these lengths, its pages in any order, and the table (-1 behind the ends)."""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // page) for n in lengths]
    pages, width = sum(counts) + spare, max(max(counts), 1)
    ids = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    for b, n in enumerate(counts):
        for j in range(n):
            table[b, j] = ids.pop()
    shape = (pages, kv_heads, page, dim)
    codes = [(torch.randn(shape, generator=g) * 40).round().clamp(-127, 127).to(torch.int8) for _ in "kv"]
    scales = [(torch.rand(shape[:2], generator=g) + 0.5) / 40 * s for s in (1.0, value_scale)]
    return layer.KVCache(*(t.to(gpu) for t in (*codes, *scales))), table


def run(q, cache, table, lengths, starts, gpu, width=0, spare=0, **kw):
    """width: tokens that the table has room for at least, spare: rows (NaN) behind the last sequence's; with long tables or
    many rows other kernels take the same sequences."""
    if width > table.shape[1] * cache.k.shape[2]:
        table = torch.nn.functional.pad(table, (0, -(-width // cache.k.shape[2]) - table.shape[1]), value=-1)
    most = max((b - a for a, b in zip(starts, starts[1:])), default=0)
    rows = q.shape[0]
    q = torch.cat([q, q.new_full((spare,) + q.shape[1:], math.nan)]) if spare else q
    out = layer.cache_attention(q, cache, table.to(gpu), torch.tensor(lengths, dtype=torch.int32, device=gpu),
                                starts=torch.tensor(starts, dtype=torch.int32, device=gpu), max_rows=kw.pop("max_rows", most), **kw)
    return out[:rows] if spare else out


def queries(rows, heads, dim, dtype, gpu, seed, sigma=1.0):
    g = torch.Generator().manual_seed(seed + 1000)
    return (torch.randn((rows, heads, dim), generator=g) * sigma).to(dtype).to(gpu)


def compare(got, want, bound):
    got = got.cpu().double()
    assert torch.isfinite(got).all()
    off = (got - want).abs()
    assert bool((off <= bound).all()), (float((off - bound).max()), float(off.max()), float((off / bound.clamp_min(1e-30)).max()))


def starts_of(rows):
    return [sum(rows[:i]) for i in range(len(rows) + 1)]


# -- rotary --------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,heads,dim,pairs,interleaved,far,bits", [
    (1, 16, 128, 64, False, 5, 64),
    (1, 1, 2, 1, False, 1, 32),
    (37, 24, 64, 16, True, 2_000_000, 64),
    (37, 5, 64, 8, False, 2_000_000_000, 32),
    (5, 33, 80, 40, False, 100, 64),
    (70, 3, 33, 13, True, 4096, 32),
    (9, 2, 33, 16, False, 4096, 64),
    (3, 2, 1024, 512, True, 1 << 20, 64),
    (515, 7, 96, 3, False, 1 << 20, 64),
])
def test_rotary(gpu, dtype, rows, heads, dim, pairs, interleaved, far, bits):
    g = torch.Generator().manual_seed(rows + dim)
    x = (torch.randn((rows, heads, dim), generator=g) * 2).to(dtype)
    positions = torch.randint(-far, far + 1, (rows,), generator=g).to(torch.int64 if bits == 64 else torch.int32)
    f, _ = layer.rotary_frequencies(pairs)
    scale = 1.25
    got = layer.rotary(x.to(gpu), positions.to(gpu), f.to(gpu), interleaved=interleaved, scale=scale).cpu()
    want = turn64(x, positions, f, interleaved, scale)
    assert torch.equal(got[..., 2 * pairs:], x[..., 2 * pairs:])
    # cosine and sine to 4 steps of fp32 of 1 (the turn's rounding to fp32 times 2 pi, the polynomials' roundings, the
    # scale's), an angle to 2^-51 of itself, two products and a sum; the output's rounding, subnormal halves included.
    size = x.double().abs()
    pair = torch.zeros_like(size)
    i = slice(0, 2 * pairs, 2) if interleaved else slice(0, pairs)
    j = slice(1, 2 * pairs, 2) if interleaved else slice(pairs, 2 * pairs)
    pair[..., i] = pair[..., j] = (size[..., i] + size[..., j]) * scale
    bound = pair * (6 * 2.0 ** -23 + far * 2.0 ** -50) + half_step(dtype) * want.abs() + 2.0 ** -25
    off = (got.double() - want).abs()[..., :2 * pairs]
    assert bool((off <= bound[..., :2 * pairs]).all()), float((off / bound[..., :2 * pairs]).max())


def test_rotary_views_and_in_place(gpu):
    g = torch.Generator().manual_seed(3)
    fused = torch.randn((11, (4 + 2 + 2) * 64 + 6), generator=g).to(torch.bfloat16).to(gpu)
    positions, (f, _) = torch.arange(11, device=gpu), layer.rotary_frequencies(32, device=gpu)
    q = fused[:, 2:2 + 256].unflatten(1, (4, 64))  # not 16-byte aligned
    want = layer.rotary(q.contiguous(), positions, f)
    assert torch.equal(layer.rotary(q, positions, f), want)
    by_head = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(layer.rotary(by_head, positions, f, out=torch.empty_like(by_head)), want)
    shared = q[:, :1].expand(-1, 3, -1)
    assert torch.equal(layer.rotary(shared, positions, f), want[:, :1].expand(-1, 3, -1))
    rest = fused.clone()
    assert layer.rotary(q, positions, f, out=q) is q
    assert torch.equal(q, want)
    assert torch.equal(fused[:, :2], rest[:, :2]) and torch.equal(fused[:, 258:], rest[:, 258:])
    part = torch.randn((11, 4, 64), generator=g).to(torch.float16).to(gpu)
    half, (f8, _) = part.clone(), layer.rotary_frequencies(8, device=gpu)
    layer.rotary(half, positions, f8, out=half)
    assert torch.equal(half, layer.rotary(part, positions, f8))
    assert layer.rotary(part[:0], positions[:0], f8).shape == (0, 4, 64)


def test_rotary_refusals(gpu):
    x, p = torch.zeros((4, 2, 64), dtype=torch.bfloat16, device=gpu), torch.arange(4, device=gpu)
    f, _ = layer.rotary_frequencies(32, device=gpu)
    for bad, err in ((dict(x=x.float()), NotImplementedError), (dict(x=x[0]), ValueError), (dict(x=x[..., ::2]), ValueError),
                     (dict(positions=p[:3]), ValueError), (dict(positions=p.float()), ValueError), (dict(positions=p.cpu()), ValueError),
                     (dict(frequencies=f.float()), ValueError), (dict(frequencies=f.cpu()), ValueError),
                     (dict(frequencies=torch.cat([f, f])), RuntimeError), (dict(out=x[:2]), ValueError),
                     (dict(out=x.half()), ValueError), (dict(out=x[:1].expand(4, 2, 64)), RuntimeError),
                     (dict(scale=math.nan), RuntimeError)):
        with pytest.raises(err):
            layer.rotary(**{**dict(x=x, positions=p, frequencies=f), **bad})


# -- append and read -----------------------------------------------------------

def append_steps(cache, k, v, table, lengths, starts):
    """The definition of an append without rotation, in fp32 on the CPU: bit for bit."""
    pages, kv_heads, page, dim = cache[0].shape
    codes, scales = cache[:2], cache[2:]
    for b, (start, n, length) in enumerate(sequences_of(starts, lengths, table, page)):
        first = length - n
        for j in range(max(first, 0) // page, -(-length // page)):
            begin, end = max(first, 0, j * page), min(length, (j + 1) * page)
            at = int(table[b, j])
            if begin >= end or not 0 <= at < pages:
                continue
            p = begin - j * page
            for c, s, x in zip(codes, scales, (k, v)):
                new = x[start + begin - first:start + end - first].float()  # [tokens, heads, dim]
                for h in range(kv_heads):
                    old = s[at, h].clone() if p else torch.zeros(())
                    now = torch.maximum(old, new[:, h].abs().max().clamp_min(2.0 ** -40) / torch.tensor(127.0))
                    if not bool(torch.isfinite(new[:, h]).all()) or not bool(torch.isfinite(old)):
                        now = torch.tensor(math.nan)
                    if p and now > old:
                        c[at, h, :p] = (c[at, h, :p].float() * (old / now)).round().to(torch.int8)
                    made = (new[:, h] * (torch.tensor(1.0) / now)).round() if bool(now == now) else torch.zeros_like(new[:, h])
                    c[at, h, p:p + end - begin] = made.to(torch.int8)
                    s[at, h] = now


def same_cache(cache, want):
    for got, w in zip(cache, want):
        g = got.cpu()
        assert torch.equal(torch.isnan(g.float()), torch.isnan(w.float())) and torch.equal(torch.nan_to_num(g.float()), torch.nan_to_num(w.float()))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("page,kv_heads,dim", [(16, 3, 64), (16, 2, 128), (32, 1, 64), (64, 2, 128), (128, 1, 128), (256, 1, 128), (256, 2, 64)])
def test_append_is_its_definition(gpu, dtype, page, kv_heads, dim):
    """Several steps of several sequences: pages begun, filled, ended inside; scales that grow and that stay; bit for bit."""
    g = torch.Generator().manual_seed(page + dim)
    steps = [[page + 3, 1, 0, 2 * page], [1, 1, 5, 1], [0, 2, 1, 1], [page - 4, 1, 1, page + 1]]
    totals = [sum(s[b] for s in steps) for b in range(4)]
    cache, table = make(gpu, totals, kv_heads, page, dim, seed=page)
    want = [t.cpu().clone() for t in cache]
    lengths = [0] * 4
    for i, rows in enumerate(steps):
        lengths = [n + r for n, r in zip(lengths, rows)]
        starts = starts_of(rows)
        total = starts[-1] + 2  # rows behind the last sequence
        k, v = ((torch.randn((total, kv_heads, dim), generator=g) * (1 + i)).to(dtype) for _ in "kv")
        layer.cache_append(k.to(gpu), v.to(gpu), cache, table.to(gpu), torch.tensor(lengths, dtype=torch.int32, device=gpu),
                           starts=torch.tensor(starts, dtype=torch.int32, device=gpu), max_rows=max(rows))
        append_steps(want, k, v, table, lengths, starts)
        same_cache(cache, want)
    for kind in (torch.float32, torch.bfloat16, torch.float16):
        back = 2 * page + 1
        rk, rv = layer.cache_read(cache, table.to(gpu), torch.tensor(lengths, dtype=torch.int32, device=gpu), back, kind)
        for got, codes, scales in ((rk, want[0], want[2]), (rv, want[1], want[3])):
            got = got.cpu().view(4, back, kv_heads, dim)
            for b, n in enumerate(lengths):
                for i in range(back):
                    t = n - back + i
                    if t < 0:
                        assert not got[b, i].any()
                    else:
                        at = int(table[b, t // page])
                        assert torch.equal(got[b, i], (codes[at, :, t % page].float() * scales[at][:, None]).to(kind))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("dim,pairs,interleaved", [(64, 32, False), (128, 64, False), (128, 64, True), (64, 8, False), (128, 24, True)])
def test_append_turns_keys(gpu, dtype, dim, pairs, interleaved):
    page, rows, lengths = 32, [45, 1, 70], [45, 100, 1070]
    cache, table = make(gpu, lengths, 2, page, dim, seed=dim + pairs)
    g = torch.Generator().manual_seed(5)
    k, v = (torch.randn((116, 2, dim), generator=g).to(dtype) for _ in "kv")
    f, _ = layer.rotary_frequencies(pairs)
    starts = starts_of(rows)
    position = torch.cat([torch.arange(n - r, n) for r, n in zip(rows, lengths)])
    turned = turn64(k, position, f, interleaved, 1.25)
    before = [t.cpu().clone() for t in cache]
    layer.cache_append(k.to(gpu), v.to(gpu), cache, table.to(gpu), torch.tensor(lengths, dtype=torch.int32, device=gpu),
                       starts=torch.tensor(starts, dtype=torch.int32, device=gpu), max_rows=70, frequencies=f.to(gpu),
                       interleaved=interleaved, rotary_scale=1.25)
    append_steps(before, turned.float(), v, table, lengths, starts)  # keys turned in 64 bits
    got = [t.cpu() for t in cache]
    assert torch.equal(got[1], before[1]) and torch.equal(got[3], before[3])
    # A turned key is right to 2^-19 of its pair (the angle's 2^-50 of 1070 turns included), which is at most 2^-17 of a
    # page's largest, and so is its scale; a code then differs only where its value lies that near to a tie, by one.
    assert bool(((got[2] - before[2]).abs() <= 2.0 ** -18 * before[2]).all())
    off = (got[0].int() - before[0].int()).abs()
    assert int(off.max()) <= 1 and float(off.float().mean()) <= 2 * 127 * 2.0 ** -17


def test_append_strides_and_same_length_batches(gpu):
    page, n = 16, 5
    cache, table = make(gpu, [20, 33], 2, page, 64, seed=1)
    other = layer.KVCache(*(t.clone() for t in cache))
    fused = torch.randn((2 * n, 6 * 64 + 2), device=gpu).to(torch.bfloat16)
    k, v = fused[:, 2 * 64 + 1:4 * 64 + 1].unflatten(1, (2, 64)), fused[:, 4 * 64 + 1:6 * 64 + 1].unflatten(1, (2, 64))
    lengths = torch.tensor([20, 33], dtype=torch.int32, device=gpu)
    layer.cache_append(k, v, cache, table.to(gpu), lengths)  # without starts: five rows each
    layer.cache_append(k.contiguous(), v.transpose(0, 1).contiguous().transpose(0, 1), other, table.to(gpu), lengths,
                       starts=torch.tensor([0, 5, 10], dtype=torch.int32, device=gpu))
    for a, b in zip(cache, other):
        assert torch.equal(a, b)


def test_append_leaves_what_is_not_its_own(gpu):
    """Rows at negative positions, pages that are none, lengths past the table, rows behind the last sequence."""
    page, dim = 16, 64
    cache, table = make(gpu, [40, 40, 40], 1, page, dim, seed=9)
    table[1, 1] = -1
    table[1, 2] = cache.k.shape[0]
    lengths, rows = [3, 40, 1000], [10, 40, 20]
    k, v = (torch.randn((75, 1, dim)).to(torch.float16) for _ in "kv")
    want = [t.cpu().clone() for t in cache]
    layer.cache_append(k.to(gpu), v.to(gpu), cache, table.to(gpu), torch.tensor(lengths, dtype=torch.int32, device=gpu),
                       starts=torch.tensor(starts_of(rows), dtype=torch.int32, device=gpu), max_rows=40)
    append_steps(want, k, v, table, lengths, starts_of(rows))
    same_cache(cache, want)
    strange = torch.tensor([70, -5, 1 << 30, 3], dtype=torch.int32, device=gpu)  # starts that no batch has: nothing leaves the arrays
    layer.cache_append(k.to(gpu), v.to(gpu), cache, table.to(gpu), torch.tensor([-3, 40, 40], dtype=torch.int32, device=gpu),
                       starts=strange, max_rows=40)
    torch.cuda.synchronize()


def test_append_not_finite(gpu):
    page, dim = 16, 64
    cache, table = make(gpu, [20, 20], 2, page, dim, seed=4)
    want = [t.cpu().clone() for t in cache]
    for step, (lengths, rows) in enumerate([([10, 18], [10, 18]), ([12, 20], [2, 2]), ([8, 4], [8, 4])]):
        k, v = (torch.randn((sum(rows), 2, dim)).to(torch.bfloat16) for _ in "kv")
        if step == 0:
            k[3, 0, 5], v[12, 1, 0] = math.inf, math.nan
        layer.cache_append(k.to(gpu), v.to(gpu), cache, table.to(gpu), torch.tensor(lengths, dtype=torch.int32, device=gpu),
                           starts=torch.tensor(starts_of(rows), dtype=torch.int32, device=gpu), max_rows=18)
        append_steps(want, k, v, table, lengths, starts_of(rows))
        same_cache(cache, want)
        assert bool(torch.isnan(want[2]).any()) == (step < 2)  # a page that starts anew is whole again


# -- attention -----------------------------------------------------------------

@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("heads,kv_heads,dim,page,rows,lengths,causal,window", [
    (2, 2, 128, 64, [1], [1], True, 0),
    (2, 2, 64, 16, [1, 1, 1, 1, 1], [1, 17, 0, 130, 33], True, 0),
    (6, 2, 64, 16, [1, 0, 1, 1], [300, 12, 31, 32], True, 0),
    (8, 2, 128, 32, [1, 1], [257, 100], True, 40),
    (8, 1, 128, 16, [4, 2, 3], [100, 2, 65], True, 0),
    (6, 2, 64, 128, [5, 5], [70, 500], True, 7),
    (4, 2, 128, 64, [5, 16, 7], [5, 200, 150], False, 0),
    (40, 1, 64, 16, [1, 2], [90, 161], True, 0),
    (2, 2, 128, 64, [65, 3, 130], [65, 80, 200], True, 0),
    (3, 1, 64, 32, [43, 90], [43, 300], True, 33),
    (4, 2, 64, 256, [100, 33], [300, 33], False, 0),
    (7, 1, 128, 128, [37], [129], True, 1),
    (2, 1, 64, 16, [100], [64], True, 0),
    (1, 1, 128, 16, [20, 4], [3, 0], True, 0),
])
def test_attention(gpu, dtype, heads, kv_heads, dim, page, rows, lengths, causal, window):
    cache, table = make(gpu, lengths, kv_heads, page, dim, seed=sum(lengths) + dim)
    q = queries(sum(rows), heads, dim, dtype, gpu, seed=page)
    starts = starts_of(rows)
    got = run(q, cache, table, lengths, starts, gpu, causal=causal, window=window)
    compare(got, *attend64(q, cache, table, lengths, starts, dim ** -0.5, causal, window))
    assert torch.equal(got, run(q, cache, table, lengths, starts, gpu, causal=causal, window=window))  # the same bits again


@pytest.mark.parametrize("heads,kv_heads,dim,rows,length,window", [
    (2, 2, 128, 1, 3001, 0), (6, 2, 64, 1, 2500, 0), (8, 2, 128, 7, 2100, 0), (8, 2, 64, 9, 2100, 1500), (3, 3, 64, 50, 1500, 0),
    (2, 1, 128, 40, 1300, 1000)])
def test_attention_in_parts(gpu, heads, kv_heads, dim, rows, length, window):
    """Long sequences that several workgroups share, beside a short one and an empty one."""
    lengths, n = [length, 5, 0], [rows, 1, 1]
    cache, table = make(gpu, lengths, kv_heads, 16, dim, seed=length)
    q = queries(sum(n), heads, dim, torch.float16, gpu, seed=dim)
    got = run(q, cache, table, lengths, starts_of(n), gpu, window=window)
    compare(got, *attend64(q, cache, table, lengths, starts_of(n), dim ** -0.5, True, window))


# Rows of a sequence with two heads a key head, the table's room, rows behind the batch: one kernel of 16 columns a workgroup,
# one of 32 (with few and many rows), and tiles of 64, 128 and 256.
FORMS = [(1, 0, 0), (9, 0, 0), (40, 0, 0), (40, 0, 4500), (40, 500000, 0), (68, 500000, 0)]


@pytest.mark.parametrize("rows,width,spare", FORMS)
def test_sharp_scores(gpu, rows, width, spare):
    """Scores tens of steps of the running maximum apart, rising and falling along the tokens; sign and size of the scale."""
    lengths = [390 if spare else 700]
    cache, table = make(gpu, lengths, 2, 16, 64, seed=8)
    ramp = torch.ones((cache.k_scales.shape[0], 1), device=gpu)
    ramp[table[0].long(), 0] = torch.linspace(0.02, 3.0, table.shape[1], device=gpu)
    q = queries(rows, 4, 64, torch.bfloat16, gpu, seed=1)
    for scales in (cache.k_scales * 3, cache.k_scales * ramp, cache.k_scales * (3.02 - ramp)):
        c = cache._replace(k_scales=scales)
        for scale in (0.125, -0.125, 0.0, 1e-30):
            got = run(q, c, table, lengths, [0, rows], gpu, width, spare, scale=scale)
            compare(got, *attend64(q, c, table, lengths, [0, rows], scale, True, 0))


@pytest.mark.parametrize("rows,width,spare", FORMS)
@pytest.mark.parametrize("spread", [2.0 ** 20, 2.0 ** 60, 2.0 ** 90])
def test_pages_of_very_different_values(gpu, rows, width, spare, spread):
    """Zero pages and small ones beside large ones: each row is right to its own terms."""
    lengths = [200]
    cache, table = make(gpu, lengths, 1, 16, 64, seed=21)
    used = table[0].long().to(gpu)
    for order in (used[::2], used[1::2], used[:3]):
        vs, v = cache.v_scales.clone(), cache.v.clone()
        vs[order] /= spread
        v[order[:1]] = 0
        c = cache._replace(v_scales=vs, v=v)
        q = queries(rows, 2, 64, torch.bfloat16, gpu, seed=2)
        got = run(q, c, table, lengths, [0, rows], gpu, width, spare)
        compare(got, *attend64(q, c, table, lengths, [0, rows], 0.125, True, 0))


@pytest.mark.parametrize("rows,width,spare", FORMS)
def test_scales_of_zero(gpu, rows, width, spare):
    """Pages that hold zeros by their scale (never written, say) take their part of the weight and add nothing; so do all."""
    lengths = [200]
    cache, table = make(gpu, lengths, 1, 16, 64, seed=22)
    used = table[0].long().to(gpu)
    q = queries(rows, 2, 64, torch.bfloat16, gpu, seed=2)
    for zero_k, zero_v in ((used[::2], used[:0]), (used[:0], used[1::2]), (used[:4], used[:4]), (used[5:], used[5:]), (used, used)):
        ks, vs = cache.k_scales.clone(), cache.v_scales.clone()
        ks[zero_k], vs[zero_v] = 0, 0
        c = cache._replace(k_scales=ks, v_scales=vs)
        want, bound = attend64(q, c, table, lengths, [0, rows], 0.125, True, 0)
        # a value scale below 2^-100 counts as that: 128 of it at most
        compare(run(q, c, table, lengths, [0, rows], gpu, width, spare), want, bound + 2.0 ** -93)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,width,spare", FORMS)
def test_queries_of_any_size(gpu, dtype, rows, width, spare):
    """Halves as they are, bf16 from its smallest normals to 2^100: products stay exact."""
    lengths = [90]
    cache, table = make(gpu, lengths, 1, 32, 64, seed=30)
    for size in ((1.0, 2.0 ** -13, 2.0 ** 8) if dtype == torch.float16 else (1.0, 2.0 ** -126, 2.0 ** -60, 2.0 ** 100)):
        q = (queries(rows, 2, 64, torch.float32, gpu, seed=3) * size).to(dtype)
        scale = float(torch.tensor(0.125 / size, dtype=torch.float32))
        if not math.isfinite(scale * 1.5):
            continue
        got = run(q, cache, table, lengths, [0, rows], gpu, width, spare, scale=scale)
        compare(got, *attend64(q, cache, table, lengths, [0, rows], scale, True, 0))


@pytest.mark.parametrize("rows,width,spare", FORMS)
def test_not_finite_where_nothing_is_seen(gpu, rows, width, spare):
    """NaN scales of pages that no row, or only later rows, see; unused pages and entries; NaN queries of one row."""
    page, lengths = 16, [100, max(50, rows + 2)]
    cache, table = make(gpu, lengths, 2, page, 64, seed=40)
    starts, n = [0, rows, 2 * rows], 2 * rows
    q = queries(n, 4, 64, torch.bfloat16, gpu, seed=4)
    free = sorted(set(range(cache.k.shape[0])) - set(table.flatten().tolist()))
    ks, vs = cache.k_scales.clone(), cache.v_scales.clone()
    ks[free], vs[free] = math.nan, math.inf
    c = cache._replace(k_scales=ks, v_scales=vs)
    want, bound = attend64(q, cache, table, lengths, starts, 0.125, True, 0)
    compare(run(q, c, table, lengths, starts, gpu, width, spare), want, bound)
    # A poisoned page reaches the rows that see it, and no other.
    bad = c._replace(v_scales=vs.clone(), k_scales=ks.clone())
    bad.v_scales[table[0, 6]] = math.nan  # tokens 96 ..
    bad.k_scales[table[1, 0]] = math.nan  # tokens 0 .. 15
    got = run(q, bad, table, lengths, starts, gpu, width, spare).cpu()
    position = torch.arange(100 - rows, 100)
    first = got[:rows]
    assert bool(torch.isnan(first[position >= 96]).all())
    if (position < 96).any():
        compare(first[position < 96], want[:rows][position < 96], bound[:rows][position < 96])
    assert bool(torch.isnan(got[rows:]).all())
    windowed = run(q, bad, table, lengths, starts, gpu, width, spare, window=3)[rows:].cpu()  # rows past token 18 see nothing of page 0
    w, bd = attend64(q, cache, table, lengths, starts, 0.125, True, 3)
    far = torch.arange(lengths[1] - rows, lengths[1]) >= 18
    compare(windowed[far], w[rows:][far], bd[rows:][far])
    q2 = q.clone()
    q2[0, 1] = math.nan
    got = run(q2, c, table, lengths, starts, gpu, width, spare).cpu()
    assert bool(torch.isnan(got[0, 1]).all())
    keep = torch.ones(n, 4, dtype=torch.bool)
    keep[0, 1] = False
    compare(got[keep], want[keep], bound[keep])


@pytest.mark.parametrize("rows,width,spare", FORMS)
def test_bad_pages_and_odd_batches(gpu, rows, width, spare):
    page, lengths = 16, [100, 100, 64]
    cache, table = make(gpu, lengths, 1, page, 64, seed=50)
    table[0, 2], table[1, 6], table[2, 0] = -1, 10 ** 9, cache.k.shape[0]
    q = queries(3 * rows, 2, 64, torch.float16, gpu, seed=5)
    starts = [0, rows, 2 * rows, 3 * rows]
    compare(run(q, cache, table, lengths, starts, gpu, width, spare), *attend64(q, cache, table, lengths, starts, 0.125, True, 0))
    none = torch.full_like(table, -1)
    assert not run(q, cache, none, lengths, starts, gpu, width, spare).any()
    # Lengths past the table and below zero; starts that no batch has: nothing leaves the arrays.
    run(q, cache, table, [10 ** 9, -4, 100], starts, gpu, width, spare)
    run(q, cache, table, lengths, [5, -3, 1 << 30, 2], gpu, width, spare, max_rows=rows)
    torch.cuda.synchronize()


def test_rows_behind_the_last_sequence_stay(gpu):
    lengths = [40, 9]
    cache, table = make(gpu, lengths, 2, 16, 64, seed=60)
    for rows in ([1, 1], [9, 4], [40, 9]):
        total = sum(rows)
        q = queries(total + 3, 4, 64, torch.bfloat16, gpu, seed=6)
        q[total:] = math.nan
        out = torch.full_like(q, 7.0)
        assert run(q, cache, table, lengths, starts_of(rows), gpu, out=out) is out
        assert bool((out[total:] == 7.0).all())
        compare(out[:total], *(t[:total] for t in attend64(q, cache, table, lengths, starts_of(rows), 0.125, True, 0)))


def test_strided_and_unaligned_queries(gpu):
    lengths, rows = [70, 33], [2, 2]
    cache, table = make(gpu, lengths, 2, 32, 64, seed=70)
    fused = torch.randn((4, 4 * 64 + 7), device=gpu).to(torch.bfloat16)
    q = fused[:, 3:3 + 256].unflatten(1, (4, 64))
    want = run(q.contiguous(), cache, table, lengths, starts_of(rows), gpu)
    assert torch.equal(run(q, cache, table, lengths, starts_of(rows), gpu), want)
    assert torch.equal(run(q.transpose(0, 1).contiguous().transpose(0, 1), cache, table, lengths, starts_of(rows), gpu), want)
    one = q[:1, :1].expand(4, 4, 64)
    assert torch.equal(run(one, cache, table, lengths, starts_of(rows), gpu),
                       run(one.contiguous(), cache, table, lengths, starts_of(rows), gpu))
    lens = torch.tensor(lengths, dtype=torch.int32, device=gpu)
    assert torch.equal(layer.cache_attention(q, cache, table.to(gpu), lens), want)  # without starts: two rows each
    loose = layer.cache_attention(q, cache, table.to(gpu), lens, starts=torch.tensor([0, 2, 4], dtype=torch.int32, device=gpu))
    compare(loose, *attend64(q, cache, table, lengths, starts_of(rows), 0.125, True, 0))


def test_refusals(gpu):
    cache, table = make(gpu, [40, 9], 2, 16, 64, seed=80)
    table, lengths = table.to(gpu), torch.tensor([40, 9], dtype=torch.int32, device=gpu)
    q = queries(2, 4, 64, torch.bfloat16, gpu, seed=8)
    base = dict(q=q, cache=cache, table=table, lengths=lengths)
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device=gpu)
    for bad, err in ((dict(q=q.float()), NotImplementedError), (dict(q=q[0]), ValueError), (dict(q=q[:1]), ValueError),
                     (dict(q=q[:, :3]), RuntimeError), (dict(q=q[..., :32]), ValueError), (dict(table=table.long()), ValueError),
                     (dict(table=table.cpu()), ValueError), (dict(table=table[:1]), ValueError), (dict(lengths=lengths.long()), ValueError),
                     (dict(starts=starts[:2]), ValueError), (dict(starts=starts.long()), ValueError), (dict(max_rows=1), ValueError),
                     (dict(starts=starts, max_rows=-1), ValueError), (dict(window=-1), ValueError),
                     (dict(window=4, causal=False), RuntimeError), (dict(scale=math.inf), RuntimeError),
                     (dict(cache=cache._replace(v=cache.v[..., :32].contiguous())), ValueError),
                     (dict(cache=cache._replace(k=cache.k.transpose(1, 2))), ValueError),
                     (dict(cache=cache._replace(k_scales=cache.k_scales.double())), ValueError),
                     (dict(cache=cache._replace(v_scales=cache.v_scales[:1])), ValueError),
                     (dict(out=q), RuntimeError), (dict(out=q[:1]), ValueError)):
        with pytest.raises(err):
            layer.cache_attention(**{**base, **bad})
    k = queries(2, 2, 64, torch.bfloat16, gpu, seed=9)
    f, _ = layer.rotary_frequencies(32, device=gpu)
    base = dict(k=k, v=k.clone(), cache=cache, table=table, lengths=lengths)
    for bad, err in ((dict(k=k.float()), NotImplementedError), (dict(v=k.half()), ValueError), (dict(k=k[:1]), ValueError),
                     (dict(k=q, v=q), ValueError), (dict(frequencies=f[:12].contiguous()), NotImplementedError),
                     (dict(frequencies=f.float()), ValueError), (dict(frequencies=f, rotary_scale=math.nan), RuntimeError)):
        with pytest.raises(err):
            layer.cache_append(**{**base, **bad})
    for bad in (dict(rows=-1), dict(rows=1 << 30), dict(dtype=torch.float64), dict(dtype="bf16")):
        with pytest.raises(ValueError):
            layer.cache_read(**{**dict(cache=cache, table=table, lengths=lengths, rows=1), **bad})
    assert layer.cache_read(cache, table, lengths, 0)[0].shape == (0, 2, 64)
    assert layer.cache_attention(q[:0], cache, table, lengths).shape == (0, 4, 64)
