"""Rotary positions, the 8-bit cache and attention over it as they are used: large and ragged batches, streams, graphs, a
whole layer, sequences that are taken back."""
import math

import pytest
import torch

from tests.test_gpu_attention import append_steps, attend64, compare, half_step, make, queries, run, same_cache, starts_of, turn64
from trifuse_amd import layer
from trifuse_amd import moe as tmoe
from trifuse_amd import workload as wl

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def i32(values, gpu):
    return torch.tensor(values, dtype=torch.int32, device=gpu)


# -- sizes that pick each kernel, and each way of sharing the work ---------------

@pytest.mark.parametrize("dtype,heads,kv_heads,dim,page,rows,lengths,width,window", [
    (BF16, 4, 2, 128, 64, [200, 131, 256], [2500, 131, 3001], 0, 0),       # 32 columns, in parts
    (F16, 6, 2, 64, 16, [170, 43], [4500, 4200], 0, 0),
    (BF16, 2, 1, 128, 128, [250], [6000], 0, 1000),                         # of which the window leaves a few
    (F16, 2, 2, 64, 256, [1023], [1023], 0, 0),                             # 32 columns, whole
    (BF16, 3, 1, 128, 16, [5, 0, 90, 21], [1000, 16, 90, 900], 0, 65),
    (F16, 12, 12, 128, 16, [380, 300], [380, 333], 0, 0),                   # 64 columns
    (BF16, 24, 12, 64, 32, [130, 200, 60], [130, 390, 100], 0, 77),
    (BF16, 4, 2, 128, 64, [150, 131, 140], [2500, 131, 3001], 100000, 0),   # 128 columns, in parts
    (F16, 4, 4, 64, 16, [100, 43], [4500, 4200], 200000, 0),
    (F16, 24, 24, 128, 64, [1400, 700, 900], [1400, 700, 1000], 0, 129),    # 128, whole
    (F16, 6, 2, 64, 16, [170, 43], [4500, 4200], 200000, 0),                # 256, in parts
    (BF16, 4, 4, 128, 32, [256, 255], [4900, 257], 50000, 0),
    (BF16, 32, 32, 64, 16, [700, 515, 1300, 513, 900, 200], [700, 600, 1300, 513, 950, 333], 0, 0),  # 256, whole
])
def test_tiles(gpu, dtype, heads, kv_heads, dim, page, rows, lengths, width, window):
    cache, table = make(gpu, lengths, kv_heads, page, dim, seed=sum(lengths))
    q = queries(sum(rows), heads, dim, dtype, gpu, seed=dim)
    starts = starts_of(rows)
    got = run(q, cache, table, lengths, starts, gpu, width, window=window)
    some = list(range(0, kv_heads, max(1, kv_heads // 2)))  # a few key heads are enough for the reference
    group = heads // kv_heads
    part = layer.KVCache(*(t[:, some].contiguous() for t in cache))
    columns = [g * group + i for g in some for i in range(group)]
    compare(got[:, columns], *attend64(q[:, columns], part, table, lengths, starts, dim ** -0.5, True, window))
    assert torch.equal(got, run(q, cache, table, lengths, starts, gpu, width, window=window))


@pytest.mark.parametrize("rows,heads", [(1, 4), (3, 4), (20, 2)])
def test_many_sequences(gpu, rows, heads):
    """More sequences than a wave has lanes, empty ones and one long one among them."""
    lengths = [(37 * i) % 211 + rows for i in range(150)]
    lengths[70], lengths[3], lengths[149] = 2900, 0, rows
    n = [rows if i % 9 else 0 for i in range(150)]
    cache, table = make(gpu, lengths, 1, 16, 64, seed=rows)
    q = queries(sum(n), heads, 64, BF16, gpu, seed=rows)
    got = run(q, cache, table, lengths, starts_of(n), gpu)
    compare(got, *attend64(q, cache, table, lengths, starts_of(n), 0.125, True, 0))


@pytest.mark.parametrize("rows", [1, 16])
def test_more_parts_than_a_join_holds(gpu, rows):
    """One key head and 70000 tokens: over 256 parts of the one tile."""
    lengths = [70000]
    cache, table = make(gpu, lengths, 1, 256, 64, seed=1)
    q = queries(rows, 2, 64, F16, gpu, seed=1)
    compare(run(q, cache, table, lengths, [0, rows], gpu), *attend64(q, cache, table, lengths, [0, rows], 0.125, True, 0))


def test_pages_past_32_bits(gpu):
    """Codes whose offsets pass 2^31 and 2^32 bytes; most of the cache stays as it was given."""
    page, dim, heads = 256, 128, 2
    pages = 2 ** 32 // (heads * page * dim) + 40
    shape = (pages, heads, page, dim)
    cache = layer.KVCache(*(torch.empty(shape, dtype=torch.int8, device=gpu) for _ in "kv"),
                          *(torch.full(shape[:2], 7.0, device=gpu) for _ in "kv"))
    ids = [pages - 1, 2 ** 31 // (heads * page * dim), pages - 39, 0, pages - 20]
    for t in cache[:2]:
        t[:, :, :2].fill_(3)  # enough to see a stray write in the pages between
    rows, lengths = [600, 500], [600, 500]
    table = i32([[ids[0], ids[1], ids[2]], [ids[3], ids[4], -1]], gpu)
    k, v = (torch.randn((1100, heads, dim), device=gpu).to(BF16) for _ in "kv")
    layer.cache_append(k, v, cache, table, i32(lengths, gpu), starts=i32(starts_of(rows), gpu), max_rows=600)
    small = layer.KVCache(*(t[ids] for t in cache))
    want = [torch.zeros_like(t.cpu()) for t in small]
    local = torch.tensor([[0, 1, 2], [3, 4, -1]])
    append_steps(want, k.cpu(), v.cpu(), local, lengths, starts_of(rows))
    for b, j, used in ((0, 0, 256), (0, 1, 256), (0, 2, 88), (1, 0, 256), (1, 1, 244)):
        at = int(local[b, j])
        for got, w in zip(small, want):
            assert torch.equal(got[at].cpu()[:, :used] if got.dim() == 4 else got[at].cpu(), w[at][:, :used] if got.dim() == 4 else w[at])
    rest = torch.ones(pages, dtype=torch.bool)
    rest[ids] = False
    for t in cache[:2]:
        assert bool((t[:, :, :2].cpu()[rest] == 3).all())
    for t in cache[2:]:
        assert bool((t.cpu()[rest] == 7).all())
    back = layer.cache_read(cache, table, i32(lengths, gpu), 600, torch.float32)
    for got, c, s in zip(back, want[:2], want[2:]):
        for b, n in ((0, 600), (1, 500)):
            t = torch.arange(n)
            at = local[b][t // page]
            assert torch.equal(got.view(2, 600, heads, dim)[b, 600 - n:].cpu(), c[at, :, t % page].float() * s[at][..., None])
    for take in (1, 30, 100):
        q = queries(2 * take, 4, dim, BF16, gpu, seed=take)
        got = run(q, cache, table, lengths, [0, take, 2 * take], gpu)
        compare(got, *attend64(q, small, local, lengths, [0, take, 2 * take], dim ** -0.5, True, 0))


@pytest.mark.parametrize("dtype,sequences,rows,kv_heads,page,dim,pairs,interleaved", [
    (BF16, 40, 350, 7, 16, 64, 32, False),    # four heads a workgroup
    (F16, 40, 200, 7, 16, 64, 8, True),       # two
    (F16, 25, 600, 5, 256, 128, 64, False),   # four
    (BF16, 38, 520, 3, 64, 128, 24, True),    # two, of two items a thread
    (BF16, 30, 100, 7, 32, 128, 0, False),    # two
])
def test_appends_of_many_heads(gpu, dtype, sequences, rows, kv_heads, page, dim, pairs, interleaved):
    """Heads that share a workgroup get the bits that they get alone, on new pages and on pages that held tokens."""
    g = torch.Generator().manual_seed(rows)
    first = [(31 * i) % rows for i in range(sequences)]
    second = [rows if i == 3 else (17 * i + 5) % (rows + 1) for i in range(sequences)]
    lengths = [a + b for a, b in zip(first, second)]
    cache, table = make(gpu, lengths, kv_heads, page, dim, seed=rows)
    alone = [layer.KVCache(*(t[:, h:h + 1].contiguous() for t in cache)) for h in range(kv_heads)]
    table, f = table.to(gpu), None
    if pairs:
        f, _ = layer.rotary_frequencies(pairs, device=gpu)
    for step, (n, to) in enumerate(((first, first), (second, lengths))):
        k, v = ((torch.randn((sum(n), kv_heads, dim), generator=g) * (1 + step)).to(dtype).to(gpu) for _ in "kv")
        kw = dict(starts=i32(starts_of(n), gpu), max_rows=rows, frequencies=f, interleaved=interleaved)
        layer.cache_append(k, v, cache, table, i32(to, gpu), **kw)
        for h, one in enumerate(alone):
            layer.cache_append(k[:, h:h + 1], v[:, h:h + 1], one, table, i32(to, gpu), **kw)
            for all_heads, t in zip(cache, one):
                assert torch.equal(all_heads[:, h:h + 1], t)


def test_odd_rotary_widths(gpu):
    """Items with fewer than eight pairs or copied channels, in place and into wider rows, every shape of the ends."""
    g = torch.Generator().manual_seed(0)
    for dim in (2, 7, 18, 31, 64, 100):
        for pairs in sorted({1, dim // 4, dim // 2} - {0}):
            for interleaved in (False, True):
                x = torch.randn((13, 3, dim), generator=g).to(BF16)
                wide = torch.full((13, 3, dim + 5), 9.0, dtype=BF16, device=gpu)
                wide[..., 2:2 + dim] = x.to(gpu)
                f, _ = layer.rotary_frequencies(pairs)
                positions = torch.arange(13)
                want = layer.rotary(x.to(gpu), positions.to(gpu), f.to(gpu), interleaved=interleaved)
                exact = turn64(x, positions, f, interleaved, 1.0)
                # as of any rotation: a few steps of fp32 of the pair (at most 8 here), and the output's rounding
                assert bool(((want.cpu().double() - exact).abs() <= half_step(BF16) * exact.abs() + 8 * 2.0 ** -20).all())
                view = wide[..., 2:2 + dim]
                layer.rotary(view, positions.to(gpu), f.to(gpu), interleaved=interleaved, out=view)
                assert torch.equal(view, want)
                assert bool((wide[..., :2] == 9).all()) and bool((wide[..., 2 + dim:] == 9).all())


# -- sequences that are taken back -------------------------------------------------

def test_drafts_taken_back(gpu):
    """Tokens behind a shorter length are gone: what is written over them is what counts, and their scale stays."""
    page, dim = 16, 64
    cache, table = make(gpu, [60], 2, page, dim, seed=3)
    want = [t.cpu().clone() for t in cache]
    g = torch.Generator().manual_seed(4)
    for length, rows in ((20, 20), (25, 5), (22, 2), (27, 6), (16, 1), (40, 24)):
        k, v = (torch.randn((rows, 2, dim), generator=g).to(F16) for _ in "kv")
        layer.cache_append(k.to(gpu), v.to(gpu), cache, table.to(gpu), i32([length], gpu))
        append_steps(want, k, v, table, [length], [0, rows])
        same_cache(cache, want)
        q = queries(rows, 4, dim, F16, gpu, seed=length)
        compare(run(q, cache, table, [length], [0, rows], gpu), *attend64(q, cache, table, [length], [0, rows], 0.125, True, 0))


def test_shared_pages(gpu):
    """Sequences that share the pages of a common beginning read the same tokens."""
    cache, table = make(gpu, [100, 100, 100], 2, 16, 128, seed=5)
    table[1:, :4] = table[0, :4]
    q = queries(3, 8, 128, BF16, gpu, seed=5)
    compare(run(q, cache, table, [100, 70, 64], [0, 1, 2, 3], gpu),
            *attend64(q, cache, table, [100, 70, 64], [0, 1, 2, 3], 128 ** -0.5, True, 0))


# -- streams and graphs -------------------------------------------------------------

class Step:
    """A layer's attention with everything around it: norm, projection, rotation, append, attention, projection, norm,
    experts, norm. The cache is the step's own."""

    def __init__(self, gpu, rows, lengths, seed, heads=16, kv_heads=4, dim=64, page=16, window=0):
        g = torch.Generator().manual_seed(seed)
        rand = lambda *s, sigma=1.0, mean=0.0: (torch.randn(s, generator=g) * sigma + mean).to(BF16).to(gpu)  # noqa: E731
        self.rows, self.heads, self.kv_heads, self.dim, self.window = rows, heads, kv_heads, dim, window
        width, total = wl.GRANITE.hidden, sum(rows)
        self.cache, table = make(gpu, lengths, kv_heads, page, dim, seed)
        self.table, self.lengths, self.starts = table.to(gpu), i32(lengths, gpu), i32(starts_of(rows), gpu)
        self.positions = torch.cat([torch.arange(n - r, n) for r, n in zip(rows, lengths)]).to(gpu)
        self.h, self.y = rand(total, width, sigma=2.0), rand(total, width)
        self.w1, self.w2, self.w3 = (rand(width, sigma=0.1, mean=1.0) for _ in range(3))
        self.qkv, self.qkv_s = layer.quantize_rows(rand((heads + 2 * kv_heads) * dim, width, sigma=width ** -0.5))
        self.o, self.o_s = layer.quantize_rows(rand(width, heads * dim, sigma=(heads * dim) ** -0.5))
        self.f, _ = layer.rotary_frequencies(dim // 2, device=gpu)

    def attend(self):
        """-> (h, q, k, v, attention's output)"""
        h, codes, scales = layer.norm_residual(self.y, self.h, residual_multiplier=0.22, pre_weight=self.w1, eps=1e-5, quantize=True)
        fused = layer.int8_qmm(codes, scales, self.qkv, self.qkv_s, dtype=BF16)
        n, m = self.heads * self.dim, self.kv_heads * self.dim
        q, k, v = (t.unflatten(1, (-1, self.dim)) for t in fused.split([n, m, m], 1))
        most = max(self.rows)
        turned = layer.rotary(q, self.positions, self.f)
        layer.cache_append(k, v, self.cache, self.table, self.lengths, starts=self.starts, max_rows=most, frequencies=self.f)
        out = layer.cache_attention(turned, self.cache, self.table, self.lengths, starts=self.starts, max_rows=most, window=self.window)
        return h, q, k, v, out

    def __call__(self, blk=None, experts=None):
        h, _, _, _, out = self.attend()
        mid = layer.int8_linear(out.flatten(1), self.o, self.o_s)
        h = layer.norm_residual(mid, h, residual_multiplier=0.22)
        if blk is None:
            return h, out, *(t.clone() for t in self.cache)
        return blk.forward_norms(h, experts, self.w2, 1e-5, next_weight=self.w3)

    def fresh(self):
        return [t.clone() for t in self.cache]

    def reset(self, kept):
        for t, k in zip(self.cache, kept):
            t.copy_(k)


def same(got, want):
    return all(torch.equal(a, b) for a, b in zip(got, want))


BATCHES = [([1, 1, 1], [1, 40, 333]), ([5, 1, 40], [70, 16, 40]), ([129, 700], [500, 1700])]


@pytest.mark.parametrize("rows,lengths", BATCHES)
def test_a_whole_layer(gpu, rows, lengths):
    s = Step(gpu, rows, lengths, seed=sum(rows))
    before = [t.cpu().clone() for t in s.cache]
    kept = s.fresh()
    h, q, k, v, out = s.attend()
    # Each stage against its definition on the stage's own inputs.
    starts = starts_of(rows)
    exact = turn64(q.cpu(), s.positions.cpu(), s.f.cpu(), False, 1.0)
    turned = layer.rotary(q, s.positions, s.f)
    limit = half_step(BF16) * exact.abs() + 2.0 ** -18 * float(q.abs().max())
    assert bool(((turned.cpu().double() - exact).abs() <= limit).all())
    append_steps(before, turn64(k.cpu(), s.positions.cpu(), s.f.cpu(), False, 1.0).float(), v.cpu(), s.table.cpu(), lengths, starts)
    assert torch.equal(s.cache.v.cpu(), before[1]) and torch.equal(s.cache.v_scales.cpu(), before[3])
    assert int((s.cache.k.cpu().int() - before[0].int()).abs().max()) <= 1
    compare(out, *attend64(turned, s.cache, s.table.cpu(), lengths, starts, s.dim ** -0.5, True, 0))
    # And behind it: the same layer with this output in 64 bits. An 8-bit row's element is off by at most half
    # a step, a / 254, evenly spread: its deviation is 1 / sqrt(3) of that, a product's that times the weights' norm. Six of
    # them over a million elements: one in a thousand such tests.
    mid = layer.int8_linear(out.flatten(1), s.o, s.o_s)
    x, w = out.flatten(1).double(), s.o.double() * s.o_s.double()[:, None]
    spread = x.abs().amax(1, keepdim=True) / 254 / math.sqrt(3) * w.pow(2).sum(1).sqrt()
    want = x @ w.t()
    assert bool(((mid.double() - want).abs() <= 6 * 1.01 * spread + half_step(BF16) * want.abs()).all())
    s.reset(kept)
    geom = wl.GRANITE
    experts = tmoe.ExpertWeights.from_layer(wl.make_layer(geom, 0, gpu, seed_tag="attention"))
    blk = tmoe.MoEBlock(geom.hidden, geom.intermediate, geom.experts, geom.top_k, route=geom.route, residual_multiplier=0.22)
    first = s(blk, experts)
    s.reset(kept)
    assert same(s(blk, experts), first) and all(bool(torch.isfinite(t).all()) for t in first)


@pytest.mark.parametrize("rows,lengths", BATCHES)
def test_captured_and_replayed(gpu, rows, lengths):
    """A captured step gives the eager bits on every replay: other inputs, other lengths, other pages, eager work between."""
    a, b = Step(gpu, rows, lengths, seed=1), Step(gpu, rows, [n + 37 for n in lengths], seed=2)
    room = max(a.table.shape[1], b.table.shape[1])
    for s in (a, b):
        s.table = torch.nn.functional.pad(s.table, (0, room - s.table.shape[1]), value=-1)
    live = Step(gpu, rows, lengths, seed=1)
    pages = max(a.cache.k.shape[0], b.cache.k.shape[0])
    live.cache = layer.KVCache(*(t.new_zeros((pages,) + t.shape[1:]) for t in a.cache))
    live.table = a.table.clone()

    def load(s):
        for name in ("table", "lengths", "starts", "positions", "h", "y", "w1", "qkv", "qkv_s", "o", "o_s"):
            getattr(live, name).copy_(getattr(s, name))
        for t, k in zip(live.cache, kept[s]):
            t.zero_()[:k.shape[0]].copy_(k)

    kept = {s: s.fresh() for s in (a, b)}
    want = {}
    for s in (a, b):
        want[s] = s()
        s.reset(kept[s])
    load(a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        live()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two of the same step, in one pool's memory: their workspaces may share it
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0][0].pool() if graphs else None):
            out = live()
        graphs.append((graph, out))
    for i, s in enumerate((a, b, b, a, b, a)):
        load(s)
        graph, out = graphs[i % 2]
        graph.replay()
        eager = (a, b)[i % 2]()  # eager work beside it
        torch.cuda.synchronize()
        for got, w in zip(out, want[s]):
            assert torch.equal(got[:w.shape[0]], w)
        (a, b)[i % 2].reset(kept[(a, b)[i % 2]])
        del eager


@pytest.mark.parametrize("rows,lengths", BATCHES)
def test_two_streams_at_once(gpu, rows, lengths):
    """Steps on two streams share nothing: each gives its own bits."""
    states = [Step(gpu, rows, lengths, seed=i) for i in (1, 2)]
    kept = [s.fresh() for s in states]
    want = []
    for s, k in zip(states, kept):
        want.append(s())
        s.reset(k)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in states], [[], []]
    for _ in range(5):
        for i, (s, st) in enumerate(zip(states, streams)):
            with torch.cuda.stream(st):
                got[i].append(s())
                s.reset(kept[i])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(same(g, want[i]) for g in got[i])


def test_threads_at_once(gpu):
    """Calls from several threads, each on its stream."""
    import threading

    states = [Step(gpu, *BATCHES[i % 3], seed=i) for i in range(4)]
    kept = [s.fresh() for s in states]
    want = []
    for s, k in zip(states, kept):
        want.append(s())
        s.reset(k)
    torch.cuda.synchronize()
    good, streams = [], [torch.cuda.Stream() for _ in states]

    def work(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(5):
                out = states[i]()
                states[i].reset(kept[i])
                streams[i].synchronize()
                good.append(same(out, want[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert len(good) == 20 and all(good)
