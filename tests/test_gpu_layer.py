"""The operators around the block on the GPU, each against a plain implementation in 64 bits.

Tolerances. U is half a step of the storage type relative to the value (bf16
2^-8, f16 2^-11, fp32 2^-24) and TINY half its smallest step (subnormals). In
front of the one rounding stands fp32 arithmetic: a norm's sum of at most 32
sequential terms a lane, a tree of 6 and up to 16 waves, each term rounded
once more, is within 64 * 2^-24 = 2^-18 of its value (all terms are positive),
its inverse root within 2^-19, and a handful of products follow: 2^-18
relative to the magnitudes that are added bounds the fp32 part throughout."""
import math

import numpy as np
import pytest
import torch

from trifuse_amd import layer
from trifuse_amd import moe as tmoe
from trifuse_amd import workload as wl

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}
F = 2.0 ** -18
EPS = 1e-5
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def rand(shape, seed, sigma=1.0, dtype=BF16, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * sigma + mean).to(dtype).cuda()


def close(got, ref, fp32, dtype):
    """|got - ref| within one rounding of ref and `fp32`, the bound on the arithmetic before it."""
    got, ref = got.double(), ref.double()
    tol = (ref.abs() + fp32) * U[dtype] + fp32 + TINY[dtype]
    bad = (got - ref).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} off, worst {((got - ref).abs() / tol).max():.3f} of the tolerance"


# -- norm_residual -------------------------------------------------------------

def norm64(x, w, eps=EPS):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w


def step64(y, r, post, gate, m, pre, eps=EPS, post_eps=EPS):
    """(h, bound on h's fp32 error, x, bound on x's)."""
    b = y.double()
    if post is not None:
        b = norm64(b, post.double(), post_eps)
    if gate is not None:
        g = gate.double()
        b = b * (g.reshape(*y.shape[:-1], 1) if gate.dtype == F32 else g)
    h = m * b if r is None else r.double() + m * b
    eh = F * (m * b).abs() + (F * r.double().abs() if r is not None else 0)
    if pre is None:
        return h, eh, None, None
    inv = torch.rsqrt((h * h).mean(-1, keepdim=True) + eps)
    # x's own arithmetic, h's error through the product, and through the row's inverse root.
    through = (eh * h.abs()).mean(-1, keepdim=True) * inv * inv
    x = h * inv * pre.double()
    return h, eh, x, F * x.abs() + eh * inv * pre.double().abs() + through * x.abs()


@pytest.mark.parametrize("width", [1, 5, 8, 63, 512, 513, 1000, 1024, 1536, 2048, 2050, 4096, 5003, 8192, 8200, 32768])
@pytest.mark.parametrize("rows,dtype,post,gate", [(1, BF16, True, "channel"), (5, F16, False, "token"),
                                                  (67, BF16, True, "full"), (6, F16, True, "none")])
def test_norm_residual(gpu, width, rows, dtype, post, gate):
    y, r = rand((rows, width), 1, 0.7, dtype), rand((rows, width), 2, 2.0, dtype)
    pw = rand((width,), 3, 0.1, dtype, 1.0) if post else None
    w = rand((width,), 4, 0.1, dtype, 1.0)
    g = {"none": lambda: None, "channel": lambda: rand((width,), 5, 0.3, dtype, 0.5),
         "token": lambda: rand((rows,), 6, 0.3, F32, 0.5), "full": lambda: rand((rows, width), 7, 0.3, dtype, 0.5)}[gate]()
    h64, eh, x64, ex = step64(y, r, pw, g, 0.22, w, post_eps=1e-3)
    h, x = layer.norm_residual(y, r, post_weight=pw, gate=g, residual_multiplier=0.22, pre_weight=w, eps=EPS,
                               post_eps=1e-3)
    close(h, h64, eh, dtype)
    close(x, x64, ex, dtype)
    # Each output alone, the codes, and h written over y and over residual give the same bits.
    kw = dict(post_weight=pw, gate=g, residual_multiplier=0.22, eps=EPS, post_eps=1e-3)
    assert torch.equal(layer.norm_residual(y, r, **kw), h)
    h2, codes, scales = layer.norm_residual(y, r, pre_weight=w, quantize=True, **kw)
    assert torch.equal(h2, h)
    largest = x64.abs().amax(-1, keepdim=True)
    elargest = ex.amax(-1, keepdim=True)
    assert ((scales.double()[:, None] * 127 - largest).abs() <= elargest + largest * 2.0 ** -23).all()
    step = scales.double()[:, None]
    assert ((codes.double() * step - x64).abs() <= step * (0.5 + 2.0 ** -15) + ex + elargest).all()
    for into in (y.clone(), r.clone()):
        src = (into, r) if torch.equal(into, y) else (y, into)
        h3, x3 = layer.norm_residual(*src, pre_weight=w, out=into, **kw)
        assert h3.data_ptr() == into.data_ptr() and torch.equal(h3, h) and torch.equal(x3, x)


def test_norm_residual_without_residual_and_rms_norm(gpu):
    y, w = rand((3, 2, 640), 1, 3.0), rand((640,), 2, 0.1, mean=1.0)
    h64, eh, x64, ex = step64(y, None, w, None, -1.5, w)
    h, x = layer.norm_residual(y, post_weight=w, residual_multiplier=-1.5, pre_weight=w, eps=EPS)
    assert h.shape == x.shape == y.shape
    close(h, h64, eh, BF16)
    close(x, x64, ex, BF16)
    plain = norm64(y.double(), w.double())
    x = layer.rms_norm(y, w, EPS)
    close(x, plain, F * plain.abs(), BF16)
    codes, scales = layer.rms_norm(y, w, EPS, quantize=True)
    assert codes.shape == y.shape and scales.shape == y.shape[:-1] and codes.abs().max() == 127
    gate = rand((3, 2, 1), 3, 1.0, F32)
    assert torch.equal(layer.norm_residual(y, gate=gate), layer.norm_residual(y, gate=gate.reshape(3, 2)))


def test_norm_residual_of_zeros_infinities_and_nan(gpu):
    width = 512
    y = rand((5, width), 1)
    y[0], y[1, 7], y[2, 9], y[3] = 0, math.inf, math.nan, 3.3e38
    w = torch.ones(width, dtype=BF16, device="cuda")
    x = layer.rms_norm(y, w, 0.0 + 1e-30)
    assert (x[0] == 0).all() and x[1, 7].isnan() and (x[1, :7] == 0).all() and x[2].isnan().all()
    assert (x[3] == 0).all()  # the sum of squares is past fp32: inverse root 0, as the formula in fp32 gives
    assert torch.isfinite(x[4]).all()
    codes, scales = layer.rms_norm(y, w, 1e-30, quantize=True)
    assert scales[1].isnan() and scales[2].isnan() and (codes[:4] == 0).all() and scales[0] > 0
    assert codes[4].abs().max() == 127


def test_unaligned_views(gpu):
    """Rows that start at any element give the same bits as aligned ones."""
    for width in (512, 515):
        flat = rand((3 * width + 1,), 1)
        y, w = flat[1:].view(3, width), rand((width + 3,), 2, 0.1, mean=1.0)[3:]
        h, x = layer.norm_residual(y, post_weight=w, pre_weight=w)
        h2, x2 = layer.norm_residual(y.clone(), post_weight=w.clone(), pre_weight=w.clone())
        assert torch.equal(h, h2) and torch.equal(x, x2)
        a, b = layer.quantize_rows(y), layer.quantize_rows(y.clone())
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_norm_residual_leaves_what_is_not_its_own(gpu):
    buf = torch.full((7, 520), 9.0, dtype=BF16, device="cuda")
    y = rand((3, 520), 1)
    layer.norm_residual(y, out=buf[2:5])
    assert (buf[:2] == 9).all() and (buf[5:] == 9).all() and torch.equal(buf[2:5], y)
    from trifuse_amd._lib import TfmError
    with pytest.raises(TfmError, match="overlaps"):
        layer.norm_residual(buf[1:4], out=buf[2:5])
    empty = layer.norm_residual(y[:0], y[:0], pre_weight=y[0])
    assert empty[0].shape == empty[1].shape == (0, 520)


# -- codes ---------------------------------------------------------------------

@pytest.mark.parametrize("width", [1, 7, 16, 512, 1025, 2048, 4096, 9000, 40000, 131072])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_quantize_rows_is_its_formula_in_fp32(gpu, width, dtype):
    x = rand((9, width), width, 2.0, dtype)
    x[1] = 0
    x[2] *= 1e-4
    x[3, width // 2], x[4, width - 1] = math.inf, math.nan
    x[5, 0] = -100.0
    if dtype == BF16:
        x[6] = x[6] * 1e-36  # 127 / max|x| would overflow
        x[7] = x[7] * 1e37
    codes, scales = layer.quantize_rows(x)
    v = x.float().cpu().numpy()
    amax = np.abs(v).max(1)
    a = np.maximum(np.where(np.isfinite(amax), amax, np.float32(1)), np.float32(2.0 ** -100)).astype(np.float32)
    good = np.isfinite(v).all(1)
    ref = np.rint(np.where(good[:, None], v, 0) * (np.float32(127) / a)[:, None]).astype(np.int8)
    assert np.array_equal(codes.cpu().numpy(), ref)
    s = scales.cpu().numpy()
    assert np.array_equal(np.isnan(s), ~good) and np.array_equal(s[good], (a / np.float32(127))[good])


# -- products --------------------------------------------------------------------

def product64(codes, scales, w, ws, bias):
    acc = (codes.cpu().double() @ w.cpu().double().t()).cuda()  # exact: below 2^53
    v = acc * scales.double()[:, None] * ws.double()
    # conversion, two scales and the bias, each rounded once
    bound = v.abs() * 2.0 ** -22
    return (v, bound) if bias is None else (v + bias.double(), bound + (v.abs() + bias.double().abs()) * 2.0 ** -24)


def codes_of(shape, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-127, 128, shape, generator=g, dtype=torch.int8).cuda()


def scales_of(n, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.rand(n, generator=g) * 0.02 + 0.001).cuda()


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 32, 33, 63, 64, 65, 128, 129, 257, 515])
@pytest.mark.parametrize("n,k", [(1, 16), (63, 48), (64, 64), (65, 128), (130, 144), (257, 1040), (515, 2048), (96, 4112)])
def test_int8_qmm(gpu, rows, n, k):
    dtype = [BF16, F16, F32][(rows + n) % 3]
    codes, w, scales, ws = codes_of((rows, k), 1), codes_of((n, k), 2), scales_of(rows, 3), scales_of(n, 4)
    bias = rand((n,), 5, 1.0, dtype) if (rows + k) % 2 else None
    out = layer.int8_qmm(codes, scales, w, ws, bias=bias, dtype=dtype)
    assert out.shape == (rows, n) and out.dtype == dtype
    close(out, *product64(codes, scales, w, ws, bias), dtype)


@pytest.mark.parametrize("rows,n,k", [(700, 1537, 512), (1024, 2048, 2048), (2049, 3000, 192), (4096, 520, 1040),
                                      (3, 50304, 1536), (40, 20000, 2064)])
def test_int8_qmm_large(gpu, rows, n, k):
    codes, w, scales, ws = codes_of((rows, k), 1), codes_of((n, k), 2), scales_of(rows, 3), scales_of(n, 4)
    out = layer.int8_qmm(codes, scales, w, ws, dtype=F32)
    close(out, *product64(codes, scales, w, ws, None), F32)


@pytest.mark.parametrize("rows,n", [(2047, 8190), (2041, 6143), (2040, 2552), (1023, 2050)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_int8_qmm_every_tile_and_type(gpu, rows, n, dtype):
    """Sizes that take the 256 x 256, 256 x 192 (fp32: another), 128 x 128 and 64 x 64 tiles, with ragged last ones."""
    k = 272
    codes, w, scales, ws, bias = codes_of((rows, k), 1), codes_of((n, k), 2), scales_of(rows, 3), scales_of(n, 4), rand((n,), 5, 1.0, dtype)
    out = layer.int8_qmm(codes, scales, w, ws, bias=bias, dtype=dtype)
    close(out, *product64(codes, scales, w, ws, bias), dtype)


@pytest.mark.parametrize("rows", [1, 20, 70, 300])
def test_int8_qmm_longest_sum(gpu, rows):
    """Every product at its largest: the sum stays below 2^31 at the longest k."""
    k = 131056
    codes = torch.full((rows, k), -128, dtype=torch.int8, device="cuda")
    w = torch.full((3, k), -128, dtype=torch.int8, device="cuda")
    w[1] = 127
    one, ones = torch.ones(rows, device="cuda"), torch.ones(3, device="cuda")
    out = layer.int8_qmm(codes, one, w, ones, dtype=F32).double()
    ref = torch.tensor([16384.0 * k, -16256.0 * k, 16384.0 * k], dtype=torch.float64, device="cuda")
    assert ((out - ref).abs() <= ref.abs() * 2.0 ** -24).all()


@pytest.mark.parametrize("rows", [1, 7, 33, 200])
def test_int8_qmm_scales_bias_and_neighbours(gpu, rows):
    """NaN scales stay in their row and column; nothing outside the output is written; bit-equal repeats."""
    k, n = 272, 70
    codes, w, scales, ws = codes_of((rows, k), 1), codes_of((n, k), 2), scales_of(rows, 3), scales_of(n, 4)
    clean = layer.int8_qmm(codes, scales, w, ws)
    assert torch.equal(clean, layer.int8_qmm(codes, scales, w, ws))
    bad_s, bad_w = scales.clone(), ws.clone()
    bad_s[rows // 2], bad_w[11] = math.nan, math.inf
    out = layer.int8_qmm(codes, bad_s, w, bad_w)
    keep = torch.ones_like(out, dtype=torch.bool)
    keep[rows // 2], keep[:, 11] = False, False
    assert torch.equal(out[keep], clean[keep]) and out[rows // 2].isnan().all()
    from trifuse_amd import _lib
    buf = torch.full((rows * n + 200,), 5.0, dtype=BF16, device="cuda")
    _lib.call("tfm_int8_qmm", codes.data_ptr(), scales.data_ptr(), rows, w.data_ptr(), ws.data_ptr(), None, n, k, 0,
              buf[100:].data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert (buf[:100] == 5).all() and (buf[100 + rows * n:] == 5).all()
    assert torch.equal(buf[100:100 + rows * n].view(rows, n), clean)


@pytest.mark.parametrize("rows,k,n,dtype", [(1, 2048, 2048, BF16), (1, 16, 1, F16), (3, 1536, 515, F16), (8, 4096, 640, BF16),
                                            (16, 2048, 1000, BF16), (17, 512, 96, F16), (64, 1040, 130, BF16),
                                            (130, 272, 70, F16), (515, 2048, 300, BF16), (5, 272, 8200, F16),
                                            (6, 2048, 33000, BF16), (3, 528, 32771, F16)])
def test_int8_linear_is_quantize_then_product(gpu, rows, k, n, dtype):
    x, w, ws, bias = rand((rows, k), 1, 1.0, dtype), codes_of((n, k), 2), scales_of(n, 4), rand((n,), 5, 1.0, dtype)
    codes, scales = layer.quantize_rows(x)
    assert torch.equal(layer.int8_linear(x, w, ws, bias=bias), layer.int8_qmm(codes, scales, w, ws, bias=bias, dtype=dtype))
    assert torch.equal(layer.int8_linear(x, w, ws), layer.int8_qmm(codes, scales, w, ws, dtype=dtype))
    x[rows - 1, k - 1] = math.nan
    out = layer.int8_linear(x, w, ws)
    assert out[rows - 1].isnan().all() and torch.isfinite(out[:rows - 1]).all()
    assert layer.int8_linear(x[:0], w, ws).shape == (0, n)


# -- log probabilities -------------------------------------------------------------

def logprobs64(logits, tokens, top, scale):
    """In 64 bits: (logprobs, entropy, ids, top_logprobs), ids by value descending, ties to the lower id, NaN last."""
    raw = logits.double().cpu()
    # Differences first and the maximum's own term apart: z - logsumexp(z) would itself be off by 2^-52 |z|,
    # more than a nearly sure token's log probability is held to.
    d = (raw - raw.max(-1, keepdim=True).values) * scale
    others = d.exp().scatter(-1, d.argmax(-1, keepdim=True), 0.0)
    lp = d - torch.log1p(others.sum(-1, keepdim=True))
    p = lp.exp()
    entropy = -torch.special.xlogy(p, p).sum(-1)
    order = torch.where(raw.isnan(), torch.full_like(raw, -math.inf), raw)
    # -inf above NaN: a stable sort by (is NaN, value)
    ids = torch.stack([torch.from_numpy(np.lexsort((np.arange(raw.shape[-1]), -o, n)))
                       for o, n in zip(order.numpy(), raw.isnan().numpy())])[:, :top]
    logp = None if tokens is None else lp.gather(1, tokens.cpu().long()[:, None])[:, 0]
    return logp, entropy, ids, lp.gather(1, ids)


def check_logprobs(logits, tokens, top, scale=1.0):
    """S is a sum of up to V terms: a thread's sequential sum (each of at most V / 256 / 8 vectors of 8), the tree
    and the waves, at most V / 256 + 32 roundings; the exponent's argument (differences times scale, |argument| up
    to 150 before the term vanishes) adds 2^-24 of itself twice and exp2 two units. Relative to S that is
    (V / 256 + 340) * 2^-24, absolute in ln S; scale * (l - M) and the last sum add 2^-23 of their own size.
    R = S - 1 has the same relative bound, so ln S near 0 keeps it relative: ln S <= R."""
    V = logits.shape[-1]
    logp, entropy, ids, best = layer.token_logprobs(logits, tokens, top=top, scale=scale)
    rp, re, rids, rbest = logprobs64(logits, tokens, top, scale)
    rel = (V / 256 + 340) * 2.0 ** -24

    def near(got, ref, extra=0.0):
        got, ref = got.double().cpu(), ref
        assert torch.equal(got.isnan(), ref.isnan())
        same = got == ref  # infinities
        off = (got - ref).abs()
        ok = same | ref.isnan() | (off <= torch.minimum(ref.abs(), torch.ones_like(ref)) * rel * 2
                                   + ref.abs() * 2.0 ** -22 + extra)
        assert ok.all(), f"worst {off[~ok].max()}"

    assert torch.equal(ids.cpu().long(), rids)
    near(best, rbest)
    if tokens is not None:
        near(logp, rp)
    # entropy = sum p (-ln p): each term within rel + 2^-22 (1 + |ln p|) of itself
    near(entropy, re, extra=re.abs() * rel * 2 + rel * 2 * torch.minimum(re, torch.ones_like(re)))


@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 63, 64, 65, 511, 513, 2048, 2055, 8191, 8192, 10007, 50304, 131071])
@pytest.mark.parametrize("dtype,scale", [(BF16, 1.0), (F16, 1.3), (F32, 0.25)])
def test_token_logprobs(gpu, vocab, dtype, scale):
    rows = 3
    logits = rand((rows, vocab), vocab, 2.5, dtype)
    logits[1, vocab // 3] += 20  # nearly sure: ln S far below 1
    tokens = torch.tensor([0, vocab // 3, vocab - 1], device="cuda")
    for top in sorted({0, 1, min(vocab, 5), min(vocab, 20), min(vocab, 64)}):
        check_logprobs(logits, tokens, top, scale)


@pytest.mark.parametrize("rows", [1, 2, 17, 600, 1025])
def test_token_logprobs_rows(gpu, rows):
    for vocab in (1000, 9001):
        logits = rand((rows, vocab), rows, 2.5)
        tokens = torch.arange(rows, device="cuda", dtype=torch.int32) * 7 % vocab
        check_logprobs(logits, tokens, 5)


@pytest.mark.parametrize("vocab", [40, 700, 9000, 33000])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_token_logprobs_ties_and_masks(gpu, vocab, dtype):
    g = torch.Generator().manual_seed(vocab)
    rows = [torch.zeros(vocab),                                              # one value everywhere
            torch.randint(0, 3, (vocab,), generator=g).float(),              # many ties
            torch.where(torch.rand(vocab, generator=g) < 0.9, -math.inf, torch.randn(vocab, generator=g)),
            torch.cat([torch.full((vocab - 1,), -math.inf), torch.tensor([2.0])]),  # one token left
            torch.full((vocab,), torch.finfo(dtype).min),                   # the type's lowest value as the mask
            torch.where(torch.arange(vocab) % 3 == 0, torch.finfo(dtype).min, 1.0),
            torch.cat([-torch.zeros(vocab // 2), torch.zeros(vocab - vocab // 2)]),  # -0 ties with 0
            torch.arange(vocab).float() * -0.001,                            # sorted, falling
            torch.arange(vocab).float() * 0.001]
    logits = torch.stack(rows).to(dtype).cuda()
    tokens = torch.randint(0, vocab, (len(rows),), generator=g).cuda()
    for top in (1, 6, min(vocab, 64)):
        check_logprobs(logits, tokens, top)


def test_token_logprobs_of_empty_infinite_and_nan_rows(gpu):
    for vocab in (10, 3000, 20000):
        logits = rand((5, vocab), 1, 1.0, F32)
        logits[0] = -math.inf
        logits[1, 3] = math.inf
        logits[2, 5] = math.nan
        logits[3] = math.nan
        tokens = torch.tensor([1, 2, 3, 4, 5], device="cuda")
        logp, entropy, ids, best = layer.token_logprobs(logits, tokens, top=4)
        assert logp[0] == -math.inf and entropy[0] == 0 and (best[0] == -math.inf).all()
        assert ids[0].tolist() == [0, 1, 2, 3]
        assert logp[1:4].isnan().all() and entropy[1:4].isnan().all() and best[1:4].isnan().all()
        assert ids[1, 0] == 3 and ids[3].tolist() == [0, 1, 2, 3]
        row = logits[2].clone()
        row[5] = -math.inf
        assert ids[2].tolist() == torch.sort(row, descending=True, stable=True).indices[:4].tolist()
        assert torch.isfinite(logp[4]) and torch.isfinite(entropy[4]) and torch.isfinite(best[4]).all()
        nan = torch.full((1, vocab), math.nan, device="cuda")
        nan[0, vocab - 2] = -math.inf  # above NaN
        assert layer.token_logprobs(nan, top=3)[2][0].tolist() == [vocab - 2, 0, 1]


def test_token_logprobs_with_most_logits_in_few_threads(gpu):
    """The largest logits all in vectors that one thread reads: more candidates than the list holds."""
    for rows, vocab in ((2, 262144), (1024, 131072)):
        for threads in (256, 512):
            logits = torch.zeros((rows, vocab), dtype=BF16, device="cuda")
            vec = torch.arange(vocab, device="cuda") // 8 % threads
            few = vec < 12
            g = torch.Generator(device="cuda").manual_seed(3)
            logits[:, few] = (torch.rand((rows, int(few.sum())), generator=g, device="cuda") + 8).to(BF16)
            logits = logits[:2] if rows == 2 else logits
            _, _, ids, best = layer.token_logprobs(logits, top=40)
            some = logits[:2]
            _, _, rids, rbest = logprobs64(some, None, 40, 1.0)
            assert torch.equal(ids[:2].cpu().long(), rids)
            assert (best[:2].double().cpu() - rbest).abs().max() < 1e-5


def test_token_logprobs_views_types_and_bad_tokens(gpu):
    wide = rand((6, 1203), 1, 2.0)
    view = wide[:, :1001]  # a padded vocabulary: rows start at odd elements
    tokens = torch.tensor([0, 5, 1000, 77, 1001, -1], device="cuda")
    logp, entropy, ids, best = layer.token_logprobs(view, tokens, top=3)
    ref = layer.token_logprobs(view.contiguous(), tokens.int(), top=3)
    for a, b in zip((logp, entropy, ids, best), ref):
        assert torch.equal(a, b) or (torch.equal(a.isnan(), b.isnan()) and torch.equal(a[:4], b[:4]))
    assert logp[4:].isnan().all() and torch.isfinite(logp[:4]).all()
    check_logprobs(view[:4], tokens[:4], 3)
    none = layer.token_logprobs(view)
    assert none[0] is None and none[2].shape == (6, 0) and torch.equal(none[1], entropy)
    cube = rand((2, 3, 50), 2)
    out = layer.token_logprobs(cube, torch.zeros((2, 3), dtype=torch.int64, device="cuda"), top=2)
    assert [tuple(t.shape) for t in out] == [(2, 3), (2, 3), (2, 3, 2), (2, 3, 2)]
    empty = layer.token_logprobs(wide[:0], tokens[:0], top=2)
    assert [tuple(t.shape) for t in empty] == [(0,), (0,), (0, 2), (0, 2)]
    with pytest.raises(ValueError, match="contiguous"):
        layer.token_logprobs(wide.t())
    from trifuse_amd._lib import TfmError
    with pytest.raises(TfmError, match="row_stride"):
        layer.token_logprobs(wide[:1].expand(3, 1203))


# -- refusals of the host mirror ---------------------------------------------------

def test_host_mirror_refusals(gpu):
    y, w = rand((4, 64), 1), rand((64,), 2)
    codes, scales = layer.quantize_rows(y)
    cases = [
        lambda: layer.norm_residual(y, y[:3]),
        lambda: layer.norm_residual(y, y.half()),
        lambda: layer.norm_residual(y, post_weight=w[:63]),
        lambda: layer.norm_residual(y, pre_weight=w.half()),
        lambda: layer.norm_residual(y, gate=w.float()),
        lambda: layer.norm_residual(y, gate=y[:2]),
        lambda: layer.norm_residual(y, quantize=True),
        lambda: layer.norm_residual(y, out=y[:2]),
        lambda: layer.norm_residual(y.t()),
        lambda: layer.rms_norm(y, w.cpu(), 1e-5),
        lambda: layer.int8_qmm(y, scales, codes, scales),
        lambda: layer.int8_qmm(codes, scales[:2], codes, scales),
        lambda: layer.int8_qmm(codes, scales, codes[:, :32], scales),
        lambda: layer.int8_qmm(codes, scales, codes, scales.half()),
        lambda: layer.int8_qmm(codes, scales, codes, scales, bias=y[:, 0].contiguous(), dtype=F16),
        lambda: layer.int8_qmm(codes, scales, codes, scales, dtype=torch.float64),
        lambda: layer.int8_linear(y, codes.t(), scales),
        lambda: layer.token_logprobs(y, torch.zeros(4, device="cuda")),
        lambda: layer.token_logprobs(y, torch.zeros(3, dtype=torch.int64, device="cuda")),
        lambda: layer.token_logprobs(y, top=65),
    ]
    for i, f in enumerate(cases):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"case {i} was taken")


# -- together ------------------------------------------------------------------------

def _layer_pass(s, into=None):
    """A layer's dense side: block output -> norms and residual -> projection -> norm -> head -> log probabilities."""
    h, codes, scales = layer.norm_residual(s["y"], s["h"], post_weight=s["w1"], gate=s["gate"], residual_multiplier=0.22,
                                           pre_weight=s["w2"], eps=EPS, quantize=True)
    mid = layer.int8_qmm(codes, scales, s["p"], s["ps"], dtype=BF16)
    h = layer.norm_residual(mid, h, residual_multiplier=0.22)
    codes, scales = layer.rms_norm(h, s["w3"], EPS, quantize=True)
    logits = layer.int8_qmm(codes, scales, s["head"], s["hs"], dtype=F32)
    return (h, logits) + layer.token_logprobs(logits, s["tokens"], top=5, scale=0.5)


def _layer_state(rows, width, vocab, seed=1):
    n = lambda shape, i, sigma=1.0, mean=0.0: rand(shape, seed * 100 + i, sigma, BF16, mean)  # noqa: E731
    s = dict(y=n((rows, width), 1), h=n((rows, width), 2, 2.0), w1=n((width,), 3, 0.1, 1.0), w2=n((width,), 4, 0.1, 1.0),
             w3=n((width,), 5, 0.1, 1.0), gate=n((rows, width), 6, 0.3, 0.5), tokens=torch.arange(rows, device="cuda") * 3)
    s["p"], s["ps"] = layer.quantize_rows(n((width, width), 7, width ** -0.5))
    s["head"], s["hs"] = layer.quantize_rows(n((vocab, width), 8, 3 * width ** -0.5))
    return s


@pytest.mark.parametrize("rows", [1, 5, 70, 300])
def test_together(gpu, rows):
    width, vocab = 512, 3001
    s = _layer_state(rows, width, vocab)
    h, logits, logp, entropy, ids, best = _layer_pass(s)
    d = {k: v.double() for k, v in s.items() if v.is_floating_point()}
    h64 = d["h"] + 0.22 * d["gate"] * norm64(d["y"], d["w1"])
    x = norm64(h64, d["w2"])
    p = s["p"].double() * d["ps"][:, None]
    h64 = h64 + 0.22 * (x @ p.t())
    x = norm64(h64, d["w3"])
    z = x @ (s["head"].double() * d["hs"][:, None]).t()
    # 8-bit codes of x: an element is off by half a step, a / 254, a product of n of them by sqrt(n) / sqrt(3)
    # of that times the weights' size, in the mean; five times that bounds all.
    step = x.abs().amax(1, keepdim=True) / 254
    spread = step / math.sqrt(3) * (s["head"].double() * d["hs"][:, None]).pow(2).sum(1).sqrt()
    # the stream's own error: the projection's codes (the same bound) and two roundings of h
    assert ((h.double() - h64).abs() <= h64.abs() * 2.0 ** -7 + 0.25).all()
    assert ((logits.double() - z).abs() <= 8 * spread + 0.05 * z.abs().amax()).all()
    check_logprobs(logits, s["tokens"], 5, 0.5)
    again = _layer_pass(s)
    assert all(torch.equal(a, b) for a, b in zip((h, logits, logp, entropy, ids, best), again))


@pytest.mark.parametrize("rows", [1, 12, 130])
def test_captured_and_replayed(gpu, rows):
    """A captured pass gives the eager bits on every replay, with new inputs and eager work between."""
    s, other = _layer_state(rows, 512, 3001), _layer_state(rows, 512, 3001, seed=2)
    want = [_layer_pass(dict(s, y=y)) for y in (s["y"], other["y"])]
    y = s["y"].clone()
    live = dict(s, y=y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _layer_pass(live)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _layer_pass(live)
    for i in (0, 1, 0, 1, 1):
        y.copy_((s["y"], other["y"])[i])
        graph.replay()
        eager = _layer_pass(other)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[i]))
        del eager


def test_two_streams_at_once(gpu):
    """Calls on two streams share nothing: each gives its eager bits."""
    states = [_layer_state(33, 512, 3001, seed=i) for i in (1, 2)]
    want = [_layer_pass(s) for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    got = [[], []]
    for _ in range(5):
        for i, (s, st) in enumerate(zip(states, streams)):
            with torch.cuda.stream(st):
                got[i].append(_layer_pass(s))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[i]))


# -- the block between its norms -------------------------------------------------------

@pytest.mark.parametrize("geom_name,T,rm", [("olmoe", 1, 1.0), ("olmoe", 9, 1.0), ("granite", 33, 0.22)])
def test_forward_norms(gpu, geom_name, T, rm):
    geom = wl.OLMOE if geom_name == "olmoe" else wl.GRANITE
    w = tmoe.ExpertWeights.from_layer(wl.make_layer(geom, 0, gpu, seed_tag="norms"))
    blk = tmoe.MoEBlock(geom.hidden, geom.intermediate, geom.experts, geom.top_k, route=geom.route, residual_multiplier=rm)
    unit = tmoe.MoEBlock(geom.hidden, geom.intermediate, geom.experts, geom.top_k, route=geom.route)
    h = (wl.make_x(geom, T, tag="norms") * 3.0).to(gpu)
    n = [rand((geom.hidden,), i, 0.1, BF16, 1.0) for i in (1, 2, 3)]
    gate = rand((T,), 4, 0.3, F32, 0.5)
    out, nxt = blk.forward_norms(h, w, n[0], EPS, post_weight=n[1], gate=gate, next_weight=n[2])
    y = unit.forward(layer.rms_norm(h, n[0], EPS), w)  # the block itself, then the formula in 64 bits
    h64, eh, x64, ex = step64(y, h, n[1], gate, rm, n[2])
    close(out, h64, eh, BF16)
    close(nxt, x64, ex, BF16)
    plain = blk.forward_norms(h, w, n[0], EPS)
    h64, eh, _, _ = step64(y, h, None, None, rm, None)
    close(plain, h64, eh, BF16)
    assert blk.forward_norms(h[:0], w, n[0], EPS).shape == (0, geom.hidden)


# -- sizes past 32 bits ----------------------------------------------------------------

def test_offsets_past_32_bits(gpu):
    """The last rows of calls of more than 2^32 bytes and 2^31 elements equal the same rows alone."""
    rows, width = 70001, 32768
    y = torch.empty((rows, width), dtype=BF16, device="cuda")
    y[:-3] = 1.0
    y[-3:] = rand((3, width), 1)
    w = rand((width,), 2, 0.1, BF16, 1.0)
    h, x = layer.norm_residual(y, y, post_weight=w, gate=y, pre_weight=w, out=y.clone())
    h2, x2 = layer.norm_residual(y[-3:], y[-3:], post_weight=w, gate=y[-3:], pre_weight=w)
    assert torch.equal(h[-3:], h2) and torch.equal(x[-3:], x2)
    del h, x
    codes, scales = layer.quantize_rows(y)
    last = layer.quantize_rows(y[-3:])
    assert torch.equal(codes[-3:], last[0]) and torch.equal(scales[-3:], last[1])
    del codes, scales
    tokens = torch.full((rows,), width - 1, device="cuda")
    got, ref = layer.token_logprobs(y, tokens, top=4), layer.token_logprobs(y[-3:].contiguous(), tokens[-3:], top=4)
    assert torch.equal(got[2][-3:], ref[2])
    for a, b in zip((got[0], got[1], got[3]), (ref[0], ref[1], ref[3])):
        assert ((a[-3:] - b).abs() <= b.abs() * 2.0 ** -20).all()  # another workgroup width: another order of the sum
    del got, y
    for k, n in ((32768, 16), (16, 32784)):  # the left operand, then the output, past 2^31 elements
        codes = torch.ones((rows, k), dtype=torch.int8, device="cuda")
        codes[-3:] = codes_of((3, k), 1)
        one, wq, ws = scales_of(rows, 2), codes_of((n, k), 3), scales_of(n, 4)
        out = layer.int8_qmm(codes, one, wq, ws)
        assert torch.equal(out[-3:], layer.int8_qmm(codes[-3:], one[-3:], wq, ws))
        del codes, out
    w = torch.ones((140003, 16384), dtype=torch.int8, device="cuda")  # the weights past 2^31 bytes
    w[-70:] = codes_of((70, 16384), 5)
    ws = scales_of(140003, 6)
    for m in (2, 40):
        codes, one = codes_of((m, 16384), 7), scales_of(m, 8)
        out = layer.int8_qmm(codes, one, w, ws)
        assert torch.equal(out[:, -70:], layer.int8_qmm(codes, one, w[-70:], ws[-70:].clone()))
