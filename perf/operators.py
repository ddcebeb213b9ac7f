"""The operators around a MoE feed-forward block, as they are measured: norms and residuals, 8-bit products, log probabilities.

A decoder layer runs them between its expert blocks and behind the last one:

* ``norm``: a block's output y is normed (post norm), gated, scaled and added to the residual stream h, and h is normed for
  the next block (pre norm): h = residual + m * gate * norm(y) * w_post, x = norm(h) * w_pre;
* ``project``: the same step with x rounded to 8-bit codes and one scale a token, and the next product on those codes;
* ``linear``: a product in 8-bit integers, y = x . W^T, with a scale for each token of x (made in the call) and for each
  channel of W (made when the weights were stored);
* ``logprobs``: from a step's logits, the log probability of each given token, the entropy and the most likely alternatives.

Widths are those of ``trifuse_amd.workload`` (2048 and 1536, and their projections) or generic; vocabularies are generic, an odd
one among them. Calls are eager, as a serving loop in Python makes them.
"""
import math

import torch

own = False

EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# -- cases -------------------------------------------------------------------

def norm(name, rows, width, dtype="bf16", post=True, gate="none", multiplier=1.0):
    return {"name": name, "kind": "norm", "rows": rows, "width": width, "dtype": dtype, "post": post, "gate": gate,
            "multiplier": multiplier}


def project(name, rows, width, out, dtype="bf16", post=True, gate="none", multiplier=1.0):
    return {**norm(name, rows, width, dtype, post, gate, multiplier), "kind": "project", "out": out}


def linear(name, rows, width, out, dtype="bf16", bias=False):
    return {"name": name, "kind": "linear", "rows": rows, "width": width, "out": out, "dtype": dtype, "bias": bias}


def logprobs(name, rows, vocab, top, dtype="bf16", scale=1.0, masked=False):
    return {"name": name, "kind": "logprobs", "rows": rows, "vocab": vocab, "top": top, "dtype": dtype, "scale": scale,
            "masked": masked}


def listed():
    return [
        # One sequence being decoded, between two blocks: latency.
        norm("norm 1", 1, 2048, gate="channel"),
        # A batch of prompts of odd length, a gate for each token and a scaled residual, half storage.
        norm("norm 613 half", 613, 1536, dtype="f16", gate="token", multiplier=0.22),
        # The tokens of a long prefill, gated element by element: memory.
        norm("norm 16384", 16384, 2048, gate="full"),
        # The same step in front of an attention's fused projections, in 8 bits.
        project("project 4096", 4096, 2048, 6144, multiplier=0.22),
        # One token through a square projection: latency.
        linear("linear 1", 1, 2048, 2048),
        # The output head of a decode batch: its weights are read once.
        linear("head 8", 8, 2048, 50304),
        # A small odd batch on the smaller width, half storage, with a bias.
        linear("linear 37 half", 37, 1536, 2560, dtype="f16", bias=True),
        # A prompt through a square projection.
        linear("linear 1024", 1024, 2048, 2048),
        # Many prompts through a wide feed-forward product.
        linear("linear 8192 wide", 8192, 4096, 12288),
        # One sampled token: latency.
        logprobs("logprobs 1", 1, 50304, 5),
        # A speculative or beam batch, odd vocabulary, half logits, a grammar's mask, temperature.
        logprobs("logprobs 333 half", 333, 49155, 8, dtype="f16", scale=1 / 0.7, masked=True),
        # Scoring of whole prompts.
        logprobs("logprobs 4096", 4096, 50304, 20),
    ]


def _spread(rng, low, high):
    return round(math.exp(rng.uniform(math.log(low), math.log(high))))


def draw(rng):
    kind = rng.choice(["norm", "project", "linear", "linear", "logprobs", "logprobs"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if kind == "logprobs":
        vocab = _spread(rng, 1000, 200000)
        rows = _spread(rng, 1, min(4096, 200_000_000 // vocab))
        if rng.random() < 0.2:
            dtype, rows = "f32", max(1, rows // 2)
        case = logprobs("", rows, vocab, rng.choice([0, 1, 5, 10, 20]), dtype, rng.choice([1.0, 1.0, 1.25, 0.125]),
                        rng.random() < 0.3)
    elif kind == "linear":
        width = rng.choice([512, 1024, 1536, 2048, 4096, 16 * _spread(rng, 4, 256)])
        rows, out = _spread(rng, 1, 8192), _spread(rng, 64, 12288)
        case = linear("", rows, width, out, dtype, rng.random() < 0.3)
    else:
        width = rng.choice([512, 1024, 1536, 2048, 16 * _spread(rng, 4, 256)])
        gate, multiplier = rng.choice(["none", "channel", "token", "full"]), rng.choice([1.0, 0.22])
        if kind == "norm":
            if rng.random() < 0.25:
                width = _spread(rng, 65, 4095)
            case = norm("", _spread(rng, 1, 33_000_000 // width), width, dtype, rng.random() < 0.75, gate, multiplier)
        else:
            case = project("", _spread(rng, 1, 4096), width, _spread(rng, 64, 6144), dtype, rng.random() < 0.75, gate,
                           multiplier)
    del case["name"]
    return case


# -- inputs ------------------------------------------------------------------

class State:
    pass


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, sigma=1.0, mean=0.0, to=dtype):
        return (torch.randn(shape, generator=gen, device="cuda") * sigma + mean).to(to)

    s = State()
    s.kind, s.dtype, rows = case["kind"], dtype, case["rows"]
    if s.kind == "logprobs":
        vocab = case["vocab"]
        s.top, s.scale = case["top"], case["scale"]
        s.logits = normal(rows, vocab, sigma=2.5)
        # Half of the rows are sure of one token, the others are not.
        sure = torch.randint(0, vocab, (rows, 1), generator=gen, device="cuda")
        lift = 14.0 * torch.rand((rows, 1), generator=gen, device="cuda").round()
        s.logits.scatter_add_(1, sure, lift.to(dtype))
        if case["masked"]:
            banned = torch.rand((rows, vocab), generator=gen, device="cuda") < 0.3
            s.logits.masked_fill_(banned, -math.inf)
        other = torch.randint(0, vocab, (rows, 1), generator=gen, device="cuda")
        s.tokens = torch.where(torch.rand((rows, 1), generator=gen, device="cuda") < 0.7, sure, other).reshape(-1)
        return s
    width = case["width"]
    if s.kind in ("norm", "project"):
        # The residual stream of a deep model has a few channels much larger than the others.
        s.residual = normal(rows, width, sigma=2.0)
        s.residual[:, ::257] *= 8
        s.y = normal(rows, width, sigma=0.7)
        s.post = normal(width, sigma=0.1, mean=1.0) if case["post"] else None
        s.pre = normal(width, sigma=0.1, mean=1.0)
        s.gate = {"none": lambda: None, "channel": lambda: normal(width, sigma=0.3, mean=0.5),
                  "token": lambda: torch.rand((rows,), generator=gen, device="cuda"),
                  "full": lambda: normal(rows, width, sigma=0.3, mean=0.5)}[case["gate"]]()
        s.multiplier = case["multiplier"]
    else:
        s.x = normal(rows, width)
        s.x[:, ::129] *= 6
        s.bias = normal(case["out"], sigma=0.5) if case["bias"] else None
    if s.kind != "norm":  # the stored weights: codes in [-127, 127] and a scale for each channel
        w = torch.randn((case["out"], width), generator=gen, device="cuda") * width ** -0.5
        s.w_scales = w.abs().amax(1).clamp_min(1e-20) / 127
        s.w_codes = (w / s.w_scales[:, None]).round().to(torch.int8)
    return s


# -- one pass ----------------------------------------------------------------

def run(s):
    if own:
        from trifuse_amd import layer
        if s.kind == "logprobs":
            logp, entropy, ids, top = layer.token_logprobs(s.logits, s.tokens, top=s.top, scale=s.scale)
            return {"logprobs": logp, "entropy": entropy, "top_ids": ids, "top_logprobs": top}
        if s.kind == "linear":
            return {"out": layer.int8_linear(s.x, s.w_codes, s.w_scales, bias=s.bias)}
        step = dict(post_weight=s.post, gate=s.gate, residual_multiplier=s.multiplier, pre_weight=s.pre, eps=EPS)
        if s.kind == "norm":
            h, x = layer.norm_residual(s.y, s.residual, **step)
            return {"h": h, "x": x}
        h, codes, scales = layer.norm_residual(s.y, s.residual, quantize=True, **step)
        return {"h": h, "out": layer.int8_qmm(codes, scales, s.w_codes, s.w_scales, dtype=s.dtype)}
    if s.kind == "logprobs":
        return _plain_logprobs(s)
    if s.kind == "linear":
        out = _plain_product(s.x.float(), s)
        return {"out": (out if s.bias is None else out + s.bias.float()).to(s.dtype)}
    branch = s.y.float()
    if s.post is not None:
        branch = _plain_norm(branch, s.post)
    if s.gate is not None:
        branch = branch * (s.gate[:, None] if s.gate.dim() == 1 and s.gate.dtype == torch.float32 else s.gate).float()
    h = s.residual.float() + s.multiplier * branch
    x = _plain_norm(h, s.pre)
    if s.kind == "norm":
        return {"h": h.to(s.dtype), "x": x.to(s.dtype)}
    return {"h": h.to(s.dtype), "out": _plain_product(x, s).to(s.dtype)}


def _plain_norm(x, w):
    return x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS) * w.float()


def _plain_product(x, s):
    largest = x.abs().amax(1, keepdim=True).clamp_min(2.0 ** -100)
    codes = (x * (127 / largest)).round()
    return (codes @ s.w_codes.float().t()) * (largest / 127) * s.w_scales


def _plain_logprobs(s):
    z = s.logits.float() * s.scale
    most = z.amax(1, keepdim=True)
    d = z - most
    e = torch.exp(d)
    total = e.sum(1)
    log_total = torch.log(total)
    entropy = log_total - torch.where(e > 0, d * e, 0.0).sum(1) / total
    logp = d.gather(1, s.tokens[:, None]).squeeze(1) - log_total
    # Largest first, ties to the lowest index: one whole number for each value, its order above and its index below.
    bits = s.logits.float().view(torch.int32).to(torch.int64)
    bits = torch.where(bits == -(1 << 31), 0, bits)  # -0 is 0
    order = torch.where(bits < 0, -(bits + (1 << 31)), bits)
    place = torch.arange(z.shape[1], device=z.device)
    ids = (-torch.topk(order * (1 << 18) - place, s.top, dim=1).values) % (1 << 18)
    top = d.gather(1, ids) - log_total[:, None]
    return {"logprobs": logp, "entropy": entropy, "top_ids": ids.to(torch.int32), "top_logprobs": top}


# -- what a pass cannot do without -------------------------------------------

def work(case):
    rows, size = case["rows"], 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "logprobs":
        vocab, top = case["vocab"], case["top"]
        return {"bytes": rows * (vocab * size + 8 + 8 + 8 * top), "flops": 6 * rows * vocab}
    width = case["width"]
    if case["kind"] == "linear":
        out = case["out"]
        return {"bytes": size * rows * (width + out) + out * (width + 4) + (size * out if case["bias"] else 0),
                "flops": 2 * rows * width * out}
    gate = {"none": 0, "channel": size * width, "token": 4 * rows, "full": size * rows * width}[case["gate"]]
    weights = size * width * (2 if case["post"] else 1)
    if case["kind"] == "norm":
        return {"bytes": 4 * size * rows * width + gate + weights, "flops": 14 * rows * width}
    out = case["out"]
    return {"bytes": size * rows * (3 * width + out) + gate + weights + out * (width + 4),
            "flops": 16 * rows * width + 2 * rows * width * out}


# -- the definition in 64 bits -----------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if s.kind == "logprobs":
        parts = {"logprobs": [], "entropy": [], "top_logprobs": []}
        for at in range(0, case["rows"], 512):
            z = s.logits[at:at + 512].double() * s.scale
            lp = z - torch.logsumexp(z, dim=1, keepdim=True)
            p = lp.exp()
            parts["entropy"].append(-torch.special.xlogy(p, p).sum(1))
            parts["logprobs"].append(torch.take_along_dim(lp, s.tokens[at:at + 512, None], 1)[:, 0])
            parts["top_logprobs"].append(lp.sort(dim=1, descending=True).values[:, :s.top])
        return {**{k: torch.cat(v) for k, v in parts.items()}, "top_ids": None}
    if s.kind == "linear":
        return {"out": _exact_product(s.x.double(), s)}
    h = s.y.double()
    if s.post is not None:
        h = h / (h.pow(2).sum(1, keepdim=True) / h.shape[1] + EPS).sqrt() * s.post.double()
    if case["gate"] == "token":
        h = h * s.gate.double().unsqueeze(1)
    elif case["gate"] != "none":
        h = h * s.gate.double()
    h = s.residual.double() + s.multiplier * h
    x = h / (h.pow(2).sum(1, keepdim=True) / h.shape[1] + EPS).sqrt() * s.pre.double()
    return {"h": h, "x": x} if s.kind == "norm" else {"h": h, "out": _exact_product(x, s)}


def _exact_product(x, s):
    step = x.abs().max(dim=1, keepdim=True).values / 127
    codes = torch.round(x / step)
    out = torch.matmul(codes, s.w_codes.double().t()) * step * s.w_scales.double()
    return out + s.bias.double() if getattr(s, "bias", None) is not None else out
