"""Dense scores and the distribution over them: rows in 8 bits, their integer
product with a scale for each row and column, log probabilities of given
columns with entropy and top alternatives, and their gradient.

Sizes are those of the searches (catalogues of 128, 100 and 96 dimensions of up
to a million rows, 1 to 10,000 queries, top-10) and generic ones of embedding
models and linear layers.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_TINY = 2.0 ** -119  # a row whose largest magnitude is below this counts as zeros


def _quantize(name, n, d, dtype):
    return dict(name=name, kind="quantize", n=n, d=d, dtype=dtype)


def _product(name, m, n, k, dtype, bias=False):
    return dict(name=name, kind="product", m=m, n=n, k=k, dtype=dtype, bias=bias)


def _log_probs(name, n, v, dtype, t, k, temperature=1.0, masked=0.0):
    return dict(name=name, kind="log_probs", n=n, v=v, dtype=dtype, t=t, k=k, temperature=temperature, masked=masked)


def _train(name, n, v, dtype, t, k, temperature=1.0, masked=0.0):
    return dict(name=name, kind="train", n=n, v=v, dtype=dtype, t=t, k=k, temperature=temperature, masked=masked)


def listed():
    return [
        # a service's small batch of float queries, before it is scored: latency
        _quantize("quantize 16 queries", 16, 96, "f32"),
        # a catalogue laid out once, and again whenever its vectors change
        _quantize("quantize 1M rows", 1_000_000, 128, "f32"),
        # one user's question against the whole catalogue
        _product("one query, 1M rows", 1, 1_000_000, 128, "f32"),
        # a small batch with a bias for each item, some filtered out
        _product("16 queries, 300k rows", 16, 300_000, 96, "f32", bias=True),
        # rows of 100 dimensions, which no 16-byte load divides, and an odd catalogue
        _product("1,000 queries, ragged", 1_000, 50_001, 100, "f16"),
        # a linear layer over a batch of tokens
        _product("linear layer", 4_096, 4_096, 4_096, "bf16"),
        # a query file of a benchmark, the scores of a shard written out
        _product("10k queries, 50k rows", 10_000, 50_001, 128, "bf16"),
        # the search's top-100 of every query, re-scored: their probabilities and the best ten
        _log_probs("10k lists of 100", 10_000, 100, "f32", 1, 10, 0.05),
        # one question's distribution over the whole catalogue
        _log_probs("one row of 1M", 1, 1_000_000, "f32", 1, 10, 0.05, 0.05),
        # a decoding batch, or a batch of queries: the answer's probability and 20 alternatives
        _log_probs("256 rows of 200k", 256, 200_000, "bf16", 1, 20, 1.0, 0.05),
        # a contrastive step: every other item of the batch is a negative
        _train("in-batch negatives", 4_096, 4_096, "bf16", 1, 0, 0.05),
        # several relevant items in a large odd catalogue, and the 50 hardest negatives, with an entropy term
        _train("catalogue loss", 1_000, 100_003, "f32", 4, 50, 1.0, 0.05),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantize", "product", "product", "product", "log_probs", "log_probs", "train", "train"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if kind == "quantize":
        d = rng.choice([64, 96, 100, 128, 256, 384, 769, 1024, 4096])
        c = _quantize("", _spread(rng, 1, 120_000_000 // d if d >= 128 else 900_000), d, dtype)
    elif kind == "product":
        m = rng.choice([1, 2, 7, 16, 33, 64, 100, 256, _spread(rng, 300, 8_000), _spread(rng, 300, 8_000)])
        k = rng.choice([64, 96, 100, 128, 128, 200, 256, 384, 768, 1_000, 1_024, 2_048, 4_096])
        n = _spread(rng, 200, min(900_000, 100_000_000 // k, 900_000_000 // (m * _SIZE[dtype]), 60_000_000_000 // (m * k)))
        c = _product("", m, n, k, dtype, rng.random() < 0.3)
    else:
        most = 80_000_000 if kind == "train" else 50_000_000
        n = _spread(rng, 1, 10_000)
        v = _spread(rng, 64, min(1_000_000, most // n))
        t = rng.choice([1, 1, 1, 2, 4])
        k = rng.choice([0, 1, 5, 10, 10, 20, 50])
        c = (_train if kind == "train" else _log_probs)("", n, v, dtype, t, k, rng.choice([0.05, 0.25, 1.0, 1.0]),
                                                        rng.choice([0.0, 0.05, 0.3]))
    del c["name"]
    return c


def _codes(g, rows, dim):
    """Normal vectors in 8 bits with a scale for each row, as a program keeps them."""
    x = torch.randn((rows, dim), generator=g, device="cuda")
    top = x.abs().amax(1, keepdim=True)
    return (x * (127.0 / top)).round_().to(torch.int8), (top / 127.0).flatten().contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _TYPES[case["dtype"]]
    s = {"case": case}
    if case["kind"] == "quantize":
        # embedding rows: normal entries, rows of different lengths
        length = torch.rand((case["n"], 1), generator=g, device="cuda") * 3 + 0.1
        s["x"] = (torch.randn((case["n"], case["d"]), generator=g, device="cuda") * length).to(dtype)
    elif case["kind"] == "product":
        s["a"], s["a_scales"] = _codes(g, case["m"], case["k"])
        s["b"], s["b_scales"] = _codes(g, case["n"], case["k"])
        s["bias"] = None
        if case["bias"]:
            bias = torch.randn(case["n"], generator=g, device="cuda")
            s["bias"] = torch.where(torch.rand(case["n"], generator=g, device="cuda") < 0.02, -math.inf, bias)
    else:
        n, v, t = case["n"], case["v"], case["t"]
        # scores of about three natural units' spread at the temperature, higher at the given columns
        x = torch.randn((n, v), generator=g, device="cuda") * (3.0 * case["temperature"])
        targets = torch.randint(0, v, (n, t), generator=g, device="cuda")
        if case["masked"]:
            x.masked_fill_(torch.rand((n, v), generator=g, device="cuda") < case["masked"], -math.inf)
        likely = (torch.randn((n, 1), generator=g, device="cuda") + 2.5) * (3.0 * case["temperature"])
        x.scatter_(1, targets, likely.expand(n, t))
        s["x"] = x.to(dtype)
        if t > 1:  # rows with fewer relevant items than others
            targets[:, 1:].masked_fill_(torch.rand((n, t - 1), generator=g, device="cuda") < 0.3, -1)
        s["targets"] = targets.to(torch.int32)
        if case["kind"] == "train":
            # a mean loss over the rows, weighted, with an entropy term; the negatives' own weights
            s["g_target"] = -torch.rand((n, t), generator=g, device="cuda") / n
            s["g_entropy"] = torch.full((n,), 0.01 / n, device="cuda")
            s["g_top"] = torch.rand((n, case["k"]), generator=g, device="cuda") / (n * max(1, case["k"]))
    return s


def _plain_quantize(s):
    x = s["x"].float()
    top = x.abs().amax(1, keepdim=True)
    some = top >= _TINY
    codes = torch.where(some, (x * (127.0 / top)).round(), 0.0)
    scales = torch.where(some, top / 127.0, 0.0)
    return {"values": codes * scales, "scales": scales.flatten()}


def _plain_product(s):
    out = (s["a"].float() @ s["b"].float().T) * s["a_scales"][:, None] * s["b_scales"][None, :]
    if s["bias"] is not None:
        out = out + s["bias"][None, :]
    return {"scores": out.to(_TYPES[s["case"]["dtype"]])}


def _plain_log_probs(s, train):
    c, targets = s["case"], s["targets"].long()
    x = s["x"].float()
    z = x * (1.0 / c["temperature"])
    top = z.amax(1, keepdim=True)
    y = z - top
    e = torch.exp(y)
    total = e.sum(1, keepdim=True)
    lp = y - torch.log(total)
    p = e / total
    entropy = -torch.where(p > 0, p * lp, 0.0).sum(1, keepdim=True)
    there = targets >= 0
    at = targets.clamp(min=0)
    out = {"target": torch.where(there, lp.gather(1, at), 0.0), "entropy": entropy.flatten()}
    if c["k"]:
        # whole numbers that order as the values do, the lower column first among equal ones
        bits = (x + 0.0).view(torch.int32).long()
        order = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF)
        column = torch.arange(c["v"], device=x.device)
        keys = torch.topk(order * 2 ** 32 + (2 ** 32 - 1 - column), min(c["k"], c["v"]), dim=1, sorted=True).values
        ids = 2 ** 32 - 1 - (keys & (2 ** 32 - 1))
        best = lp.gather(1, ids)
        out["top_ids"], out["top"] = torch.where(best > -math.inf, ids, -1).to(torch.int32), best
    if train:
        g_target = torch.where(there, s["g_target"], 0.0)
        total_g = g_target.sum(1, keepdim=True)
        if c["k"]:
            g_top = torch.where(best > -math.inf, s["g_top"], 0.0)
            total_g = total_g + g_top.sum(1, keepdim=True)
        dz = -p * total_g - s["g_entropy"][:, None] * torch.where(p > 0, p * (lp + entropy), 0.0)
        dz.scatter_add_(1, at, g_target)
        if c["k"]:
            dz.scatter_add_(1, ids, g_top)
        out["grad"] = (dz * (1.0 / c["temperature"])).to(s["x"].dtype)
    else:
        out["logsumexp"] = (top + torch.log(total)).flatten()
    return out


def _scoring():
    package = str(Path.cwd() / "quiver-ae_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from quiver import scoring

    return scoring


def _own(s):
    scoring, c = _scoring(), s["case"]
    if c["kind"] == "quantize":
        s["out"] = codes, scales = scoring.quantize_rows(s["x"], out=s.get("out"))
        return {"values": codes * scales[:, None], "scales": scales}
    if c["kind"] == "product":
        s["out"] = scoring.int8_product(s["a"], s["a_scales"], s["b"], s["b_scales"], bias=s["bias"],
                                        dtype=_TYPES[c["dtype"]], out=s.get("out"))
        return {"scores": s["out"]}
    r = scoring.log_probs(s["x"], s["targets"], top_k=c["k"], temperature=c["temperature"], out=s.get("out"))
    s["out"] = r
    out = {"target": r.target, "entropy": r.entropy}
    if c["k"]:
        out["top_ids"], out["top"] = r.top_ids, r.top
    if c["kind"] == "train":
        s["grad"] = out["grad"] = scoring.log_probs_grad(
            s["x"], r, s["targets"], grad_target=s["g_target"], grad_entropy=s["g_entropy"],
            grad_top=s["g_top"] if c["k"] else None, out=s.get("grad"))
    else:
        out["logsumexp"] = r.logsumexp
    return out


def run(s):
    if own:
        return _own(s)
    if s["case"]["kind"] == "quantize":
        return _plain_quantize(s)
    if s["case"]["kind"] == "product":
        return _plain_product(s)
    return _plain_log_probs(s, s["case"]["kind"] == "train")


def work(case):
    size = _SIZE[case["dtype"]]
    if case["kind"] == "quantize":
        n, d = case["n"], case["d"]
        return {"bytes": n * d * (size + 1) + 4 * n, "flops": 3 * n * d}
    if case["kind"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m + n) * (k + 4) + (4 * n if case["bias"] else 0) + m * n * size, "flops": 2 * m * n * k}
    n, v, t, k = case["n"], case["v"], case["t"], case["k"]
    forward = n * v * size + n * (8 * t + 8 + 8 * k)
    if case["kind"] == "log_probs":
        return {"bytes": forward, "flops": 6 * n * v}
    return {"bytes": forward + n * v * size + n * (4 * t + 4 + 4 * k), "flops": 14 * n * v}


def exact(case, seed):
    """The definitions in 64 bits: softmax and its entropy by torch's own, the gradient by the chain rule
    over the matrix of first derivatives' diagonal and rank-one part."""
    s = prepare(case, seed)
    if case["kind"] == "quantize":
        x = s["x"].double()
        scale = x.abs().max(dim=1).values / 127.0
        codes = torch.round(x / scale.clamp(min=1e-300)[:, None])
        return {"values": codes * scale[:, None], "scales": scale}
    if case["kind"] == "product":
        a = s["a"].double() * s["a_scales"].double()[:, None]
        b = s["b"].double() * s["b_scales"].double()[:, None]
        scores = torch.mm(a, b.t())
        return {"scores": scores if s["bias"] is None else scores + s["bias"].double()}
    x = s["x"].double() / case["temperature"]
    lp = torch.log_softmax(x, dim=1)
    p = torch.softmax(x, dim=1)
    entropy = torch.special.entr(p).sum(1)
    targets = s["targets"].long()
    rows = torch.arange(case["n"], device="cuda")[:, None]
    present = (targets >= 0).double()
    out = {"target": torch.nan_to_num(lp[rows, targets.clamp(min=0)] * present, nan=0.0), "entropy": entropy}
    ids = None
    if case["k"]:
        ids = torch.sort(s["x"].double(), dim=1, descending=True, stable=True).indices[:, :case["k"]]
        best = lp[rows, ids]
        out["top_ids"], out["top"] = torch.where(torch.isinf(best), -1, ids).to(torch.int32), best
    if case["kind"] == "log_probs":
        out["logsumexp"] = torch.logsumexp(x, dim=1)
        return out
    # d out / d z for out = sum of weights w_j lp_j is w - p sum(w); for the entropy it is -p (lp + H)
    w = torch.zeros_like(x)
    w.index_put_((rows.expand_as(targets), targets.clamp(min=0)), s["g_target"].double() * present, accumulate=True)
    if ids is not None:
        w.index_put_((rows.expand_as(ids), ids), s["g_top"].double() * torch.isfinite(best), accumulate=True)
    h = -torch.special.entr(p) + p * entropy[:, None]
    dz = w - p * w.sum(1, keepdim=True) - s["g_entropy"].double()[:, None] * h
    out["grad"] = dz / case["temperature"]
    return out
