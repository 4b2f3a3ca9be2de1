"""Log probabilities, entropy, alternatives and their gradient against the definitions in 64 bits.

With U = 2^-24: y = (x - max) / T rounds three times (the difference, the
constant, the product), so exp(y) is off by 3 U |y| of itself and 2 U of the
function's; terms with y < -24 are below U of the sum, so every term that
counts is within 74 U.  The sum adds at most L = cols / 64 + 80 roundings (a
lane's chain and the joins; more lanes, fewer).  So S is within E = (74 + L) U,
ln S within E + U |ln S|, a log probability within E + 4 U (|y| + |ln S| + 1), the
entropy's second sum within (E + 4 U 24) of sum |y| exp(y) <= S |y| ..., that is
(E + 100 U) (|H| + 2 |ln S| + 2) altogether.  p = exp(lp) is within the bound of
lp of itself (relative), and a gradient's terms add that up, with 3 U of each
and one rounding to the logits' type.
"""
from __future__ import annotations

import math
import sys

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ROUND = {torch.float32: (U, 2.0 ** -149), torch.bfloat16: (2.0 ** -8, 2.0 ** -134), torch.float16: (2.0 ** -11, 2.0 ** -25)}
TYPES = list(ROUND)
INF = math.inf
FLOAT_MAX = float(np.finfo(np.float32).max)


@pytest.fixture(scope="module")
def scoring():
    from quiver import _lib, scoring

    if _lib.device_count() == 0:
        pytest.skip("no GPU")
    yield scoring
    torch.cuda.empty_cache()  # the memory is the other tests' again


def say(*a):
    print("[gpu]", *a, flush=True)


class Plain:
    """The definitions in 64 bits, for rows without NaN or +inf."""

    def __init__(self, x, targets, k, T):
        x64 = x.double().cpu().numpy()
        n, v = x64.shape
        self.x, self.T, self.k = x64, float(np.float32(T)), k
        self.m = x64.max(1, initial=-INF)
        self.empty = self.m == -INF
        ref = np.where(self.empty, 0.0, self.m)
        self.y = (x64 - ref[:, None]) / self.T
        with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
            e = np.exp(self.y)
            s = e.sum(1)
            self.ln_s = np.log(s)
            self.lp = np.where(x64 == -INF, -INF, self.y - self.ln_s[:, None])
            self.p = np.exp(self.lp)
            plogp = np.where(self.p > 0, self.p * self.lp, 0.0)
            self.entropy = -plogp.sum(1)
            self.lse = np.where(self.empty, -INF, ref / self.T + self.ln_s)
        self.targets = np.zeros((n, 0), np.int64) if targets is None else targets.cpu().numpy().reshape(n, -1)
        t = self.targets
        self.target = np.where(t < 0, 0.0, np.take_along_axis(self.lp, np.clip(t, 0, max(v - 1, 0)), 1) if v else -INF)
        self.target = np.where(t >= v, np.nan, self.target)
        order = np.argsort(-x64, axis=1, kind="stable")[:, :k]
        best = np.take_along_axis(x64, order, 1)
        ids = np.where(best == -INF, -1, order)
        self.ids = np.full((n, k), -1)
        self.ids[:, :ids.shape[1]] = ids
        self.top = np.full((n, k), -INF)
        self.top[:, :ids.shape[1]] = np.where(best == -INF, -INF, np.take_along_axis(self.lp, order, 1))
        ln = np.abs(np.where(self.empty, 0, self.ln_s))
        self.e = (74 + v / 64 + 80) * U
        self.slack_lp = self.e + 4 * U * (np.where(np.isfinite(self.y), np.abs(self.y), 0) + ln[:, None] + 1)
        self.slack_h = (self.e + 100 * U) * (np.abs(self.entropy) + 2 * ln + 2)
        self.ln = ln

    def grad(self, gt, ge, gl, gk):
        n, v = self.x.shape
        w = np.zeros((n, v))
        size = np.zeros((n, v))  # sum of the terms' magnitudes
        for ids, g in ((self.targets, gt), (self.ids, gk)):
            if g is None:
                continue
            for i in range(n):
                for j, a in zip(ids[i], g[i]):
                    if 0 <= j < v:
                        w[i, j] += a
                        size[i, j] += abs(a)
        total = w.sum(1) - (0 if gl is None else gl)
        reach = size.sum(1) + (0 if gl is None else np.abs(gl))
        ge = np.zeros(n) if ge is None else ge
        with np.errstate(invalid="ignore"):
            bend = np.where(self.p > 0, self.p * (self.lp + self.entropy[:, None]), 0.0)
            # magnitudes: p (|lp| + H) rather than their sum
            bend_size = np.where(self.p > 0, self.p * (np.abs(self.lp) + np.abs(self.entropy)[:, None]), 0.0)
        dz = w - self.p * total[:, None] - ge[:, None] * bend
        few = size.shape[1] and 130 * U  # the sum over up to 128 weights, and the terms' own roundings
        slack = (size + self.p * reach[:, None] + np.abs(ge)[:, None] * bend_size) * (few + self.slack_lp) \
            + np.abs(ge)[:, None] * self.p * (self.slack_lp + self.slack_h[:, None])
        dz[self.empty] = 0
        return dz / self.T, slack / self.T


def _near(got, want, slack, what):
    got = got.double().cpu().numpy()
    assert got.shape == want.shape, what
    want = np.where(np.abs(want) > FLOAT_MAX, np.sign(want) * INF, want)  # past the largest float: an infinity
    fine = np.isfinite(want)
    np.testing.assert_array_equal(got[~fine], want[~fine], err_msg=what)
    err = np.where(fine, np.abs(np.where(fine, got, 0) - np.where(fine, want, 0)), 0)
    bad = err > np.broadcast_to(slack, err.shape) + 2.0 ** -126
    assert not bad.any(), f"{what}: {bad.sum()} values, first at {np.argwhere(bad)[:3].tolist()}: " \
                          f"{got[bad][:3]} for {want[bad][:3]}"


def _check(r, plain):
    v, t = plain.x.shape[1], plain.targets
    slack_t = np.take_along_axis(plain.slack_lp, np.clip(t, 0, max(v - 1, 0)), 1) if v else np.zeros(t.shape)
    _near(r.target, plain.target, slack_t, "target")
    _near(r.entropy, plain.entropy, plain.slack_h, "entropy")
    m = np.where(plain.empty, 0, np.abs(plain.m)) / plain.T
    _near(r.logsumexp, plain.lse, plain.e + 4 * U * (m + plain.ln + 1), "logsumexp")
    np.testing.assert_array_equal(r.top_ids.cpu().numpy(), plain.ids)
    at = np.clip(plain.ids, 0, None)
    _near(r.top, plain.top, np.take_along_axis(plain.slack_lp, at, 1) if v else 0.0, "top")


def _inputs(dtype, n, v, t, seed, T=1.0, masked=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((n, v), generator=g, device="cuda") * 3 * T
    if masked:
        x.masked_fill_(torch.rand((n, v), generator=g, device="cuda") < masked, -INF)
    targets = torch.randint(0, max(v, 1), (n, t), generator=g, device="cuda").to(torch.int32) if v else None
    return x.to(dtype), targets


def _run(scoring, x, targets, k, T, seed=1, grads=True):
    r = scoring.log_probs(x, targets, top_k=k, temperature=T)
    plain = Plain(x, targets, k, T)
    _check(r, plain)
    if not grads:
        return r, plain
    n, t = x.shape[0], plain.targets.shape[1]
    rng = np.random.default_rng(seed)
    gt, ge, gl, gk = (rng.standard_normal(s).astype(np.float32) for s in ((n, t), n, n, (n, k)))
    g = [torch.from_numpy(a).cuda() for a in (gt, ge, gl, gk)]
    for use in ((1, 0, 0, 0), (1, 1, 1, 1), (0, 1, 0, 0), (0, 0, 0, 1)):
        if (use[0] and not t and sum(use) == 1) or (use[3] and not k and sum(use) == 1):
            continue
        a = [x_ if u else None for x_, u in zip(g, use)]
        out = scoring.log_probs_grad(x, r, targets, grad_target=a[0], grad_entropy=a[1], grad_logsumexp=a[2],
                                     grad_top=a[3])
        want, slack = plain.grad(*[x_.astype(np.float64) if u else None for x_, u in zip((gt, ge, gl, gk), use)])
        rel, least = ROUND[x.dtype]
        assert out.dtype == x.dtype
        _near(out, want, slack + (np.abs(want) + slack) * rel + least, f"gradient {use}")
    return r, plain


# lengths around a wave's and a workgroup's loads and the splits; odd ones; one row and many
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, v, t, k, T", [
    (1, 1, 1, 1, 1.0), (3, 2, 1, 2, 0.5), (5, 7, 2, 10, 1.0), (70, 63, 1, 10, 0.05), (9, 64, 1, 64, 1.0),
    (33, 65, 3, 5, 2.0), (1000, 100, 1, 10, 0.05), (17, 128, 0, 20, 1.0), (40, 255, 1, 0, 1.0), (6, 256, 4, 64, 0.1),
    (12, 257, 1, 33, 1.0), (7, 511, 1, 10, 1.0), (300, 513, 1, 1, 1.0), (20, 1000, 5, 50, 0.3), (4, 1023, 1, 10, 1.0),
    (4, 1025, 64, 64, 1.0), (31, 2048, 1, 10, 1.0), (3, 2049, 1, 64, 1.0), (100, 4096, 1, 10, 0.05), (5, 4099, 2, 7, 1.0),
    (2, 16385, 1, 64, 1.0), (13, 20001, 1, 10, 1.0), (1, 70003, 3, 50, 0.05), (300, 9001, 1, 20, 1.0), (210, 17001, 1, 20, 1.0),
    (250, 16385, 2, 64, 0.2), (256, 16400, 1, 1, 1.0), (4100, 1030, 1, 5, 1.0)])
def test_rows(scoring, dtype, n, v, t, k, T):
    say("log probs", dtype, n, v, t, k, T)
    x, targets = _inputs(dtype, n, v, t, n + v, T)
    _run(scoring, x, targets if t else None, k, T)
    x, targets = _inputs(dtype, n, v, t, n + v + 1, T, masked=0.4)
    _run(scoring, x, targets if t else None, k, T)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v, rows", [(50, 14), (300, 14), (5000, 14), (40000, 14), (16500, 252)])
def test_masks(scoring, dtype, v, rows):
    """Rows with nothing, one value, all equal, the type's lowest value as a mask, huge and tiny values, signed zeros."""
    say("log probs, masks", dtype, v, rows)
    low = torch.finfo(dtype).min
    x = torch.randn((14, v), device="cuda").to(dtype)
    x[0] = -INF
    x[1] = -INF
    x[1, v - 1] = -3.0
    x[2] = 0.0
    x[2, ::2] = -0.0
    x[3] = low
    x[4, : v - 2] = low
    x[5] = -low
    x[6, 5:] = -INF
    x[7] = low
    x[7, v // 2] = -low
    x[8] *= 1e-4
    x[9] = torch.finfo(dtype).tiny
    x[10] = torch.arange(v, device="cuda").to(dtype)          # ascending: every value is a new largest one
    x[11] = -torch.arange(v, device="cuda").to(dtype)
    x[12] = torch.arange(v, device="cuda").to(dtype) % 3      # ties everywhere
    x[13, : v // 2] = -INF
    targets = torch.stack([torch.zeros(14, device="cuda"), torch.full((14,), v - 1, device="cuda"),
                           torch.full((14,), -1, device="cuda")], 1).to(torch.int32)
    x, targets = x.repeat(rows // 14, 1), targets.repeat(rows // 14, 1)  # (more rows: more waves for each)
    for T in (1.0, 0.125):
        _run(scoring, x, targets, 12, T)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [40, 700, 30000])
def test_no_distribution(scoring, dtype, v):
    """A NaN or +inf anywhere in a row makes its numbers NaN and its ids -1, and no other row's."""
    say("log probs, NaN and infinities", dtype, v)
    x, targets = _inputs(dtype, 7, v, 1, v)
    clean = x.clone()
    x[1, 0] = float("nan")
    x[2, v - 1] = INF
    x[3] = float("nan")
    x[4, v // 2] = float("nan")
    x[4, v // 3] = -INF
    x[5] = -INF
    x[5, 3] = float("nan")
    r = scoring.log_probs(x, targets, top_k=3)
    ones = torch.ones((7, 3), device="cuda")
    grad = scoring.log_probs_grad(x, r, targets, grad_target=ones[:, :1].contiguous(), grad_top=ones)
    for i in range(1, 6):
        for part in (r.target, r.entropy, r.logsumexp, r.top, grad):
            assert torch.isnan(part[i]).all(), (i, part[i])
        assert (r.top_ids[i] == -1).all()
    keep = torch.tensor([0, 6], device="cuda")
    rc = scoring.log_probs(clean[keep].contiguous(), targets[keep].contiguous(), top_k=3)
    for part in ("target", "entropy", "logsumexp", "top", "top_ids"):
        np.testing.assert_allclose(getattr(r, part)[keep].double().cpu(), getattr(rc, part).double().cpu(), rtol=1e-4)


def test_targets(scoring):
    """Absent targets, repeated ones, ones that are alternatives too, and ones past the row's end."""
    say("log probs, targets")
    for v in (90, 3000, 50000):
        x, _ = _inputs(torch.float32, 6, v, 1, v)
        best = x.argmax(1).to(torch.int32)
        targets = torch.full((6, 5), -1, dtype=torch.int32, device="cuda")
        targets[1] = 3
        targets[2, :3] = best[2]
        targets[3] = torch.tensor([0, v - 1, -7, 0, v // 2])
        targets[4, 0] = best[4]
        _run(scoring, x, targets, 4, 0.5)
        targets[5, 1] = v
        targets[5, 2] = 2 ** 31 - 1
        r = scoring.log_probs(x, targets, top_k=4)
        assert torch.isnan(r.target[5, 1:3]).all() and (r.target[5, [0, 3, 4]] == 0).all()
        assert torch.isfinite(r.target[:5]).all() and torch.isfinite(r.entropy).all()
        one = scoring.log_probs(x, best, top_k=1)  # targets of one dimension
        assert torch.equal(one.target, one.top) and torch.equal(one.top_ids[:, 0], best)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, v, wide, off", [(9, 100, 131, 3), (5, 1000, 1001, 1), (3, 30001, 30007, 5), (300, 64, 65, 1)])
def test_strides(scoring, dtype, n, v, wide, off):
    """Logits and gradient inside wider matrices, at odd addresses; nothing beside the gradient is written; in place."""
    say("log probs strides", dtype, n, v, wide, off)
    store, targets = _inputs(dtype, n, wide, 2, v)
    targets %= v
    x = store[:, off:off + v]
    r, plain = _run(scoring, x, targets, 6, 1.0)
    g = torch.randn((n, 2), device="cuda")
    h = torch.randn((n,), device="cuda")
    want = scoring.log_probs_grad(x, r, targets, grad_target=g, grad_entropy=h)
    other = torch.full((n, wide + 3), 5.0, dtype=dtype, device="cuda")
    scoring.log_probs_grad(x, r, targets, grad_target=g, grad_entropy=h, out=other[:, off:off + v])
    assert torch.equal(other[:, off:off + v], want)
    assert (other[:, :off] == 5).all() and (other[:, off + v:] == 5).all()
    before = store.clone()
    scoring.log_probs_grad(x, r, targets, grad_target=g, grad_entropy=h, out=x)
    assert torch.equal(x, want)
    assert torch.equal(store[:, :off], before[:, :off]) and torch.equal(store[:, off + v:], before[:, off + v:])


def test_differences(scoring):
    """The gradient along random directions against central differences of the 64-bit definitions.

    With steps of h = 1e-4 in each z a difference is off by h^2 / 6 of third derivatives, which for these functions are
    below 8 (sum of weights) (1 + |lp|): under 1e-6 of the weights; the gradient's own bound is added.
    """
    say("log probs, gradient against differences")
    for v, T in ((30, 1.0), (3000, 0.25)):
        x, targets = _inputs(torch.float32, 4, v, 2, v, T)
        r = scoring.log_probs(x, targets, top_k=5, temperature=T)
        rng = np.random.default_rng(v)
        gt, ge, gl, gk = (rng.standard_normal(s).astype(np.float32) for s in ((4, 2), 4, 4, (4, 5)))
        grad = scoring.log_probs_grad(x, r, targets, grad_target=torch.from_numpy(gt).cuda(),
                                      grad_entropy=torch.from_numpy(ge).cuda(),
                                      grad_logsumexp=torch.from_numpy(gl).cuda(), grad_top=torch.from_numpy(gk).cuda())
        ids = r.top_ids.long().cpu().numpy()

        def value(x64):
            z = torch.from_numpy(x64) / T
            lp = torch.log_softmax(z, 1).numpy()
            at = targets.long().cpu().numpy()
            return ((np.take_along_axis(lp, at, 1) * gt).sum() + ((-np.exp(lp) * lp).sum(1) * ge).sum()
                    + (torch.logsumexp(z, 1).numpy() * gl).sum() + (np.take_along_axis(lp, ids, 1) * gk).sum())

        x64 = x.double().cpu().numpy()
        slack = Plain(x, targets, 5, T).grad(gt, ge, gl, gk)[1]
        weights = np.abs(gt).sum() + np.abs(ge).sum() + np.abs(gl).sum() + np.abs(gk).sum()
        for _ in range(5):
            d = rng.standard_normal(x64.shape)
            d *= T / np.abs(d).max()
            h = 1e-4
            along = (value(x64 + h * d) - value(x64 - h * d)) / (2 * h)
            got = (grad.double().cpu().numpy() * d).sum()
            grad_slack = (np.abs(d) * (slack + U * np.abs(grad.double().cpu().numpy()))).sum()
            assert abs(along - got) <= 1e-5 * weights + grad_slack, (along, got)


def test_autograd(scoring):
    """The results take part in autograd; the gradient is log_probs_grad's."""
    say("log probs, autograd")
    for dtype in TYPES:
        x, targets = _inputs(dtype, 8, 500, 2, 3)
        leaf = x.clone().requires_grad_()
        r = scoring.log_probs(leaf, targets, top_k=4, temperature=0.5)
        loss = -r.target.mean() + 0.1 * r.entropy.sum() + r.logsumexp.square().sum() * 1e-3 + r.top[:, 1:].sum()
        loss.backward()
        plain = scoring.log_probs(x, targets, top_k=4, temperature=0.5)
        gk = torch.ones((8, 4), device="cuda")
        gk[:, 0] = 0
        want = scoring.log_probs_grad(x, plain, targets, grad_target=torch.full((8, 2), -1 / 16, device="cuda"),
                                      grad_entropy=torch.full((8,), 0.1, device="cuda"),
                                      grad_logsumexp=2e-3 * plain.logsumexp, grad_top=gk)
        assert leaf.grad.dtype == dtype
        torch.testing.assert_close(leaf.grad, want, rtol=4 * ROUND[dtype][0], atol=1e-6)
        leaf.grad = None
        scoring.log_probs(leaf, targets).target.sum().backward()  # the other gradients are absent
        r1 = scoring.log_probs(x, targets)
        assert torch.equal(leaf.grad, scoring.log_probs_grad(x, r1, targets, grad_target=torch.ones((8, 2), device="cuda")))
        with pytest.raises(ValueError, match="out="):
            scoring.log_probs(leaf, targets, out=plain)


def test_no_second_gradient(scoring):
    """A second derivative is refused, not taken as zero."""
    from quiver import _lib

    say("log probs, second derivative")
    leaf = torch.randn((4, 50), device="cuda").requires_grad_()
    (grad,) = torch.autograd.grad(scoring.log_probs(leaf).entropy.sum(), leaf, create_graph=True)
    want = scoring.log_probs_grad(leaf.detach(), scoring.log_probs(leaf.detach()), grad_entropy=torch.ones(4, device="cuda"))
    assert torch.equal(grad, want)
    with pytest.raises(_lib.QuiverError, match="differentiated again"):
        (grad.square().sum() + leaf.sum()).backward()


def test_overwritten(scoring):
    """A backward pass that needs what out= has overwritten since is refused."""
    say("results written again before the backward pass")
    codes, scales = scoring.quantize_rows(torch.randn((40, 64), device="cuda"))
    logits, weight = scoring.int8_product(codes[:8], scales[:8], codes, scales), torch.ones(8, device="cuda", requires_grad=True)
    r = scoring.log_probs(logits, top_k=2)

    def writes():
        yield logits, lambda: scoring.int8_product(codes[:8], scales[:8], codes, scales, out=logits)
        yield logits, lambda: scoring.log_probs_grad(logits, r, grad_entropy=torch.ones(8, device="cuda"), out=logits)
        yield r.entropy, lambda: scoring.log_probs(logits, top_k=2, out=r)
        yield scales, lambda: scoring.quantize_rows(torch.randn((40, 64), device="cuda"), out=(codes, scales))

    for held, write in writes():
        (held.reshape(-1)[:8] * weight).sum().backward()
        loss = (held.reshape(-1)[:8] * weight).sum()
        write()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


def test_empty_sizes(scoring):
    say("log probs, no rows and no columns")
    r = scoring.log_probs(torch.empty((0, 5), device="cuda"), top_k=2)
    assert r.top_ids.shape == (0, 2) and r.entropy.shape == (0,)
    x = torch.empty((3, 0), device="cuda")
    targets = torch.tensor([[-1], [0], [4]], dtype=torch.int32, device="cuda")
    r = scoring.log_probs(x, targets, top_k=2)
    assert (r.logsumexp == -INF).all() and (r.entropy == 0).all() and (r.top_ids == -1).all() and (r.top == -INF).all()
    assert r.target[0, 0] == 0 and torch.isnan(r.target[1:, 0]).all()
    assert scoring.log_probs_grad(x, r, targets, grad_target=torch.ones((3, 1), device="cuda")).shape == (3, 0)


def test_long_matrix(scoring):
    """Rows that begin past 2^31 elements."""
    say("log probs, offsets past 32 bits")
    n, v = 3, 1_500_000_000
    x = torch.empty((n, v), dtype=torch.bfloat16, device="cuda")
    x.fill_(-40.0)
    x[2, v - 1], x[2, 7], x[1, 0] = 3.0, 2.0, 1.0
    targets = torch.tensor([[5], [0], [v - 1]], dtype=torch.int32, device="cuda")
    r = scoring.log_probs(x, targets, top_k=3)
    assert r.top_ids.tolist() == [[0, 1, 2], [0, 1, 2], [v - 1, 7, 0]]
    s = math.exp(-43) * (v - 2) + 1 + math.exp(-1)
    assert abs(r.target[2, 0].item() + math.log(s)) < 1e-6
    assert abs(r.logsumexp[0].item() - (math.log(v) - 40)) < 1e-4
    grad = scoring.log_probs_grad(x, r, targets, grad_target=torch.ones((3, 1), device="cuda"), out=x)
    assert abs(grad[2, v - 1].item() - (1 - 1 / s)) < 2e-3 and abs(grad[2, 7].item() + math.exp(-1) / s) < 2e-3


def test_many_rows(scoring):
    """More rows than one launch has threads for (2^32, 64 a row)."""
    n = 2 ** 26 + 77
    say("log probs and gradient,", n, "rows")
    place = torch.arange(n, device="cuda") % 11
    x = torch.stack([torch.zeros(n, device="cuda"), (place - 5).float()], 1)
    targets = torch.ones(n, dtype=torch.int32, device="cuda")
    r = scoring.log_probs(x, targets, top_k=1)
    d = torch.arange(-5, 6, dtype=torch.float64, device="cuda")
    lp = -torch.log1p(torch.exp(-d))
    bound = (74 + 82) * U + 4 * U * 7 + U * 6  # |y| <= 5, ln S < 1; lp to a float below
    assert ((r.target[:, 0] - lp.float()[place]).abs() <= bound).all()
    assert (r.top_ids[:, 0] == (d > 0)[place]).all()
    grad = scoring.log_probs_grad(x, r, targets, grad_target=torch.ones((n, 1), device="cuda"), out=x)
    assert ((grad[:, 1] - (1 - lp.exp()).float()[place]).abs() <= bound + 4 * U).all()
    assert ((grad[:, 0] + (1 - lp.exp()).float()[place]).abs() <= bound + 4 * U).all()


def test_other_stream_reuse_and_repeat(scoring):
    """Results written again through out=, on a stream of their own, in a captured graph; equal calls, equal bits."""
    say("log probs, streams and graphs")
    for n, v in ((1, 200_000), (64, 5000), (2000, 100)):
        x, targets = _inputs(torch.bfloat16, n, v, 1, v)
        want = scoring.log_probs(x, targets, top_k=10)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            y = x * 1.0
            r = scoring.log_probs(y, targets, top_k=10)
            r = scoring.log_probs(y, targets, top_k=10, out=r)
        side.synchronize()
        for part in ("target", "entropy", "logsumexp", "top", "top_ids", "stats"):
            assert torch.equal(getattr(r, part), getattr(want, part)), part
        g = -torch.ones((n, 1), device="cuda")
        grad = scoring.log_probs_grad(x, want, targets, grad_target=g)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            scoring.log_probs(y, targets, top_k=10, out=r)
            out = scoring.log_probs_grad(y, r, targets, grad_target=g)
        for turn in range(3):
            y.copy_(x * (turn + 1))
            graph.replay()
            torch.cuda.synchronize()
            fresh = scoring.log_probs(y.clone(), targets, top_k=10)
            assert torch.equal(r.top_ids, fresh.top_ids) and torch.equal(r.entropy, fresh.entropy)
            assert torch.equal(out, scoring.log_probs_grad(y, fresh, targets, grad_target=g))
        y.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, grad)


def test_catalogue(scoring):
    """A catalogue in 8 bits, scored and normalised batch by batch: the parts' own results, and those of float vectors
    within what 8 bits leave: entries of about 0.088 and at most about 0.28 are off by up to half of 0.28 / 127, 0.0006 rms, a
    product of 128 of them by sqrt(2 * 128) * 0.0006 * 0.088 = 0.0009, 0.017 at the temperature, six times that at most."""
    say("dense catalogue")
    g = torch.Generator(device="cuda").manual_seed(1)
    vectors = torch.nn.functional.normalize(torch.randn((5001, 128), generator=g, device="cuda"), dim=1)
    targets = torch.randint(0, 5001, (300, 1), generator=g, device="cuda")
    queries = torch.nn.functional.normalize(vectors[targets[:, 0]] + 0.05 * torch.randn((300, 128), generator=g, device="cuda"), dim=1)
    bias = torch.zeros(5001, device="cuda")
    bias[17] = -INF
    targets[targets == 17] = 18
    targets = targets.to(torch.int32)
    whole = scoring.DenseCatalogue(vectors, bias=bias)
    pieces = scoring.DenseCatalogue(vectors, bias=bias, score_bytes=77 * 5001 * 4)
    a = whole.log_probs(queries, targets, top_k=5, temperature=0.05)
    b = pieces.log_probs(queries, targets, top_k=5, temperature=0.05)
    for part in ("target", "entropy", "logsumexp", "top", "top_ids", "stats"):
        np.testing.assert_allclose(getattr(a, part).double().cpu(), getattr(b, part).double().cpu(), rtol=1e-5, atol=1e-5)
    assert not (a.top_ids == 17).any()
    exact = (queries.double() @ vectors.double().T + bias.double()) / 0.05
    lp = torch.log_softmax(exact, 1)
    assert (a.target.double() - lp.gather(1, targets.long())).abs().max() < 0.11
    assert ((a.top_ids[:, 0].long() == lp.argmax(1)).double().mean()) > 0.95


# one wave per row of one load and of more, 4 and 16 waves, chunks
RANGE_COLS = [100, 700, 5000, 20000, 40000]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", RANGE_COLS)
def test_finite_masks(scoring, dtype, v):
    """Masks of finite values, in whole lanes, whole rows, the half, the tail, here and there, all but one column."""
    say("log probs, finite masks", dtype, v)
    masks = [-1e4, -6e4] if dtype == torch.float16 else [-1e4, -1e9, -1e10, -1e12, -1e20, -1e30, -1e37]
    g = torch.Generator(device="cuda").manual_seed(v)
    rows = 6 * len(masks)
    targets = torch.tensor([0, v // 2, v - 1], dtype=torch.int32, device="cuda").repeat(rows, 1)
    for T in (0.05, 0.1, 1.0, 2.0):
        x = torch.randn((rows, v), generator=g, device="cuda") * 3 * T
        for i, mask in enumerate(masks):
            at = x[6 * i:6 * i + 6]
            at[0, :8] = mask
            at[1] = mask
            at[2, :v // 2] = mask
            at[3, v // 3:] = mask
            at[4, torch.rand(v, generator=g, device="cuda") < 0.9] = mask
            at[5, :v - 2] = mask
            at[5, v - 1] = mask
        _run(scoring, x.to(dtype), targets, 12, T)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", RANGE_COLS)
def test_large_logits(scoring, dtype, v):
    """Rows around values up to 1e37, the ones where differences begin to be taken first (2^20 / log2(e) at T = 1) among them."""
    say("log probs, large logits", dtype, v)
    g = torch.Generator(device="cuda").manual_seed(v)
    for T in (0.05, 1.0):
        limit = 2.0 ** 20 * math.log(2) * T
        bases = [s * b for b in (1e5, limit, 1e7, 1e9, 3e12, 1e20, 1e30, 1e37) for s in (1, -1)]
        spread = torch.tensor([max(20 * T, abs(b) * 2.0 ** -21) for b in bases], device="cuda")
        x = torch.tensor(bases, device="cuda")[:, None] + spread[:, None] * torch.randn((len(bases), v), generator=g, device="cuda")
        x[2::4, ::5] *= 0.5  # lanes far apart, too
        targets = torch.tensor([0, v // 2, v - 1], dtype=torch.int32, device="cuda").repeat(len(bases), 1)
        targets[:, 0] = x.argmax(1)
        _run(scoring, x.to(dtype), targets, 12, T)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", RANGE_COLS)
def test_low_temperatures(scoring, dtype, v):
    """Nearly greedy temperatures: ties share the probability, the next value has next to none."""
    say("log probs, low temperatures", dtype, v)
    g = torch.Generator(device="cuda").manual_seed(v)
    x = torch.randn((8, v), generator=g, device="cuda") * 3
    x[1] = 12.7
    x[2, :] = 12.7
    x[2, 1::3] = 12.699999
    x[3, 1:] = 29
    x[3, 0] = 30
    x[4] = 0
    x[5] = -x[1]
    x[6] = 7.1
    x[6, v // 2:] = 5
    x[7] = torch.where(x[7] > 1, 5.3, -1e4)
    x = x.to(dtype)
    targets = torch.stack([x.argmax(1), x.argmin(1)], 1).to(torch.int32)
    for T in (1e-3, 1e-6, 1e-8, 1e-9, 1e-10, 1e-12, 1e-20, 1e-37):
        # (gradients go with 1 / T: within the type's range only)
        _run(scoring, x, targets, 12, T, grads=dtype != torch.float16 and T > 1e-30)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", RANGE_COLS)
def test_far_apart(scoring, dtype, v):
    """Logits that differ by more than the largest float, at temperatures that bring them near to each other again.

    The gradient is that of weights of 1e30, so that it is no subnormal number.
    """
    say("log probs, logits far apart", dtype, v)
    g = torch.Generator(device="cuda").manual_seed(v)
    x = (torch.rand((6, v), generator=g, device="cuda") * 2 - 1) * 3.38e38
    x[1] = 3.38e38
    x[1, v // 2:] = -3.38e38
    x[2, 1:] = -3.38e38
    x[2, 0] = 3.38e38
    x[3] *= 0.01
    x = x.to(dtype)
    targets = torch.stack([x.argmax(1), x.argmin(1)], 1).to(torch.int32)
    for T in (1e36, 1e37, 1e38, 3e38):
        r, plain = _run(scoring, x, targets, 12, T)
        rng = np.random.default_rng(v)
        weights = [(rng.standard_normal(s) * 1e30).astype(np.float32) for s in ((6, 2), 6, 6, (6, 12))]
        out = scoring.log_probs_grad(x, r, targets, **{
            "grad_" + name: torch.from_numpy(w).cuda() for name, w in zip(("target", "entropy", "logsumexp", "top"), weights)})
        want, slack = plain.grad(*[w.astype(np.float64) for w in weights])
        rel, least = ROUND[dtype]
        _near(out, want, slack + (np.abs(want) + slack) * rel + least, "gradient of large weights")


@pytest.mark.parametrize("v", [90, 3000, 50000])
def test_gradient_past_the_end(scoring, v):
    """A weighed target past the row's end makes its row's gradient NaN, as the log probability is; with the weight 0 it is absent."""
    say("log probs, gradient of targets past the end", v)
    x, targets = _inputs(torch.float32, 4, v, 2, v)
    absent = targets.clone()
    targets[1, 1], targets[2, 0], absent[1, 1], absent[2, 0] = v, 2 ** 31 - 1, -1, -1
    weights = torch.randn((4, 2), device="cuda")
    weights[2, 0] = 0
    r = scoring.log_probs(x, targets)
    grad = scoring.log_probs_grad(x, r, targets, grad_target=weights)
    assert torch.isnan(r.target[1, 1]) and torch.isnan(grad[1]).all()
    want = scoring.log_probs_grad(x, r, absent, grad_target=weights)
    for i in (0, 2, 3):
        assert torch.equal(grad[i], want[i])


def test_no_tangent_of_the_gradient(scoring):
    """A backward pass whose incoming gradients have tangents is refused; without them, beside them, it runs."""
    from torch.autograd import forward_ad

    from quiver import _lib

    say("log probs, forward over reverse")
    leaf = torch.randn((4, 50), device="cuda").requires_grad_()
    targets = torch.arange(4, dtype=torch.int32, device="cuda")
    weights = torch.rand((4, 1), device="cuda")
    with forward_ad.dual_level():
        r = scoring.log_probs(leaf, targets)
        with pytest.raises(_lib.QuiverError, match="forward-mode"):
            torch.autograd.grad((r.target * forward_ad.make_dual(weights, torch.ones_like(weights))).sum(), leaf)
        (grad,) = torch.autograd.grad((scoring.log_probs(leaf, targets).target * weights).sum(), leaf)
    with torch.no_grad():
        assert torch.equal(grad, scoring.log_probs_grad(leaf, scoring.log_probs(leaf, targets), targets, grad_target=weights))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [100, 5000, 40000])
def test_gradient_at_low_temperatures(scoring, dtype, v):
    """Weights over the temperature pass the largest float times a probability's logarithm: columns without a probability stay 0."""
    say("log probs, gradient at low temperatures", dtype, v)
    g = torch.Generator(device="cuda").manual_seed(v)
    x = torch.randn((5, v), generator=g, device="cuda") * 3
    x[1] = 12.7
    x[2, v // 2:] = -1e4
    x[3, 1:] = 29
    x[3, 0] = 30
    x[4, ::2] = -INF
    x = x.to(dtype)
    targets = torch.stack([x.argmax(1), x.argmin(1)], 1).to(torch.int32)
    for T in (1e-30, 1e-35, 1e-36, 1e-37):
        _run(scoring, x, targets, 12, T)


@pytest.fixture(autouse=True)
def nan_matches_nan_only(monkeypatch):
    """`_near` asks whether an error is above its bound, which a NaN never is: here, NaN is near to nothing else."""
    near = _near

    def strict(got, want, slack, what):
        assert not np.isnan(slack).any(), what
        np.testing.assert_array_equal(np.isnan(got.double().cpu().numpy()), np.isnan(want), err_msg=what)
        near(got, want, slack, what)

    monkeypatch.setattr(sys.modules[__name__], "_near", strict)
