"""Layer norm and its gradient against the formulas in 64 bits.

With u = 2^-24: a sum of a row's terms passes at most A = 64 + d / 1,024 additions (a thread's values, a wave's lanes, the
waves), so it is off by A u of the sum of magnitudes.  A deviation x - mean rounds twice; what is left of the mean is
off by A u of mean |x - mean|, at most the standard deviation s; the variance is off by (2 A + 8) u of itself, and its
root's reciprocal by half of that and 2 u.  So x^ is off by (A + 8) u |x^| + (A + 4) u, and y by that times |w| plus two
roundings of y's terms and the type's.  dx = (h - c1 - x^ c2) / s: its parts are off by (A + 2) u mean |h|, by (3 A + 20) u
of |x^| (mean |h x^| + mean |h|) and so on; (4 A + 40) u of the sum of the parts' magnitudes covers all.  The columns' sums pass
n / 256 + 400 additions at most (rows of a workgroup, their parts).  Types round once: 2^-24, 2^-8, 2^-11.
"""
from __future__ import annotations

from dataclasses import replace

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ROUND = {torch.float32: (U, 2.0 ** -149), torch.bfloat16: (2.0 ** -8, 2.0 ** -134), torch.float16: (2.0 ** -11, 2.0 ** -25)}
TYPES = list(ROUND)
EPS = 1e-5


@pytest.fixture(scope="module")
def scoring():
    from quiver import _lib, scoring

    if _lib.device_count() == 0:
        pytest.skip("no GPU")
    yield scoring
    torch.cuda.empty_cache()  # the memory is the other tests' again


def say(*a):
    print("[gpu]", *a, flush=True)


def _within(got, want, slack, name):
    rel, least = ROUND[got.dtype]
    assert got.shape == want.shape
    err, bound = (got.double() - want).abs(), slack + (want.abs() + slack) * rel + least
    assert (err <= bound).all(), (name, (err / bound).max().item())


def _moments(x, eps):
    v = x.double()
    mean = v.mean(1, keepdim=True)
    d = v - mean
    rstd = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + eps)
    return d * rstd, rstd


def _additions(d):
    return 64 + d / 1024


def _check_forward(y, x, weight, bias, eps=EPS):
    hat, _ = _moments(x, eps)
    a = _additions(x.shape[1])
    w = 1.0 if weight is None else weight.double()
    b = 0.0 if bias is None else bias.double()
    slack = ((a + 8) * U * hat.abs() + (a + 4) * U) * abs(w) + 2 * U * ((hat * w).abs() + abs(b))
    assert y.dtype == x.dtype
    _within(y, hat * w + b, slack, "y")


def _reference(x, g, weight, eps=EPS):
    hat, rstd = _moments(x, eps)
    h = g.double() * (1.0 if weight is None else weight.double())
    c1, c2 = h.mean(1, keepdim=True), (h * hat).mean(1, keepdim=True)
    return hat, rstd, h, rstd * (h - c1 - hat * c2)


def _check_grad(r, x, g, weight, dtype, eps=EPS):
    n, d = x.shape
    hat, rstd, h, dx = _reference(x, g, weight, eps)
    k = (4 * _additions(d) + 40) * U
    mean_h, mean_hx = h.abs().mean(1, keepdim=True), (h * hat).abs().mean(1, keepdim=True)
    parts = rstd * (h.abs() + mean_h + (hat.abs() + 1) * (mean_hx + mean_h))
    if r.x is not None:
        assert r.x.dtype == x.dtype
        _within(r.x, dx, k * parts, "dx")
    a, b = _additions(d), n / 256 + 400
    for got, terms, off in ((r.weight, g.double() * hat, (a + 8) * U * hat.abs() + (a + 4) * U), (r.bias, g.double(), None)):
        if got is None:
            continue
        assert got.dtype == dtype
        slack = b * U * terms.abs().sum(0)
        if off is not None:
            slack = slack + (g.double().abs() * off).sum(0)
        _within(got, terms.sum(0), slack, "columns")


def _rows(n, d, dtype, seed, offset=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((n, d), generator=g, device="cuda") * (torch.rand((n, 1), generator=g, device="cuda") * 2 + 0.1)
    x = (x + offset * torch.randn((n, 1), generator=g, device="cuda")).to(dtype)
    weight = 1 + 0.3 * torch.randn(d, generator=g, device="cuda")
    bias = 0.2 * torch.randn(d, generator=g, device="cuda")
    grad = (0.3 * torch.randn((n, d), generator=g, device="cuda")).to(dtype)
    return x, weight, bias, grad


# around each width that 4 to 1,024 threads hold by 3 or 4 vectors, odd widths, one and many rows, long rows
SIZES = [(1, 1), (3, 2), (5, 3), (700, 4), (9, 7), (1, 48), (33, 49), (17, 64), (1000, 65), (3, 96), (50, 97), (4097, 128),
         (31, 129), (20, 192), (257, 255), (1, 384), (100, 385), (64, 512), (5, 513), (1, 768), (300, 768), (77, 769),
         (40, 1001), (1030, 1024), (3, 1025), (9, 2049), (260, 3000), (7, 4095), (30, 4096), (2, 4097), (300, 5000),
         (5, 12288), (4, 12289), (3, 16384), (2, 16385), (5, 20001), (1, 100_003), (40_000, 33), (1100, 16385)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, d", SIZES)
def test_forward_and_gradient(scoring, dtype, n, d):
    say("layer norm", dtype, n, d)
    x, weight, bias, grad = _rows(n, d, dtype, n * 3 + d)
    for params in {torch.float32, dtype}:
        w, b = weight.to(params), bias.to(params)
        _check_forward(scoring.layer_norm(x, w, b), x, w, b)
        _check_grad(scoring.layer_norm_grad(x, grad, w), x, grad, w, params)
    if n * d < 100_000:
        _check_forward(scoring.layer_norm(x), x, None, None)
        _check_forward(scoring.layer_norm(x, w), x, w, None)
        _check_forward(scoring.layer_norm(x, None, b), x, None, b)
        _check_grad(scoring.layer_norm_grad(x, grad), x, grad, None, torch.float32)


@pytest.mark.parametrize("d", [5, 96, 769, 3001, 17001])
def test_wanted(scoring, d):
    """Each of the gradients by itself: the bits that it has with the others."""
    say("layer norm, gradients wanted", d)
    x, weight, _, grad = _rows(37, d, torch.float32, d)
    whole = scoring.layer_norm_grad(x, grad, weight)
    for wanted in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 0, 1), (0, 0, 0)):
        r = scoring.layer_norm_grad(x, grad, weight, wanted=wanted)
        for got, want, there in zip((r.x, r.weight, r.bias), (whole.x, whole.weight, whole.bias), wanted):
            assert torch.equal(got, want) if there else got is None


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, d", [(6, 8), (40, 768), (5, 2500), (3, 16400)])
def test_odd_rows(scoring, dtype, n, d):
    """Rows of equal values, of zeros, with a far offset, a single large value; infinities and NaN only take their row out."""
    say("layer norm, odd rows", dtype, n, d)
    x, weight, bias, grad = _rows(n, d, dtype, d)
    x[0] = 3
    x[1] = 0
    x[2] += 1000 if dtype == torch.float32 else 60
    x[2, d // 2] = 5000
    _check_forward(scoring.layer_norm(x, weight, bias), x, weight, bias)
    _check_grad(scoring.layer_norm_grad(x, grad, weight), x, grad, weight, torch.float32)
    clean = scoring.layer_norm(x, weight, bias)
    if n > 5:
        for row, value in ((3, float("inf")), (4, float("nan")), (5, -float("inf"))):
            x[row, row % d] = value
        y = scoring.layer_norm(x, weight, bias)
        r = scoring.layer_norm_grad(x, grad, weight)
        bad = torch.zeros(n, dtype=torch.bool, device="cuda")
        bad[3:6] = True
        assert torch.isnan(y[bad]).all() and torch.equal(y[~bad], clean[~bad])
        assert torch.isnan(r.x[bad]).all() and torch.isfinite(r.x[~bad]).all()
        assert torch.isnan(r.weight).all() and torch.isfinite(r.bias).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n, d", [(70, 7), (70, 100), (20, 1024), (9, 2048), (9, 4096), (5, 12000), (4, 20000)])
def test_huge_rows(scoring, dtype, n, d):
    """Values up to the type's largest among ordinary rows: their squares, and their sum, pass the largest float."""
    say("layer norm, huge rows", dtype, n, d)
    x, weight, bias, grad = _rows(n, d, torch.float32, d)
    big = torch.finfo(dtype).max
    x[1] = x[1].clamp(-1, 1) * big
    x[2] = big
    x[2, 0] = -big
    x[3] *= 2.0 ** 63
    x[n - 1, 1] = big / 2
    x, grad = x.to(dtype), grad.to(dtype)
    _check_forward(scoring.layer_norm(x, weight, bias), x, weight, bias)
    r = scoring.layer_norm_grad(x, grad, weight)
    hat, rstd, h, dx = _reference(x, grad, weight)
    parts = rstd * (h.abs() + h.abs().mean(1, keepdim=True) * (hat.abs() + 2) + (h * hat).abs().mean(1, keepdim=True) * (hat.abs() + 1))
    # 1 / s may be subnormal (down to 2^-128): its product rounds to 2^-149
    _within(r.x, dx, (4 * _additions(d) + 40) * U * parts + 2.0 ** -148 * (1 + parts / rstd), "dx")
    assert torch.isfinite(r.weight).all()
    _check_grad(replace(r, x=None), x, grad, weight, torch.float32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 1000, 70_001])
@pytest.mark.parametrize("d", [8, 15, 16, 17, 24, 31, 32, 33, 40, 47, 48, 50, 63, 64])
def test_short_rows(scoring, dtype, n, d):
    say("layer norm, short rows", dtype, n, d)
    x, weight, bias, grad = _rows(n, d, dtype, n + d)
    _check_forward(scoring.layer_norm(x, weight, bias), x, weight, bias)
    _check_grad(scoring.layer_norm_grad(x, grad, weight), x, grad, weight, torch.float32)


@pytest.mark.parametrize("value", [3e15, -2.0 ** 125, torch.finfo(torch.float32).max])
@pytest.mark.parametrize("d", [2, 7, 64, 100, 1000, 1024, 4096, 5000, 12288, 16384, 20000, 65536])
def test_equal_values(scoring, d, value):
    """Rows of one value, up to the largest: x^ is 0, and 1 / s that of eps alone.  Where d is a power of two the mean is
    exact.  Else what is left of the deviations is at most A u of that of the mean, and its root is taken of 2^-24 of the
    square of that at least: x^ is up to (A + 2) 2^-12, and s not eps's."""
    say("layer norm, equal values", d, value)
    x, weight, bias, grad = _rows(6, d, torch.float32, d)
    x[1:4] = value
    if d & (d - 1) == 0:
        _check_forward(scoring.layer_norm(x, weight, bias), x, weight, bias)
        _check_grad(scoring.layer_norm_grad(x, grad, weight), x, grad, weight, torch.float32)
    else:
        hat = scoring.layer_norm(x)[1:4]
        assert (hat.abs() <= (_additions(d) + 2) * 2.0 ** -12).all(), hat.abs().max()
        r = scoring.layer_norm_grad(x, grad, weight)
        assert torch.isfinite(r.x).all() and torch.isfinite(r.weight).all()


@pytest.mark.parametrize("eps", [2.0 ** -126, 1e-12, 1e-3, 10.0, 1e30])
def test_eps(scoring, eps):
    say("layer norm, eps", eps)
    x, weight, bias, grad = _rows(40, 300, torch.float32, 3)
    x[5] *= 1e-12
    if eps >= 1e-12:
        x[6] = 2  # 1 / s is 1e6 and more: what is left of the deviations is 0
    eps32 = torch.tensor(eps).item()
    _check_forward(scoring.layer_norm(x, weight, bias, eps=eps), x, weight, bias, eps32)
    _check_grad(scoring.layer_norm_grad(x, grad, weight, eps=eps), x, grad, weight, torch.float32, eps32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("off", [0, 1, 3])
def test_strides(scoring, dtype, off):
    """Rows inside wider matrices, at odd addresses; nothing beside the results is written."""
    say("layer norm, strides", dtype, off)
    for n, d in ((37, 100), (300, 17), (9, 768), (5, 3001), (3, 16387)):
        x, weight, bias, grad = _rows(n, d + 8, dtype, d)
        x, grad = x[:, off:off + d], grad[:, off:off + d]
        weight, bias = weight[off:off + d], bias[off:off + d]
        store = torch.full((n, d + 9), 7.0, dtype=dtype, device="cuda")
        y = scoring.layer_norm(x, weight, bias, out=store[:, off:off + d])
        _check_forward(y, x, weight, bias)
        assert (store[:, :off] == 7).all() and (store[:, off + d:] == 7).all()
        store.fill_(7.0)
        r = scoring.layer_norm_grad(x, grad, weight)
        again = type(r).of(store[:, off:off + d], r.weight, r.bias, r._workspace, r._made_for)
        first = r.x.clone(), r.weight.clone(), r.bias.clone()
        scoring.layer_norm_grad(x, grad, weight, out=again)
        _check_grad(again, x, grad, weight, torch.float32)
        assert (store[:, :off] == 7).all() and (store[:, off + d:] == 7).all()
        assert torch.equal(again.x, first[0]) and torch.equal(again.weight, first[1]) and torch.equal(again.bias, first[2])


@pytest.mark.parametrize("n, d", [(50, 40), (3000, 768), (300, 4000), (9, 20000)])
def test_in_place(scoring, n, d):
    """The result in x's place, and the gradient in x's or its own."""
    say("layer norm in place", n, d)
    x, weight, bias, grad = _rows(n, d, torch.bfloat16, d)
    y, r = scoring.layer_norm(x, weight, bias), scoring.layer_norm_grad(x, grad, weight)
    for place in ("x", "grad"):
        a, b = x.clone(), grad.clone()
        target = a if place == "x" else b
        out = type(r).of(target, torch.empty_like(r.weight), torch.empty_like(r.bias), r._workspace, r._made_for)
        scoring.layer_norm_grad(a, b, weight, out=out)
        assert torch.equal(target, r.x) and torch.equal(out.weight, r.weight) and torch.equal(out.bias, r.bias)
    assert torch.equal(scoring.layer_norm(x, weight, bias, out=x), y)


def test_empty(scoring):
    say("layer norm, no rows and no columns")
    w = torch.ones(8, device="cuda")
    assert scoring.layer_norm(torch.empty((0, 8), device="cuda"), w).shape == (0, 8)
    r = scoring.layer_norm_grad(torch.empty((0, 8), device="cuda"), torch.empty((0, 8), device="cuda"), w)
    assert r.x.shape == (0, 8) and (r.weight == 0).all() and (r.bias == 0).all()
    assert scoring.layer_norm(torch.empty((4, 0), device="cuda")).shape == (4, 0)
    r = scoring.layer_norm_grad(torch.empty((4, 0), device="cuda"), torch.empty((4, 0), device="cuda"))
    assert r.x.shape == (4, 0) and r.weight.shape == (0,)


def test_far_rows(scoring):
    """Rows past 2^31 elements from the first, and more rows than are taken at once."""
    n, d = 2_200_000, 1025
    say("layer norm, offsets past 31 bits")
    x = torch.empty((n, d), dtype=torch.bfloat16, device="cuda").normal_()
    grad = torch.empty_like(x).normal_()
    weight, bias = torch.rand(d, device="cuda") + 0.5, torch.rand(d, device="cuda")
    y, r = scoring.layer_norm(x, weight, bias), scoring.layer_norm_grad(x, grad, weight)
    for lo in (0, n // 2, n - 100):
        _check_forward(y[lo:lo + 100], x[lo:lo + 100], weight, bias)
        part = replace(r, x=r.x[lo:lo + 100], weight=None, bias=None)
        _check_grad(part, x[lo:lo + 100], grad[lo:lo + 100], weight, torch.float32)
    del y
    sums = torch.zeros(d, dtype=torch.float64, device="cuda")
    mass = torch.zeros_like(sums)
    for lo in range(0, n, 100_000):
        sums += grad[lo:lo + 100_000].double().sum(0)
        mass += grad[lo:lo + 100_000].double().abs().sum(0)
    _within(r.bias, sums, (n / 256 + 400) * U * mass, "columns")


def test_longest_rows(scoring):
    """Rows of the greatest length that is taken."""
    from quiver import _lib

    d = _lib.QV_LAYER_NORM_MAX_DIM
    say("layer norm, rows of", d)
    x, weight, bias, grad = _rows(3, d, torch.bfloat16, 4)
    _check_forward(scoring.layer_norm(x, weight, bias), x, weight, bias)
    _check_grad(scoring.layer_norm_grad(x, grad, weight), x, grad, weight, torch.float32)


def test_differences(scoring):
    """The gradient against central differences of the definition in 64 bits, along random directions."""
    say("layer norm, gradient against differences")
    for n, d in ((7, 5), (20, 96), (3, 2000)):
        x, weight, bias, grad = _rows(n, d, torch.float32, d)
        r = scoring.layer_norm_grad(x, grad, weight)
        g = torch.Generator(device="cuda").manual_seed(d)

        def loss(x, weight, bias):
            return ((_moments(x, EPS)[0] * weight + bias) * grad.double()).sum()

        parts = [t.double() for t in (x, weight, bias)]
        for at, got in enumerate((r.x, r.weight, r.bias)):
            along = torch.randn(parts[at].shape, generator=g, device="cuda", dtype=torch.float64)

            def slope(step):
                moved = [[p + s * step * along if i == at else p for i, p in enumerate(parts)] for s in (1, -1)]
                return (loss(*moved[0]) - loss(*moved[1])) / (2 * step)

            fine, coarse = slope(1e-4), slope(2e-4)
            # the difference's own error is a third of what halving the step changes, and rounding: 2^-50 of the losses' terms
            own = (fine - coarse).abs() + 2.0 ** -50 / 1e-4 * (grad.double().abs() * 10).sum()
            terms = (got.double() * along).abs().sum()
            assert ((got.double() * along).sum() - fine).abs() <= own + 4 * (4 * _additions(d) + 440) * U * 10 * terms


@pytest.mark.parametrize("dtype", TYPES)
def test_autograd(scoring, dtype):
    """Through autograd: the bits of layer_norm_grad, for any of the arguments, expanded gradients among them."""
    say("layer norm, autograd", dtype)
    x, weight, bias, grad = _rows(33, 100, dtype, 1)
    for params in {torch.float32, dtype}:
        w, b = weight.to(params), bias.to(params)
        want = scoring.layer_norm_grad(x, grad, w)
        for mask in range(1, 8):
            leaves = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, w, b))]
            y = scoring.layer_norm(*leaves)
            assert torch.equal(y, scoring.layer_norm(x, w, b)) and y.requires_grad
            y.backward(grad)
            for leaf, wanted in zip(leaves, (want.x, want.weight, want.bias)):
                assert torch.equal(leaf.grad, wanted) if leaf.requires_grad else leaf.grad is None
        leaf = x.clone().requires_grad_()
        scoring.layer_norm(leaf, w, b).sum().backward()  # a gradient of ones, expanded from one
        assert torch.equal(leaf.grad, scoring.layer_norm_grad(x, torch.ones_like(x), w).x)
        leaf = x.clone().requires_grad_()
        scoring.layer_norm(leaf).backward(grad)
        assert torch.equal(leaf.grad, scoring.layer_norm_grad(x, grad).x)
        leaf = b.clone().requires_grad_()
        scoring.layer_norm(x, None, leaf).backward(grad)
        assert torch.equal(leaf.grad, want.bias) and leaf.grad.dtype == params


def test_second_derivative_is_refused(scoring):
    from quiver import QuiverError

    say("layer norm, a second derivative")
    x, weight, bias, _ = _rows(5, 40, torch.float32, 2)
    x.requires_grad_()
    weight.requires_grad_()
    gx, gw = torch.autograd.grad(scoring.layer_norm(x, weight, bias).square().sum(), (x, weight), create_graph=True)
    for g in (gx, gw):
        with pytest.raises(QuiverError, match="cannot be differentiated again"):
            g.sum().backward(retain_graph=True)
    with pytest.raises(ValueError, match="out= cannot"):
        scoring.layer_norm(x, weight, bias, out=torch.empty_like(x))


def test_written_results_are_marked(scoring):
    """A result written again through out= counts as changed: a backward pass that needs the old one raises."""
    say("layer norm, results written again")
    x, weight, bias, grad = _rows(9, 30, torch.float32, 6)
    y = scoring.layer_norm(x, weight, bias)
    leaf = torch.ones((9, 30), device="cuda", requires_grad=True)
    product = (leaf * y).sum()
    scoring.layer_norm(x * 2, weight, bias, out=y)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.backward()


def test_streams_and_graphs(scoring):
    """On a stream of its own; captured and replayed, two graphs with results of their own in turn; equal calls, equal bits."""
    say("layer norm, streams and graphs")
    for n, d in ((3, 768), (5000, 100), (700, 2000), (20, 17000)):
        x, weight, bias, grad = _rows(n, d, torch.bfloat16, n)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            y, r = scoring.layer_norm(x, weight, bias), scoring.layer_norm_grad(x, grad, weight)
        side.synchronize()
        graphs = []
        for turn in range(2):
            out, back = torch.empty_like(y), scoring.layer_norm_grad(x, grad, weight)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                scoring.layer_norm(x, weight, bias, out=out)
                scoring.layer_norm_grad(x, grad, weight, out=back)
            graphs.append((graph, out, back))
        assert torch.equal(scoring.layer_norm(x, weight, bias), y)
        for turn in range(4):
            x.copy_(torch.randn((n, d), device="cuda"))
            graph, out, back = graphs[turn % 2]
            graph.replay()
            torch.cuda.synchronize()
            want = scoring.layer_norm_grad(x, grad, weight)
            assert torch.equal(out, scoring.layer_norm(x, weight, bias))
            assert torch.equal(back.x, want.x) and torch.equal(back.weight, want.weight) and torch.equal(back.bias, want.bias)


def test_embeddings_to_answers(scoring):
    """The run as it is used: layer norm, rows in 4 bits, their scores, log probabilities; and the gradients back to the norm's."""
    say("layer norm, 4-bit rows, scores, loss")
    g = torch.Generator(device="cuda").manual_seed(8)
    hidden = torch.randn((2000, 256), generator=g, device="cuda") * 3 + 1
    weight, bias = torch.rand(256, generator=g, device="cuda") + 0.5, torch.randn(256, generator=g, device="cuda") * 0.1
    vectors = scoring.layer_norm(hidden, weight, bias)
    _check_forward(vectors, hidden, weight, bias)
    catalogue = scoring.DenseCatalogue(vectors, bits=4)
    near = hidden[:64] + 0.05 * torch.randn((64, 256), generator=g, device="cuda")
    targets = torch.arange(64, dtype=torch.int32, device="cuda")
    r = catalogue.log_probs(scoring.layer_norm(near, weight, bias), targets, top_k=5, temperature=16.0)
    assert (r.top_ids[:, 0] == targets).all()  # an inner product with itself is 256 and more, with others about 16 +- 20
    leaf_w, leaf_b = weight.clone().requires_grad_(), bias.clone().requires_grad_()
    y = scoring.layer_norm(near, leaf_w, leaf_b)
    logits = y @ vectors[:500].T
    loss = -scoring.log_probs(logits, targets, temperature=16.0).target.mean()
    loss.backward()
    x64 = _moments(near, EPS)[0]
    w64, b64 = weight.double().requires_grad_(), bias.double().requires_grad_()
    z = (x64 * w64 + b64) @ vectors[:500].T.double() / 16
    (-torch.log_softmax(z, 1)[torch.arange(64), torch.arange(64)].mean()).backward()
    # logits of about 256 in sums of 256 products in fp32 are off by up to 2^-13 or so, probabilities by as much of themselves;
    # the targets' p - 1, about 2^-19 here, is a difference of numbers near 1, off by 2^-23 whatever its size: as much of
    # each target's vector (over 64 rows and the temperature) goes into the bias's gradient, times x^ into the weight's
    off = 2.0 ** -23 / (64 * 16) * vectors[:64].double().abs()
    for got, want, slack in ((leaf_w.grad, w64.grad, (off * x64.abs()).sum(0)), (leaf_b.grad, b64.grad, off.sum(0))):
        assert ((got.double() - want).abs() <= 2.0 ** -10 * want.abs().max() + slack).all()


def test_example(scoring):
    """The retrieval example runs, and its tower's gradients are those of the loss in 64 bits."""
    import importlib.util
    from pathlib import Path

    say("dense retrieval example, in 4 bits and with a layer norm")
    path = Path(__file__).resolve().parents[1] / "quiver-ae_amd" / "examples" / "dense_retrieval.py"
    spec = importlib.util.spec_from_file_location("dense_retrieval_tower", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    r = example.main(rows=4_000, queries=64, steps=2)
    assert len(r["tower_losses"]) == 2 and all(0 <= x < 100 for x in r["tower_losses"])
    assert 0 <= r["in_4_bits"]["recall"] <= 1 and r["in_4_bits"]["entropy"] >= 0

    g = torch.Generator(device="cuda").manual_seed(12)
    queries, vectors = torch.randn((40, 96), generator=g, device="cuda"), torch.randn((40, 96), generator=g, device="cuda")
    leaves = [torch.randn((96, 96), generator=g, device="cuda") * 0.1, 1 + 0.1 * torch.randn(96, generator=g, device="cuda"),
              0.1 * torch.randn(96, generator=g, device="cuda")]
    labels = torch.arange(40, dtype=torch.int32, device="cuda")
    for leaf in leaves:
        leaf.requires_grad_()
    example.tower_loss(queries, vectors, labels, *leaves).backward()
    exact = [t.detach().double().requires_grad_() for t in leaves]
    hidden = queries.double() @ exact[0]
    d = hidden - hidden.mean(1, keepdim=True)
    hat = d / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
    z = (hat * exact[1] + exact[2]) @ vectors.T.double() / (0.05 * 96 ** 0.5)
    (-torch.log_softmax(z, 1)[torch.arange(40), torch.arange(40)].mean()).backward()
    # logits over the temperature are at most 500 here, off by 100 roundings of 2^-24 of their 96 terms' magnitudes: 2^-9; each
    # gradient is a sum of probabilities (as much off, relatively) times values, and the loss's other sums' errors are far less
    for got, want in zip(leaves, exact):
        assert ((got.grad.double() - want.grad).abs() <= 2.0 ** -8 * want.grad.abs().max()).all()


def test_results_follow_their_memory(scoring):
    """Where a result's tensors were given other memory, a call writes to that and leaves the old alone; or it is refused."""
    say("layer norm, results in other memory")
    x, weight, _, grad = _rows(40, 96, torch.float32, 5)
    want, r = scoring.layer_norm_grad(x, grad, weight), scoring.layer_norm_grad(x, grad, weight)
    old = [t.detach() for t in (r.x, r.weight, r.bias)]
    for t in (r.x, r.weight, r.bias):
        t.data = torch.zeros_like(t)
    for t in old:
        t.fill_(7.0)
    assert scoring.layer_norm_grad(x, grad, weight, out=r) is r
    assert all((t == 7).all() for t in old)
    assert torch.equal(r.x, want.x) and torch.equal(r.weight, want.weight) and torch.equal(r.bias, want.bias)
    r.weight.data = r.weight.data.half()
    with pytest.raises(ValueError, match="out.weight must be"):
        scoring.layer_norm_grad(x, grad, weight, out=r)
    r.weight.data = torch.zeros(96)  # on the CPU
    with pytest.raises(ValueError, match="on one GPU"):
        scoring.layer_norm_grad(x, grad, weight, out=r)


def test_lent_buffers(scoring):
    """The gradient in x's place and in its own, with buffers of the caller's and one workspace for several results."""
    say("layer norm, lent buffers")
    for n, d in ((50, 40), (9, 20000)):
        x, weight, _, grad = _rows(n, d, torch.bfloat16, d)
        want = scoring.layer_norm_grad(x, grad, weight)
        made_for = (n, d, x.dtype, weight.dtype)
        shared = scoring.LayerNormGrad.workspace(n, d, x.device)
        for place in (0, 1):
            for workspace in (None, shared):
                a, b, dw, db = x.clone(), grad.clone(), torch.empty_like(weight), torch.empty_like(weight)
                r = scoring.LayerNormGrad.of((a, b)[place], dw, db, workspace, made_for)
                assert scoring.layer_norm_grad(a, b, weight, out=r) is r
                assert torch.equal((a, b)[place], want.x) and torch.equal(dw, want.weight) and torch.equal(db, want.bias)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n, d", [(70, 7), (70, 40), (70, 100), (20, 1000), (20, 2048), (12, 4096), (12, 12000), (10, 20000)])
def test_wide_gradients(scoring, dtype, n, d):
    """Gradients and deviations whose products no float holds, or loses, while their quotients are ordinary; other rows' bits stay."""
    say("layer norm, wide gradients", dtype, n, d)
    x, weight, _, grad = _rows(n, d, torch.float32, d + 1)
    plain = scoring.layer_norm_grad(x.to(dtype), grad.to(dtype), weight)
    for row, of_x, of_grad in ((0, 1e16, 1e22), (1, 1e18, 1e30), (2, 1.0, 1e33), (4, 1e-15, 1e-30), (6, 1e30, 1e-5), (7, 1e25, 1e27)):
        x[row] *= of_x
        grad[row] *= of_grad
    x[3] = x[3].clamp(-1, 1) * 3e38
    grad[3] *= 1e25
    x, grad = x.to(dtype), grad.to(dtype)
    r = scoring.layer_norm_grad(x, grad, weight)
    assert torch.isfinite(r.x).all() and torch.isfinite(r.weight).all()
    _check_grad(r, x, grad, weight, torch.float32)
    assert torch.equal(r.x[[5, 8, 9]], plain.x[[5, 8, 9]])
    # by themselves too: sums over rows of one size
    for row in (4, 6):
        _check_grad(scoring.layer_norm_grad(x[row:row + 1], grad[row:row + 1], weight), x[row:row + 1], grad[row:row + 1], weight,
                    torch.float32)


@pytest.mark.parametrize("d", [7, 100, 1000, 4096, 20000])
def test_small_gradients(scoring, d):
    """With an eps near the smallest float, gradients and deviations whose products are lost, while their quotients are not."""
    say("layer norm, small gradients", d)
    x, weight, _, grad = _rows(20, d, torch.float32, d + 2, offset=0.0)
    for eps, of_x, of_grad in ((2.0 ** -126, 1e-18, 1e-25), (2.0 ** -100, 1e-15, 1e-28), (2.0 ** -41, 1e-6, 1e-30)):
        _check_grad(scoring.layer_norm_grad(x * of_x, grad * of_grad, weight, eps=eps), x * of_x, grad * of_grad, weight,
                    torch.float32, eps)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, d", [(600_001, 16), (300_001, 64), (300_001, 33), (270_001, 100), (140_001, 250), (70_001, 384),
                                  (40_001, 768), (20_001, 1_500), (20_001, 2_000), (9_001, 2_999), (9_001, 4_000)])
def test_gradients_of_many_rows(scoring, dtype, n, d):
    """Workgroups of 256 threads, more rows than run at once: the bias's sums of whole numbers are exact, the weight's have terms
    of one sign in some columns, so that rows left out show."""
    say("layer norm, gradients of many rows", dtype, n, d)
    x, weight, _, grad = _rows(n, d, dtype, n + d)
    r = scoring.layer_norm_grad(x, grad, weight)
    _check_grad(r, x, grad, weight, torch.float32)
    g = torch.Generator(device="cuda").manual_seed(d)
    whole = torch.randint(-2, 6, (n, d), generator=g, device="cuda").to(dtype)  # sums of up to 3.6M: every partial one is exact
    signs = torch.sign(x.float() - x.float().mean(1, keepdim=True))
    r = scoring.layer_norm_grad(x, whole, weight)
    assert torch.equal(r.bias, whole.double().sum(0).float())
    _check_grad(replace(r, x=None, bias=None), x, whole, weight, torch.float32)
    # g of x^'s own sign: every term of the weight's gradient is positive, and their sum far from 0
    r = scoring.layer_norm_grad(x, signs.to(dtype), weight, wanted=(False, True, False))
    _check_grad(r, x, signs.to(dtype), weight, torch.float32)
    assert (r.weight > 0.3 * n).all()


def test_far_columns(scoring):
    """The columns' sums of rows past 2^31 elements from the first: whole numbers, and terms of one sign."""
    n, d = 2_200_000, 1025
    say("layer norm, columns of rows past 31 bits")
    x = torch.empty((n, d), dtype=torch.bfloat16, device="cuda").normal_()
    grad = torch.ones_like(x)
    r = scoring.layer_norm_grad(x, grad, wanted=(False, False, True))
    assert (r.bias == n).all()
    grad.copy_(torch.sign(x))
    r = scoring.layer_norm_grad(x, grad, wanted=(False, True, True))
    want = torch.zeros(2, d, dtype=torch.float64, device="cuda")
    mass = torch.zeros_like(want)
    for lo in range(0, n, 100_000):
        hat = _moments(x[lo:lo + 100_000], EPS)[0]
        g = grad[lo:lo + 100_000].double()
        want[0] += (g * hat).sum(0)
        mass[0] += (g * hat).abs().sum(0)
        want[1] += g.sum(0)
        mass[1] += g.abs().sum(0)
    assert (r.weight > 0.5 * n).all()
    a = _additions(d)
    # x^ is off by (a + 8) u |x^| + (a + 4) u, the sum by n / 256 + 400 additions
    _within(r.weight, want[0], ((n / 256 + 400) + a + 8) * U * mass[0] + (a + 4) * U * n, "weight")
    assert torch.equal(r.bias, want[1].float())
