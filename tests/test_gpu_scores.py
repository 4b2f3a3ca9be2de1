"""8-bit rows and their product against the definitions in 64 bits.

Quantised rows: x ((1 / a) 127) rounds three times in fp32 before it is rounded to
a whole number, so a code is at most 0.5 + 127 * 3 * 2^-24 from the real x 127 / a; a
scale rounds once.  Products: the sum of k products is a whole number; taken to fp32
and multiplied by two scales it rounds three times, the bias adds one rounding
of the result, the output type one more: 2^-24 of a float, 2^-8 of a bfloat16,
2^-11 of a float16 (2^-25 where it is subnormal).
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ROUND = {torch.float32: (U, 2.0 ** -149), torch.bfloat16: (2.0 ** -8, 2.0 ** -134), torch.float16: (2.0 ** -11, 2.0 ** -25)}
TYPES = list(ROUND)


@pytest.fixture(scope="module")
def scoring():
    from quiver import _lib, scoring

    if _lib.device_count() == 0:
        pytest.skip("no GPU")
    yield scoring
    torch.cuda.empty_cache()  # the memory is the other tests' again


def say(*a):
    print("[gpu]", *a, flush=True)


def _check_rows(x, codes, scales):
    v = x.double().cpu().numpy()
    c, s = codes.cpu().numpy().astype(np.float64), scales.double().cpu().numpy()
    assert codes.dtype == torch.int8 and codes.shape == x.shape and scales.shape == (x.shape[0],)
    a = np.abs(v).max(1, initial=0.0)
    none = a < 2.0 ** -119
    assert (s[none] == 0).all() and (c[none] == 0).all()
    some = ~none
    np.testing.assert_allclose(s[some], a[some] / 127, rtol=U)
    assert (np.abs(v[some] * 127 / a[some][:, None] - c[some]) <= 0.5 + 127 * 3 * U).all()
    if x.shape[1]:
        assert (np.abs(c[some]).max(1) == 127).all()


# around each width that a group of lanes holds, odd widths, one and many rows
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, d", [(1, 1), (3, 2), (5, 7), (1, 16), (17, 32), (33, 33), (257, 64), (16, 96), (100, 100),
                                  (1001, 128), (65, 129), (31, 200), (9, 256), (7, 384), (40, 511), (12, 769), (5, 1024),
                                  (3, 2049), (4, 4096), (2, 8197), (1, 40003), (70001, 3)])
def test_quantize(scoring, dtype, n, d):
    say("quantize", dtype, n, d)
    g = torch.Generator(device="cuda").manual_seed(n * 7 + d)
    x = (torch.randn((n, d), generator=g, device="cuda") * torch.rand((n, 1), generator=g, device="cuda") * 5).to(dtype)
    x[n // 2] *= 1e-3
    codes, scales = scoring.quantize_rows(x)
    _check_rows(x, codes, scales)


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_odd_rows(scoring, dtype):
    """Zeros, subnormal and huge rows, infinities and NaN, halves, minus the largest."""
    say("quantize odd rows", dtype)
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).tiny
    for d in (5, 128, 1030):
        x = torch.randn((10, d), device="cuda").to(dtype)
        x[0] = 0
        x[1] = -0.0
        x[2] = tiny / 4
        x[3, 1] = big
        x[4] = -big
        x[5, d - 1] = float("inf")
        x[6, 0] = float("nan")
        x[7, 2] = -float("inf")
        x[8] = torch.arange(d, device="cuda").to(dtype) % 128 - 0.5
        x[8, 0] = 127
        codes, scales = scoring.quantize_rows(x)
        odd = torch.tensor([5, 6, 7], device="cuda")
        assert torch.isnan(scales[odd]).all() and (codes[odd] == 0).all()
        fine = torch.tensor([0, 1, 2, 3, 4, 8, 9], device="cuda")
        _check_rows(x[fine], codes[fine], scales[fine])
        # halves go to the even neighbour ((1 / 127) 127 is 1 in fp32, so the products are exact)
        np.testing.assert_array_equal(codes[8].cpu().numpy(), np.rint(x[8].float().cpu().numpy()).astype(np.int8))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("off", [0, 1, 3])
def test_quantize_strides(scoring, dtype, off):
    """Rows and codes inside wider matrices, at odd addresses; nothing beside them is written."""
    say("quantize strides", dtype, off)
    g = torch.Generator(device="cuda").manual_seed(off)
    for n, d, wide in ((37, 100, 131), (5, 768, 800), (300, 16, 19), (3, 2500, 2503)):
        x = torch.randn((n, wide), generator=g, device="cuda").to(dtype)[:, off:off + d]
        store = torch.full((n, wide + 5), 99, dtype=torch.int8, device="cuda")
        codes, scales = scoring.quantize_rows(x, out=(store[:, off:off + d], torch.empty(n, device="cuda")))
        _check_rows(x, codes, scales)
        assert (store[:, :off] == 99).all() and (store[:, off + d:] == 99).all()


def test_quantize_empty(scoring):
    say("quantize, no rows and no columns")
    codes, scales = scoring.quantize_rows(torch.empty((0, 8), device="cuda"))
    assert codes.shape == (0, 8) and scales.shape == (0,)
    codes, scales = scoring.quantize_rows(torch.empty((4, 0), device="cuda"))
    assert codes.shape == (4, 0) and (scales == 0).all()


def _inputs(m, n, k, seed, extreme=False, wide=0, off=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def codes(rows):
        c = torch.randint(-128, 128, (rows, k + wide), generator=g, device="cuda")
        if extreme:
            c = torch.where(c < 0, -128, 127)
        return c.to(torch.int8)[:, off:off + k]

    return (codes(m), torch.rand(m, generator=g, device="cuda") * 0.1 + 1e-3, codes(n),
            torch.rand(n, generator=g, device="cuda") * 0.1 + 1e-3, torch.randn(n, generator=g, device="cuda"))


def _check_product(out, a, sa, b, sb, bias, dtype):
    dots = (a.double() @ b.double().contiguous().T).cpu().numpy()  # whole numbers below 2^53: exact
    want = dots * sa.double().cpu().numpy()[:, None] * sb.double().cpu().numpy()[None, :]
    rel, least = ROUND[dtype]
    slack = 3 * U * np.abs(want)
    if bias is not None:
        want = want + bias.double().cpu().numpy()
        finite = np.isfinite(want)
        slack = slack + U * np.where(finite, np.abs(want), 0)
    got = out.double().cpu().numpy()
    assert out.dtype == dtype and got.shape == want.shape
    finite = np.isfinite(want)
    np.testing.assert_array_equal(got[~finite], want[~finite])
    # one rounding to the type on top, of a value that is itself off by the slack
    bound = slack + (np.where(finite, np.abs(want), 0) + slack) * rel + least
    err = np.abs(np.where(finite, got - np.where(finite, want, 0), 0))
    assert (err <= bound).all(), (err / bound).max()


# m and n around the tiles of 16, 32, 64, 128 and 256, k around the steps of 16, 32, 64 and 128 bytes
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m, n, k", [
    (1, 1, 1), (1, 1, 16), (1, 1000, 128), (2, 77, 5), (3, 129, 15), (16, 300, 96), (17, 31, 17), (31, 257, 100),
    (32, 512, 128), (33, 513, 129), (64, 64, 64), (65, 127, 200), (100, 1001, 33), (127, 255, 256), (128, 128, 1024),
    (129, 300, 31), (255, 257, 144), (256, 256, 384), (300, 200, 1000), (511, 513, 112), (1, 5000, 4096), (20, 700, 2049),
    (600, 700, 769), (1030, 2100, 260), (33, 70, 320), (200, 900, 4096), (1000, 3000, 576), (130, 20000, 640),
    (1500, 3300, 384), (1500, 3300, 1001), (100, 900, 4001), (4096, 3329, 2048)])
def test_product(scoring, dtype, m, n, k):
    say("product", dtype, m, n, k)
    a, sa, b, sb, bias = _inputs(m, n, k, m * 31 + n * 7 + k)
    if dtype == torch.float16:  # within its range
        sa, sb = sa * 0.05, sb * 0.05
    _check_product(scoring.int8_product(a, sa, b, sb, dtype=dtype), a, sa, b, sb, None, dtype)
    bias[::7] = -float("inf")
    _check_product(scoring.int8_product(a, sa, b, sb, bias=bias, dtype=dtype), a, sa, b, sb, bias, dtype)


# 470 to 770 tiles of 256, which a workgroup takes two or three of; stages of 64 bytes in every remainder of 4
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m, n, k, bias", [(260, 60001, 320, True), (300, 60160, 384, False), (257, 98000, 448, True),
                                           (512, 60000, 512, False), (513, 61000, 576, True)])
def test_product_many_tiles(scoring, dtype, m, n, k, bias):
    say("product", dtype, m, n, k, bias)
    a, sa, b, sb, add = _inputs(m, n, k, m + n + k)
    out = scoring.int8_product(a, sa, b, sb, bias=add if bias else None, dtype=dtype)
    _check_product(out, a, sa, b, sb, add if bias else None, dtype)


# each way that a product takes
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m, n, k", [(5, 3000, 9), (5, 3000, 100), (20, 700, 2049), (100, 3000, 128), (100, 3001, 200),
                                     (64, 4096, 1024), (700, 4000, 1024), (512, 60000, 512), (100, 900, 4001),
                                     (1500, 3300, 1001)])
def test_product_bits(scoring, dtype, m, n, k):
    """Exact sums, then fp32 in the written order and one rounding to the type: the same bits from every kernel."""
    say("product, bits", dtype, m, n, k)
    a, sa, b, sb, bias = _inputs(m, n, k, m + 3 * n + 5 * k)
    sa = sa * 0.05
    want = ((a.double() @ b.double().T.contiguous()).float() * sa[:, None]) * sb[None, :]
    assert torch.equal(scoring.int8_product(a, sa, b, sb, dtype=dtype), want.to(dtype))
    assert torch.equal(scoring.int8_product(a, sa, b, sb, bias=bias, dtype=dtype), (want + bias[None, :]).to(dtype))


@pytest.mark.parametrize("m, n, k", [(1, 40, 131071), (40, 70, 131071), (300, 300, 131071)])
def test_product_largest_sums(scoring, m, n, k):
    """Every product 127^2, -127 128 or 128^2: sums just inside 32 bits."""
    say("product, largest sums", m, n, k)
    a, sa, b, sb, _ = _inputs(m, n, k, 5, extreme=True)
    a[0], b[0] = -128, -128
    out = scoring.int8_product(a, sa, b, sb)
    _check_product(out, a, sa, b, sb, None, torch.float32)
    assert a[0].double().dot(b[0].double()) == 2 ** 31 - 2 ** 14


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m, n, k, wide, off", [(5, 300, 100, 28, 4), (70, 90, 96, 31, 1), (300, 290, 128, 16, 16),
                                               (260, 515, 257, 3, 3), (1, 600, 768, 5, 2)])
def test_product_strides(scoring, dtype, m, n, k, wide, off):
    """Operands and output inside wider matrices, at odd addresses; nothing beside the output is written."""
    say("product strides", dtype, m, n, k, wide, off)
    a, sa, b, sb, _ = _inputs(m, n, k, k, wide=wide, off=off)
    sa, sb = sa * 0.05, sb * 0.05
    store = torch.full((m, n + off + 9), 7.0, dtype=dtype, device="cuda")
    out = scoring.int8_product(a, sa, b, sb, out=store[:, off:off + n])
    _check_product(out, a, sa, b, sb, None, dtype)
    assert (store[:, :off] == 7).all() and (store[:, off + n:] == 7).all()


def test_product_empty_and_odd_scales(scoring):
    """No rows, no columns, rows of no length; a row or column whose scale is NaN, an infinity or 0."""
    say("product, empty sizes and odd scales")
    a, sa, b, sb, bias = _inputs(40, 50, 64, 3)
    assert scoring.int8_product(a[:0], sa[:0], b, sb).shape == (0, 50)
    assert scoring.int8_product(a, sa, b[:0], sb[:0]).shape == (40, 0)
    out = scoring.int8_product(a[:, :0], sa, b[:, :0], sb, bias=bias)
    assert torch.equal(out, bias.expand(40, 50))
    sa[3], sb[4], sa[5] = float("nan"), float("nan"), 0.0
    out = scoring.int8_product(a, sa, b, sb)
    assert torch.isnan(out[3]).all() and torch.isnan(out[:, 4]).all()
    fine = torch.ones(50, dtype=torch.bool, device="cuda")
    fine[4] = False
    assert (out[5][fine] == 0).all() and torch.isfinite(out[0][fine]).all()


def test_long_catalogue(scoring):
    """Rows, and outputs, past 2^31 bytes from the first."""
    say("product, offsets past 31 bits")
    n, k = 17_000_000, 130
    b = torch.randint(-128, 128, (n, k), dtype=torch.int8, device="cuda")
    sb = torch.full((n,), 0.01, device="cuda")
    a, sa = b[[0, n // 2, n - 1]].contiguous(), torch.ones(3, device="cuda")
    out = scoring.int8_product(a, sa, b, sb)
    for lo in (0, n // 2 - 50, n - 100):
        _check_product(out[:, lo:lo + 100], a, sa, b[lo:lo + 100], sb[lo:lo + 100], None, torch.float32)
    a = a.repeat(24, 1)[:70].contiguous()
    out = scoring.int8_product(a, torch.ones(70, device="cuda"), b, sb, dtype=torch.bfloat16)  # 2.4 GB
    for lo in (0, n // 2 - 50, n - 100):
        _check_product(out[:, lo:lo + 100], a, torch.ones(70, device="cuda"), b[lo:lo + 100], sb[lo:lo + 100], None,
                       torch.bfloat16)


def test_many_rows(scoring):
    """More rows, and more tiles, than one launch is given."""
    n = 2 ** 30 + 300
    say("quantize,", n, "rows")
    x = torch.full((n, 1), 2.0, dtype=torch.bfloat16, device="cuda")
    x[::3] = -1
    codes, scales = scoring.quantize_rows(x)
    negative = x[:, 0] < 0
    assert (codes[:, 0] == torch.where(negative, -127, 127).to(torch.int8)).all()
    one = torch.tensor([1 / 127, 2 / 127], device="cuda")
    assert ((scales - torch.where(negative, one[0], one[1])).abs() <= 2 ** -30).all()  # 2^-24 of 2 / 127
    del x, codes, scales, negative
    m, n, k = 46_400, 46_403, 3
    say("product,", m, n, k)
    a = torch.randint(-128, 128, (m, k), dtype=torch.int8, device="cuda")
    b = torch.randint(-128, 128, (n, k), dtype=torch.int8, device="cuda")
    sa, sb = torch.rand(m, device="cuda"), torch.rand(n, device="cuda")
    out = scoring.int8_product(a, sa, b, sb, dtype=torch.float16)
    for lo in (0, m // 2, m - 100):
        _check_product(out[lo:lo + 100], a[lo:lo + 100], sa[lo:lo + 100], b, sb, None, torch.float16)


def test_other_stream_and_order(scoring):
    """Calls follow the current stream's order, and equal calls give equal bits."""
    say("scores on a stream of their own")
    x = torch.randn((5000, 300), device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y = x * 3
        codes, scales = scoring.quantize_rows(y)
        s = scoring.int8_product(codes[:64], scales[:64], codes, scales, dtype=torch.bfloat16)
    side.synchronize()
    _check_rows(y, codes, scales)
    _check_product(s, codes[:64], scales[:64], codes, scales, None, torch.bfloat16)
    assert torch.equal(s, scoring.int8_product(codes[:64], scales[:64], codes, scales, dtype=torch.bfloat16))


def test_in_a_graph(scoring):
    """Captured calls of every kernel of the product give what eager calls give, replay after replay."""
    say("scores in a graph")
    for m, n, k in ((5, 3000, 96), (5, 300, 1024), (200, 1000, 100), (200, 900, 512), (1000, 3000, 640), (300, 700, 333),
                    (4096, 3329, 2048), (40, 40, 7)):
        g = torch.Generator(device="cuda").manual_seed(k)
        x = torch.randn((m, k), generator=g, device="cuda")
        b, sb = scoring.quantize_rows(torch.randn((n, k), generator=g, device="cuda"))
        codes = scoring.quantize_rows(x)
        out = scoring.int8_product(*codes, b, sb, dtype=torch.bfloat16)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            scoring.quantize_rows(x, out=codes)
            scoring.int8_product(*codes, b, sb, out=out)
        for turn in range(3):
            x.copy_(torch.randn((m, k), generator=g, device="cuda"))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, scoring.int8_product(*scoring.quantize_rows(x.clone()), b, sb, dtype=torch.bfloat16))


def test_distant_rows_of_scores(scoring):
    """Output rows 2^27 elements and more apart, by each way that a product takes; nothing beside the output is written."""
    rows, stride = 256, 2 ** 27 + 3
    store = torch.empty(rows * stride, dtype=torch.bfloat16, device="cuda")  # 69 GB
    for m, n, k in ((1, 300, 96), (3, 3000, 100), (32, 200, 2049), (40, 3000, 100), (100, 1001, 200), (100, 900, 301),
                    (64, 500, 320), (200, 700, 4096), (256, 56000, 320), (5, 70, 9)):
        say("product, distant rows of scores", m, n, k)
        a, sa, b, sb, bias = _inputs(m, n, k, k)
        wide = store.as_strided((m, n + 16), (stride, 1))
        wide.fill_(7.0)
        out = scoring.int8_product(a, sa, b, sb, bias=bias, out=wide[:, 5:5 + n])
        _check_product(out, a, sa, b, sb, bias, torch.bfloat16)
        assert (wide[:, :5] == 7).all() and (wide[:, 5 + n:] == 7).all()


@pytest.mark.parametrize("m, n, k", [(1, 70, 40), (20, 70, 300), (40, 50, 40), (40, 50, 300)])
def test_distant_rows_of_codes(scoring, m, n, k):
    """Operands' rows 2^23 elements and more apart."""
    say("product, distant rows of codes", m, n, k)
    a, sa, b, sb, bias = _inputs(m, n, k, k)
    stride = 2 ** 23 + 5
    store = torch.empty((m + n) * stride, dtype=torch.int8, device="cuda")
    far_a, far_b = store.as_strided((m, k), (stride, 1)), store.as_strided((n, k), (stride, 1), m * stride)
    far_a.copy_(a)
    far_b.copy_(b)
    want = scoring.int8_product(a, sa, b, sb, bias=bias)
    for x, y in ((far_a, b), (a, far_b), (far_a, far_b)):
        assert torch.equal(scoring.int8_product(x, sa, y, sb, bias=bias), want)
    _check_product(want, a, sa, b, sb, bias, torch.float32)


def test_one_query_of_a_huge_catalogue(scoring):
    """2^27 rows and more take the time of a few less (three times it at most: it was seven times where they took another way)."""
    k, most = 16, 2 ** 27 + 77
    say("product, one query,", most, "rows")
    b = torch.randint(-128, 128, (most, k), dtype=torch.int8, device="cuda")
    sb = torch.rand(most, device="cuda")
    a, sa = b[most - 2:most - 1].clone(), torch.ones(1, device="cuda")

    def timed(n):
        out = scoring.int8_product(a, sa, b[:n], sb[:n], dtype=torch.bfloat16)
        for lo in (0, n // 2 - 50, n - 100):
            _check_product(out[:, lo:lo + 100], a, sa, b[lo:lo + 100], sb[lo:lo + 100], None, torch.bfloat16)
        times = []
        for _ in range(5):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            scoring.int8_product(a, sa, b[:n], sb[:n], out=out)
            end.record()
            end.synchronize()
            times.append(start.elapsed_time(end))
        return min(times)

    under, over = timed(2 ** 27 - 77), timed(most)
    say(f"{under * 1e3:.0f} us below 2^27 rows, {over * 1e3:.0f} us above")
    assert over < 3 * under


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n, d", [(3000, 7), (400, 100), (30, 3000)])
def test_quantize_huge_rows(scoring, dtype, n, d):
    """Entries all over the type's range: codes as near to x 127 / a as anywhere, though 1 / a is subnormal."""
    say("quantize huge rows", dtype, n, d)
    g = torch.Generator(device="cuda").manual_seed(d)
    big = torch.finfo(dtype).max
    x = ((torch.rand((n, d), generator=g, device="cuda") * 2 - 1) * big).to(dtype)
    # near halves, where the reciprocal's last bits decide the code
    halves = torch.arange(d, device="cuda") % 127 + 0.5
    a = (torch.rand(n // 2, generator=g, device="cuda") * 0.74 + 0.25) * big
    x[:n // 2] = (halves * (a[:, None] / 127)).to(dtype)
    x[:n // 2, 0] = a
    if dtype == torch.float32:  # the largest errors of a search over rows
        for i, (top, value) in enumerate((("0x1.fb2cd8p+127", "0x1.f52f4cp+127"), ("0x1.f82df6p+127", "0x1.f631dap+127"),
                                          ("0x1.f40ffcp+127", "0x1.ee27f2p+127"))):
            x[i] = 0
            x[i, 1], x[i, d - 1] = float.fromhex(value), -float.fromhex(top)
    codes, scales = scoring.quantize_rows(x)
    _check_rows(x, codes, scales)
