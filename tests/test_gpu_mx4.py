"""Rows in microscaled 4-bit floating point and their product against the definitions in 64 bits.

Quantised rows: scaling by a power of two is exact and the rounding is to the nearest of eight magnitudes, so codes
and scales equal the definition's.  Products: two codes and two powers of two multiply exactly.  A matrix instruction
adds 64 (or 128) products to a running sum; with every addition off by at most a unit in the last place (2^-23 of a
partial sum, whether it rounds or cuts), a sum of k products is off by at most (128 + k / 64 + what joins partial sums,
16) 2^-23 of the sum of magnitudes.  The bias adds 2^-24 of the result, the output type its rounding: 2^-8 of a
bfloat16, 2^-11 of a float16 (2^-25 where it is subnormal).  Where scales are close to each other every partial sum is
a whole number of units below 2^24: then the result is exact to the last bit.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ROUND = {torch.float32: (U, 2.0 ** -149), torch.bfloat16: (2.0 ** -8, 2.0 ** -134), torch.float16: (2.0 ** -11, 2.0 ** -25)}
TYPES = list(ROUND)
GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


@pytest.fixture(scope="module")
def scoring():
    from quiver import _lib, scoring

    if _lib.device_count() == 0:
        pytest.skip("no GPU")
    yield scoring
    torch.cuda.empty_cache()  # the memory is the other tests' again


def say(*a):
    print("[gpu]", *a, flush=True)


def reference_rows(x):
    """(codes [n, d], scales [n, blocks]) of the definition, in 64 bits."""
    v = x.double().cpu().numpy()
    n, d = v.shape
    blocks = -(-d // 32)
    v = np.pad(v, ((0, 0), (0, blocks * 32 - d))).reshape(n, blocks, 32)
    bad = ~np.isfinite(v).all(2)
    top = np.where(bad, 0, np.abs(np.where(np.isfinite(v), v, 0)).max(2))
    e = np.full(top.shape, -127)
    some = top > 7 * 2.0 ** -127
    m, exponent = np.frexp(top[some] / 7)  # m 2^exponent with m in [1/2, 1): the least power of two above or at it
    e[some] = np.where(m == 0.5, exponent - 1, exponent)
    y = np.where(bad[:, :, None], 0, np.where(np.isfinite(v), v, 0) / 2.0 ** e[:, :, None])
    distance = np.abs(np.abs(y)[..., None] - GRID)
    # of two at the same distance the even code
    code = np.argmin(distance + np.where(np.arange(8) % 2, 1e-9, 0) * (distance == distance.min(-1, keepdims=True)), -1)
    code = code + np.where(np.signbit(y) & ~bad[:, :, None], 8, 0)
    return code.reshape(n, -1)[:, :d], np.where(bad, 255, e + 127)


def unpack(codes, d):
    c = codes.cpu().numpy()
    both = np.stack([c & 15, c >> 4], 2).reshape(c.shape[0], -1)
    assert (both[:, d:] == 0).all()  # a row of odd length ends with a zero code
    return both[:, :d]


def values_of(codes, scales, d):
    """What rows stand for, in 64 bits, on their device."""
    c = torch.stack([codes & 15, codes >> 4], 2).reshape(codes.shape[0], -1)[:, :d]
    grid = torch.tensor(np.concatenate([GRID, -GRID]), device=codes.device)
    s = torch.where(scales == 255, torch.nan, torch.exp2(scales.double() - 127))
    return grid[c.long()] * s.repeat_interleave(32, 1)[:, :d]


def _check_rows(x, codes, scales):
    n, d = x.shape
    assert codes.dtype == scales.dtype == torch.uint8
    assert codes.shape == (n, (d + 1) // 2) and scales.shape == (n, (d + 31) // 32)
    want, s = reference_rows(x)
    np.testing.assert_array_equal(scales.cpu().numpy(), s)
    np.testing.assert_array_equal(unpack(codes, d), want)


# around the blocks of 32 and the lanes' eights, odd lengths, one and many rows, rows longer than a workgroup's run
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, d", [(1, 1), (3, 2), (5, 7), (1, 8), (9, 9), (1, 31), (17, 32), (33, 33), (257, 64), (16, 96),
                                  (100, 100), (1001, 128), (65, 129), (9, 255), (7, 384), (12, 769), (5, 1024), (3, 8199),
                                  (2, 40003), (70001, 3), (1, 1_100_001)])
def test_quantize(scoring, dtype, n, d):
    say("4-bit rows", dtype, n, d)
    g = torch.Generator(device="cuda").manual_seed(n * 7 + d)
    x = (torch.randn((n, d), generator=g, device="cuda") * torch.rand((n, 1), generator=g, device="cuda") * 5).to(dtype)
    x[n // 2] *= 1e-3
    codes, scales = scoring.quantize_rows_mx4(x)
    _check_rows(x, codes, scales)
    values = scoring.mx4_values(codes, scales, d, dtype=dtype)
    assert torch.equal(values, values_of(codes, scales, d).to(dtype))
    # no value is off by more than half a step: a sixth of the largest code above, or half a step of the lowest codes
    step = torch.exp2(scales.double() - 127).repeat_interleave(32, 1)[:, :d]
    if dtype != torch.float16:
        assert ((x.double() - values.double()).abs() <= step).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_borders(scoring, dtype):
    """Values on, below and above every border between codes; largest values around 7 times a power of two."""
    say("4-bit rows, borders", dtype)
    middle = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda")
    eps = torch.finfo(dtype).eps
    v = torch.cat([middle * f for f in (1 - eps / 2, 1, 1 + eps)] + [torch.tensor([0.0, -0.0, 0.5, 1, 1.5, 2, 3, 4], device="cuda")])
    v = torch.cat([v, -v[:2], torch.tensor([6.0], device="cuda")])
    assert v.numel() == 32
    rows = [v, -v, v.flip(0)]
    for top in (6, 7 * (1 - eps / 2), 7, 7 * (1 + eps), 8, 3.5, 3.5 * (1 + eps), 4):
        r = v.clamp(-3, 3) * min(1, top / 8)
        r[11] = top
        rows.append(r)
    x = torch.stack(rows)
    x = torch.cat([x * 2.0 ** e for e in (0, -9, 11)]).to(dtype)
    codes, scales = scoring.quantize_rows_mx4(x)
    _check_rows(x, codes, scales)


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_odd_rows(scoring, dtype):
    """Zeros, subnormal and huge blocks, infinities and NaN, which only take their own block out."""
    say("4-bit rows, odd values", dtype)
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).tiny
    for d in (5, 128, 1031):
        g = torch.Generator(device="cuda").manual_seed(d)
        x = torch.randn((10, d), generator=g, device="cuda").to(dtype)
        x[0] = 0
        x[1] = -0.0
        x[2] *= tiny
        x[3, 1] = big
        x[4] = -big
        x[5, d - 1] = float("inf")
        x[6, 0] = float("nan")
        x[7, 2] = -float("inf")
        x[8] = tiny / 16
        codes, scales = scoring.quantize_rows_mx4(x)
        _check_rows(x, codes, scales)
        assert scales[5, -1] == 255 and (scales[5, :-1] < 255).all()
        values = scoring.mx4_values(codes, scales, d)
        want = values_of(codes, scales, d).float()  # (the largest float rounds to 4 2^126, an infinity in float)
        assert torch.equal(torch.isnan(values), torch.isnan(want))
        assert torch.equal(values.nan_to_num(0.0), want.nan_to_num(0.0))


def test_every_code(scoring):
    """Every code under every scale."""
    say("4-bit rows, every code and scale")
    codes = torch.arange(16, dtype=torch.uint8, device="cuda").repeat(256, 1)
    codes = codes | (codes.flip(1) << 4)
    scales = torch.arange(256, dtype=torch.uint8, device="cuda")[:, None]
    for dtype in TYPES:
        got = scoring.mx4_values(codes, scales, dtype=dtype)
        want = values_of(codes, scales, 32).float().to(dtype)  # (float holds each: 6 2^127 as an infinity)
        assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0)) and torch.equal(torch.isnan(got), torch.isnan(want))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("off", [0, 1, 3])
def test_quantize_strides(scoring, dtype, off):
    """Rows, codes and scales inside wider matrices, at odd addresses; nothing beside them is written."""
    say("4-bit rows, strides", dtype, off)
    g = torch.Generator(device="cuda").manual_seed(off)
    for n, d, wide in ((37, 100, 131), (5, 768, 800), (300, 17, 20), (3, 2501, 2504)):
        x = torch.randn((n, wide), generator=g, device="cuda").to(dtype)[:, off:off + d]
        cols, blocks = (d + 1) // 2, (d + 31) // 32
        store = torch.full((n, cols + 7), 99, dtype=torch.uint8, device="cuda")
        marks = torch.full((n, blocks + 5), 77, dtype=torch.uint8, device="cuda")
        out = store[:, off:off + cols], marks[:, off:off + blocks]
        codes, scales = scoring.quantize_rows_mx4(x, out=out)
        _check_rows(x, codes, scales)
        assert (store[:, :off] == 99).all() and (store[:, off + cols:] == 99).all()
        assert (marks[:, :off] == 77).all() and (marks[:, off + blocks:] == 77).all()
        beside = torch.full((n, d + 9), 5.0, dtype=dtype, device="cuda")
        values = scoring.mx4_values(codes, scales, d, out=beside[:, off:off + d])
        assert torch.equal(values, values_of(codes, scales, d).to(dtype))
        assert (beside[:, :off] == 5).all() and (beside[:, off + d:] == 5).all()


def test_quantize_empty(scoring):
    say("4-bit rows, none and of no length")
    for n, d in ((0, 8), (4, 0)):
        codes, scales = scoring.quantize_rows_mx4(torch.empty((n, d), device="cuda"))
        assert codes.shape == (n, d // 2) and scales.shape == (n, d // 32 + (d > 0))
        assert scoring.mx4_values(codes, scales).shape == (n, d)


def _inputs(m, n, k, seed, near=False, wide=0, off=0):
    """Codes of rows of k values and their scales; near: scales of 1/2 and 1."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    cols, blocks = (k + 1) // 2, (k + 31) // 32

    def side(rows):
        codes = torch.randint(0, 256, (rows, cols + wide), generator=g, device="cuda").to(torch.uint8)
        scales = torch.randint(126 if near else 112, 128 if near else 129, (rows, blocks + wide), generator=g, device="cuda").to(torch.uint8)
        codes, scales = codes[:, off:off + cols], scales[:, off:off + blocks]
        if k % 2:
            codes[:, -1] &= 15
        return codes, scales

    return (*side(m), *side(n), torch.randn(n, generator=g, device="cuda"))


def _check_product(out, a, sa, b, sb, bias, dtype, exact=False):
    x, y = values_of(a, sa, 2 * a.shape[1]), values_of(b, sb, 2 * b.shape[1])
    want = (x @ y.T.contiguous()).cpu().numpy()
    mass = (x.abs().nan_to_num(0) @ y.abs().nan_to_num(0).T.contiguous()).cpu().numpy()
    rel, least = ROUND[dtype]
    slack = np.zeros_like(want) if exact else (128 + 2 * a.shape[1] / 64 + 16) * 2 * U * mass
    if bias is not None:
        want = want + bias.double().cpu().numpy()
        slack = slack + U * (np.where(np.isfinite(want), np.abs(want), 0) + slack)
    got = out.double().cpu().numpy()
    assert out.dtype == dtype and got.shape == want.shape
    top = float(torch.finfo(dtype).max)
    assert (np.abs(want[np.isfinite(want)]) < top / 2).all()
    finite = np.isfinite(want)
    np.testing.assert_array_equal(got[~finite], want[~finite])
    bound = slack + (np.where(finite, np.abs(want), 0) + slack) * rel + least
    err = np.abs(np.where(finite, got - np.where(finite, want, 0), 0))
    assert (err <= bound).all(), (err / bound).max()


# m and n around the tiles of 16, 32, 64, 128 and 256, k around blocks and the steps of 64, 128, 256 and 512 values
SIZES = [
    (1, 1, 1), (1, 1, 32), (1, 1000, 128), (2, 77, 10), (3, 129, 30), (16, 300, 96), (17, 31, 33), (31, 257, 100),
    (32, 512, 128), (33, 513, 129), (64, 64, 64), (65, 127, 200), (100, 1001, 65), (127, 255, 256), (128, 128, 1024),
    (129, 300, 62), (255, 257, 288), (256, 256, 768), (300, 200, 2000), (511, 513, 224), (1, 5000, 4096), (20, 700, 2049),
    (600, 700, 769), (1030, 2100, 520), (33, 70, 640), (200, 900, 4096), (1000, 3000, 1152), (130, 20000, 1280),
    (1500, 3300, 768), (1500, 3300, 1001), (100, 900, 8002), (4096, 3329, 2048), (7, 40, 100_003), (70, 130, 40_000),
    (40, 40, 992), (260, 300, 130), (12, 5000, 480)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m, n, k", SIZES)
def test_product(scoring, dtype, m, n, k):
    say("4-bit product", dtype, m, n, k)
    a, sa, b, sb, bias = _inputs(m, n, k, m * 31 + n * 7 + k)
    if dtype == torch.float16:  # within its range
        sa, sb = sa - 6, sb - 6
    _check_product(scoring.mx4_product(a, sa, b, sb, dtype=dtype), a, sa, b, sb, None, dtype)
    bias[::7] = -float("inf")
    _check_product(scoring.mx4_product(a, sa, b, sb, bias=bias, dtype=dtype), a, sa, b, sb, bias, dtype)


@pytest.mark.parametrize("m, n, k", SIZES)
def test_product_exact(scoring, m, n, k):
    """Partial sums that fp32 holds: the result is the definition's to the last bit, whichever way it goes."""
    say("4-bit product, exact sums", m, n, k)
    a, sa, b, sb, _ = _inputs(m, n, k, m + 3 * n + 5 * k, near=True)
    assert 6 * 6 * 16 * min(k, 10_000) < 2 ** 24  # in units of 2^-4: codes are halves, scales 1/2 or 1
    if k > 10_000:  # most blocks zero
        a[:, 2_000:-2_000] = 0
    x, y = values_of(a, sa, 2 * a.shape[1]), values_of(b, sb, 2 * b.shape[1])
    want = x @ y.T.contiguous()
    for dtype in TYPES:
        assert torch.equal(scoring.mx4_product(a, sa, b, sb, dtype=dtype), want.float().to(dtype))


def _check_exact(scoring, m, n, k, dtype, with_bias):
    """Sums, and a bias in whole units of theirs, that fp32 holds, and fp32 products of the reference too."""
    a, sa, b, sb, bias = _inputs(m, n, k, m + 3 * n + 5 * k, near=True)
    assert 6 * 6 * 16 * (k + 1) < 2 ** 24
    bias = (bias * 16).round() / 16 if with_bias else None
    out = scoring.mx4_product(a, sa, b, sb, bias=bias, dtype=dtype)
    want = values_of(a, sa, 2 * a.shape[1]).float() @ values_of(b, sb, 2 * b.shape[1]).float().T.contiguous()
    assert torch.equal(out, (want if bias is None else want + bias).to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m, n, k", [(1000, 300, 100), (5000, 70, 128), (2001, 33, 64), (130, 1, 32), (77, 4097, 40), (31, 63, 200),
                                     (32, 5000, 256), (3, 20_000, 640), (32, 5000, 1024), (17, 9000, 1152), (16, 4000, 4001),
                                     (30, 3000, 2001), (24, 9001, 1001), (9, 777, 500), (64, 40_000, 768), (50, 40_001, 1024),
                                     (40_000, 64, 640), (90_001, 17, 128)])
def test_product_few_rows_or_columns(scoring, dtype, m, n, k):
    say("4-bit product", dtype, m, n, k)
    _check_exact(scoring, m, n, k, dtype, m % 2 == 1)


@pytest.mark.parametrize("m, n, k, dtype", [
    (1000, 50_001, 100, torch.float16), (70, 720_001, 32, torch.bfloat16), (17, 1_500_001, 64, torch.float32),
    (129, 375_000, 130, torch.bfloat16), (300, 160_000, 256, torch.float16), (130, 150_001, 450, torch.float32),
    (66, 300_032, 512, torch.float32), (16, 600_032, 96, torch.float32), (50, 400_064, 128, torch.float16),
    (30, 600_064, 200, torch.bfloat16), (31, 300_001, 250, torch.float32), (10, 900_032, 400, torch.float32),
    (13, 1_300_001, 300, torch.float16), (101, 100_032, 128, torch.float32), (64, 300_001, 100, torch.float16),
    (60, 300_000, 384, torch.bfloat16)])
def test_product_large_results(scoring, m, n, k, dtype):
    """Results of more than the caches hold, of whole lines and others."""
    say("4-bit product, large results", m, n, k, dtype)
    _check_exact(scoring, m, n, k, dtype, n % 2 == 1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m, n, k, bias", [(260, 60001, 640, True), (300, 60160, 768, False), (257, 98000, 896, True),
                                           (512, 60000, 1024, False), (513, 61000, 1152, True)])
def test_product_many_tiles(scoring, dtype, m, n, k, bias):
    """More large tiles than CUs."""
    say("4-bit product", dtype, m, n, k, bias)
    a, sa, b, sb, add = _inputs(m, n, k, m + n + k, near=True)
    out = scoring.mx4_product(a, sa, b, sb, bias=add if bias else None, dtype=dtype)
    _check_product(out, a, sa, b, sb, add if bias else None, dtype, exact=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m, n, k, wide, off", [(5, 300, 100, 28, 4), (70, 90, 192, 31, 1), (300, 290, 256, 16, 16),
                                               (260, 515, 257, 3, 3), (1, 600, 768, 5, 2), (9, 500, 64, 9, 8),
                                               (300, 700, 1024, 4, 0), (40, 60, 20, 3, 1)])
def test_product_strides(scoring, dtype, m, n, k, wide, off):
    """Operands, scales and output inside wider matrices, at odd addresses; nothing beside the output is written."""
    say("4-bit product, strides", dtype, m, n, k, wide, off)
    a, sa, b, sb, _ = _inputs(m, n, k, k, near=True, wide=wide, off=off)
    store = torch.full((m, n + off + 9), 7.0, dtype=dtype, device="cuda")
    out = scoring.mx4_product(a, sa, b, sb, out=store[:, off:off + n])
    _check_product(out, a, sa, b, sb, None, dtype, exact=True)
    assert (store[:, :off] == 7).all() and (store[:, off + n:] == 7).all()


@pytest.mark.parametrize("m, n, k", [(1, 300, 128), (20, 300, 4096), (70, 300, 128), (300, 300, 1024), (70, 70, 1001),
                                     (5, 70, 20), (600, 700, 768)])
def test_product_nan_and_zero_blocks(scoring, m, n, k):
    """A NaN block makes its row's results NaN, zero codes under it too; no other row's."""
    say("4-bit product, NaN blocks", m, n, k)
    a, sa, b, sb, _ = _inputs(m, n, k, k, near=True)
    b[7] = 0
    sb[7] = 0
    b[9, :1] = 0
    sb[9, -1] = 255
    b[11] = 0
    sb[11, 0] = 255
    if m > 4:
        sa[3, sa.shape[1] // 2] = 255
    out = scoring.mx4_product(a, sa, b, sb)
    want = values_of(a, sa, 2 * a.shape[1]) @ values_of(b, sb, 2 * b.shape[1]).T.contiguous()
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    assert torch.equal(out.nan_to_num(0.0), want.nan_to_num(0.0).float())
    assert (out[0, 7] == 0) and torch.isnan(out[0, 9]) and torch.isnan(out[0, 11])


@pytest.mark.parametrize("m, n, k", [(2, 64, 128), (70, 64, 256), (300, 300, 1024)])
def test_product_far_scales(scoring, m, n, k):
    """Scales from one end to the other: results past the largest float are infinities, 2^127 2^-127 is 1."""
    say("4-bit product, far scales", m, n, k)
    a, sa, b, sb, _ = _inputs(m, n, k, 5, near=True)
    sa = torch.full_like(sa, 250)
    sb = torch.full_like(sb, 4)
    _check_product(scoring.mx4_product(a, sa, b, sb), a, sa, b, sb, None, torch.float32, exact=True)
    sb[::2] = 254
    a, b = a & 0x77, b & 0x77  # none below 0
    a[:, :] |= 1
    b[:, :] |= 1
    out = scoring.mx4_product(a, sa, b, sb)
    assert torch.isinf(out[:, ::2]).all() and torch.isfinite(out[:, 1::2]).all()


def test_product_empty(scoring):
    say("4-bit product, empty sizes")
    a, sa, b, sb, bias = _inputs(40, 50, 64, 3)
    assert scoring.mx4_product(a[:0], sa[:0], b, sb).shape == (0, 50)
    assert scoring.mx4_product(a, sa, b[:0], sb[:0]).shape == (40, 0)
    for m in (1, 40):
        none = a[:m, :0], sa[:m, :0], b[:, :0], sb[:, :0]
        assert torch.equal(scoring.mx4_product(*none, bias=bias), bias.expand(m, 50))
        assert (scoring.mx4_product(*none) == 0).all()


def test_long_catalogue(scoring):
    """Rows, and outputs, past 2^31 bytes from the first."""
    say("4-bit product, offsets past 31 bits")
    n, k = 33_000_000, 130
    b = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda")
    sb = torch.full((n, 5), 126, dtype=torch.uint8, device="cuda")
    sb[::3, 1] = 128
    at = [0, n // 2, n - 1]
    a, sa = b[at].contiguous(), sb[at].contiguous()
    spans = (0, n // 2 - 50, n - 100)
    out = scoring.mx4_product(a, sa, b, sb)
    for lo in spans:
        _check_product(out[:, lo:lo + 100], a, sa, b[lo:lo + 100], sb[lo:lo + 100], None, torch.float32, exact=True)
    a, sa = a.repeat(14, 1)[:40].contiguous(), sa.repeat(14, 1)[:40].contiguous()
    out = scoring.mx4_product(a, sa, b, sb, dtype=torch.bfloat16)  # 2.6 GB
    for lo in spans:
        _check_product(out[:, lo:lo + 100], a, sa, b[lo:lo + 100], sb[lo:lo + 100], None, torch.bfloat16, exact=True)
    del out
    values = scoring.mx4_values(b, sb, dtype=torch.bfloat16)  # 8.6 GB
    for lo in spans:
        assert torch.equal(values[lo:lo + 100], values_of(b[lo:lo + 100], sb[lo:lo + 100], k).to(torch.bfloat16))
    codes, scales = scoring.quantize_rows_mx4(values)
    assert torch.equal(scoring.mx4_values(codes, scales, dtype=torch.bfloat16), values)


def test_many_rows(scoring):
    """More blocks than one launch is given."""
    n, d = 2 ** 30 + 300, 33
    torch.cuda.empty_cache()
    say("4-bit rows,", n, d)
    x = torch.full((n, d), 2.0, dtype=torch.bfloat16, device="cuda")  # 71 GB
    x[::3] = -1
    codes, scales = scoring.quantize_rows_mx4(x)
    # 2 = 4 2^-1, -1 = -4 2^-2
    assert (scales[::3] == 125).all() and (scales[1::3] == 126).all() and (scales[2::3] == 126).all()
    assert (codes[::3, :16] == 0xEE).all() and (codes[1::3, :16] == 0x66).all() and (codes[2::3, :16] == 0x66).all()
    assert (codes[::3, 16] == 0x0E).all() and (codes[1::3, 16] == 0x06).all() and (codes[2::3, 16] == 0x06).all()
    scoring.mx4_values(codes, scales, d, out=x)
    assert (x[::3] == -1).all() and (x[1::3] == 2).all() and (x[2::3] == 2).all()
    del x, codes, scales
    torch.cuda.empty_cache()


def test_many_rows_of_a_product(scoring):
    """More rows of a than the panels of one launch have."""
    m, n, k = 2 ** 30 + 129, 2, 32
    torch.cuda.empty_cache()
    say("4-bit product,", m, n, k)
    a = torch.randint(0, 256, (m, k // 2), dtype=torch.uint8, device="cuda")  # 17 GB
    sa = torch.full((m, 1), 127, dtype=torch.uint8, device="cuda")
    sa[::7] = 126
    b, sb = a[5:7].clone(), sa[5:7].clone()
    out = scoring.mx4_product(a, sa, b, sb, dtype=torch.bfloat16)
    for lo in (0, m // 2, m - 300):
        _check_product(out[lo:lo + 300], a[lo:lo + 300], sa[lo:lo + 300], b, sb, None, torch.bfloat16, exact=True)
    del a, sa, out
    torch.cuda.empty_cache()


def test_distant_rows(scoring):
    """Operands' and output rows 2^25 elements and more apart; nothing beside the output is written."""
    stride = 2 ** 25 + 3
    store = torch.empty(600 * stride, dtype=torch.uint8, device="cuda")  # 20 GB
    for m, n, k in ((1, 70, 100), (20, 70, 600), (40, 50, 100), (70, 300, 130), (250, 300, 1024), (40, 50, 2000), (40, 50, 20)):
        say("4-bit product, distant rows", m, n, k)
        a, sa, b, sb, bias = _inputs(m, n, k, k, near=True)
        far_a = store.as_strided(a.shape, (stride, 1))
        far_b = store.as_strided(b.shape, (stride, 1), m * stride)
        far_sb = store.as_strided(sb.shape, (stride, 1), m * stride + 5_000)
        far_a.copy_(a)
        far_b.copy_(b)
        far_sb.copy_(sb)
        wide = torch.empty(m * stride, dtype=torch.bfloat16, device="cuda").as_strided((m, n + 16), (stride, 1))
        wide.fill_(7.0)
        out = scoring.mx4_product(far_a, sa, far_b, far_sb, bias=bias, out=wide[:, 5:5 + n])
        _check_product(out, a, sa, b, sb, bias, torch.bfloat16, exact=True)
        assert (wide[:, :5] == 7).all() and (wide[:, 5 + n:] == 7).all()
        assert torch.equal(out, scoring.mx4_product(a, sa, b, sb, bias=bias, dtype=torch.bfloat16))


def test_other_stream_and_order(scoring):
    """Calls follow the current stream's order, and equal calls give equal bits."""
    say("4-bit scores on a stream of their own")
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn((5000, 300), generator=g, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y = x * 3
        codes, scales = scoring.quantize_rows_mx4(y)
        s = scoring.mx4_product(codes[:64], scales[:64], codes, scales, dtype=torch.bfloat16)
        values = scoring.mx4_values(codes, scales)
    side.synchronize()
    _check_rows(y, codes, scales)
    _check_product(s, codes[:64], scales[:64], codes, scales, None, torch.bfloat16)
    assert torch.equal(s, scoring.mx4_product(codes[:64], scales[:64], codes, scales, dtype=torch.bfloat16))
    assert torch.equal(values, values_of(codes, scales, 300).float())


def test_in_a_graph(scoring):
    """Captured calls of every kernel of the product give what eager calls give, replay after replay."""
    say("4-bit scores in a graph")
    for m, n, k in ((5, 3000, 96), (20, 300, 2048), (200, 1000, 100), (200, 900, 1024), (1000, 3000, 1280), (300, 700, 666),
                    (4096, 3329, 2048), (40, 40, 14)):
        g = torch.Generator(device="cuda").manual_seed(k)
        x = torch.randn((m, k), generator=g, device="cuda")
        b, sb = scoring.quantize_rows_mx4(torch.randn((n, k), generator=g, device="cuda"))
        rows = scoring.quantize_rows_mx4(x)
        out = scoring.mx4_product(*rows, b, sb, dtype=torch.bfloat16)
        values = scoring.mx4_values(*rows, k)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            scoring.quantize_rows_mx4(x, out=rows)
            scoring.mx4_product(*rows, b, sb, out=out)
            scoring.mx4_values(*rows, k, out=values)
        for turn in range(3):
            x.copy_(torch.randn((m, k), generator=g, device="cuda"))
            graph.replay()
            torch.cuda.synchronize()
            again = scoring.quantize_rows_mx4(x.clone())
            assert torch.equal(out, scoring.mx4_product(*again, b, sb, dtype=torch.bfloat16))
            assert torch.equal(values, scoring.mx4_values(*again, k))


def test_catalogue(scoring):
    """A catalogue in 4 bits: its scores are the product of its rows and the queries', cut into batches or not."""
    say("a catalogue in 4 bits")
    g = torch.Generator(device="cuda").manual_seed(9)
    vectors = torch.nn.functional.normalize(torch.randn((3001, 96), generator=g, device="cuda"), dim=1)
    queries = vectors[5:105] + 0.02 * torch.randn((100, 96), generator=g, device="cuda")
    bias = torch.zeros(3001, device="cuda")
    bias[17] = -float("inf")
    catalogue = scoring.DenseCatalogue(vectors, bias=bias, bits=4)
    assert catalogue.codes.shape == (3001, 48) and len(catalogue) == 3001
    scores = catalogue.scores(queries)
    _check_product(scores, *scoring.quantize_rows_mx4(queries), catalogue.codes, catalogue.scales, bias, torch.float32)
    targets = torch.arange(5, 105, dtype=torch.int32, device="cuda")
    whole = catalogue.log_probs(queries, targets, top_k=10, temperature=0.05)
    assert torch.equal(whole.target, scoring.log_probs(scores, targets, temperature=0.05).target)
    parts = scoring.DenseCatalogue(vectors, bias=bias, bits=4, score_bytes=3001 * 4 * 33).log_probs(
        queries, targets, top_k=10, temperature=0.05)
    assert torch.equal(whole.top_ids, parts.top_ids) and torch.equal(whole.target, parts.target)
    assert not (whole.top_ids == 17).any()


@pytest.mark.parametrize("m, n, k", [(1, 3, 130_000_000), (20, 3, 130_000_000), (17, 2, 126_400_000), (1, 2, 260_000_000)])
def test_longest_rows_of_a_product(scoring, m, n, k):
    """Rows whose codes and scales no workgroup could keep in LDS, by factors that pass 31 bits; codes are 0 but for some."""
    say("4-bit product, rows of", k)
    g = torch.Generator(device="cuda").manual_seed(k)
    at = torch.randint(0, k // 2, (3000,), generator=g, device="cuda").unique()
    at = torch.cat([at, torch.tensor([0, 15, 16, k // 2 - 1], device="cuda")]).unique()
    rows = []
    for count in (m, n):
        codes = torch.zeros((count, k // 2), dtype=torch.uint8, device="cuda")
        scales = torch.full((count, -(-k // 32)), 127, dtype=torch.uint8, device="cuda")
        scales[:, ::5] = 126
        codes[:, at] = torch.randint(0, 256, (count, at.numel()), generator=g, device="cuda", dtype=torch.uint8)
        grid = torch.tensor(np.concatenate([GRID, -GRID]), device="cuda")
        there, s = codes[:, at].long(), torch.exp2(scales[:, at // 16].double() - 127)
        rows.append((codes, scales, torch.cat([grid[there & 15] * s, grid[there >> 4] * s], 1)))
    (a, sa, va), (b, sb, vb) = rows
    out = scoring.mx4_product(a, sa, b, sb)
    # sums of up to 6,008 products, each a whole number of 2^-4 and at most 36: below 2^18, so exact
    assert torch.equal(out, (va @ vb.T.contiguous()).float())


@pytest.mark.parametrize("n, d, wide, off, dtype", [
    (500_001, 128, 128, 0, torch.float32), (300_000, 96, 128, 16, torch.bfloat16), (1_200_001, 100, 100, 0, torch.float16),
    (800_000, 52, 52, 0, torch.float32), (700_000, 100, 132, 0, torch.float32), (500_000, 31, 31, 0, torch.float32),
    (1_000_003, 33, 40, 1, torch.bfloat16), (60_001, 1001, 1001, 0, torch.float32)])
def test_values_large_results(scoring, n, d, wide, off, dtype):
    """Values of more than the L2s hold, past them and through them; nothing beside the rows is written."""
    say("4-bit values, large results", n, d, wide, off, dtype)
    g = torch.Generator(device="cuda").manual_seed(d)
    codes = torch.randint(0, 256, (n, (d + 1) // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.randint(120, 130, (n, -(-d // 32)), generator=g, device="cuda", dtype=torch.uint8)
    store = torch.full((n, wide), 99.0, dtype=dtype, device="cuda")
    scoring.mx4_values(codes, scales, d, out=store[:, off:off + d])
    assert (store[:, :off] == 99).all() and (store[:, off + d:] == 99).all()
    for lo in range(0, n, 100_000):
        want = values_of(codes[lo:lo + 100_000], scales[lo:lo + 100_000], d).to(dtype)
        assert torch.equal(store[lo:lo + 100_000, off:off + d], want)


# rows in the registers (one and two instructions), strips (of a wave, over four waves; every number of blocks in the last step),
# panels of two, four and eight steps, tiles through registers, and straight to LDS (few, many, walking; words and groups of scales)
@pytest.mark.parametrize("m, n, k", [
    (10, 700, 90), (40, 700, 130), (20, 700, 200), (16, 700, 230), (10, 700, 400), (16, 700, 262), (9, 700, 512), (16, 700, 4001),
    (30, 700, 2001), (5, 8000, 1000), (32, 300, 2080), (129, 150_000, 120), (129, 200_001, 120), (129, 150_001, 250),
    (130, 140_003, 500), (300, 700, 1001), (20, 900, 1152), (20, 900, 2048), (70, 700, 1152), (600, 700, 1152), (600, 900, 2048),
    (1024, 1500, 1152), (2000, 2500, 1024), (2000, 2100, 1001), (512, 61_000, 640), (512, 61_000, 1024), (512, 61_001, 1152)])
def test_product_nan_blocks_of_every_kernel(scoring, m, n, k):
    """NaN scales in the first, the last and the one before it, at tiles' borders on both sides: their rows are NaN, no other is."""
    say("4-bit product, NaN blocks", m, n, k)
    a, sa, b, sb, _ = _inputs(m, n, k, k, near=True)
    blocks = sa.shape[1]
    rows_a = sorted({0, m // 2, m - 1} | {r for r in (15, 16, 31, 32, 63, 64, 127, 128, 255, 256) if r < m and r % 3})
    rows_b = sorted({0, 5, n // 2, n - 1} | {r for r in (15, 16, 31, 32, 63, 64, 127, 128, 255, 256, 511, 512) if r < n and r % 3})
    at = [0, blocks - 1, max(0, blocks - 2), blocks // 2]
    want = scoring.mx4_product(a, sa, b, sb)
    _check_product(want, a, sa, b, sb, None, torch.float32, exact=True)
    for rows, codes, scales, axis in ((rows_a, a, sa, 0), (rows_b, b, sb, 1)):
        bad = scales.clone()
        for i, r in enumerate(rows):
            bad[r, at[i % 4]] = 255
        codes = codes.clone()
        codes[rows[-1]] = 0  # zero codes under a NaN scale too
        out = scoring.mx4_product(codes, bad, b, sb) if axis == 0 else scoring.mx4_product(a, sa, codes, bad)
        there = torch.zeros(m if axis == 0 else n, dtype=torch.bool, device="cuda")
        there[rows] = True
        if axis == 0:
            assert torch.isnan(out[there]).all() and torch.equal(out[~there], want[~there])
        else:
            assert torch.isnan(out[:, there]).all() and torch.equal(out[:, ~there], want[:, ~there])


@pytest.mark.parametrize("m, n, k", [(1, 40, 128), (20, 40, 128), (10, 700, 400), (16, 700, 4001), (30, 700, 2001), (20, 700, 200),
                                     (300, 300, 1024), (70, 70, 1000)])
def test_product_large_scales_of_zeros(scoring, m, n, k):
    """Values near the largest float against zeros: their blocks' scales multiply past it, the products are 0."""
    say("4-bit product, large scales", m, n, k)
    x, y = torch.zeros((m, k), device="cuda"), torch.zeros((n, k), device="cuda")
    x[:, 0::2] = 3e38
    y[:, 1::2] = -2e38
    for dtype in TYPES:
        out = scoring.mx4_product(*scoring.quantize_rows_mx4(x), *scoring.quantize_rows_mx4(y), dtype=dtype)
        assert (out == 0).all()
