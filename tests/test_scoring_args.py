"""Dense scoring calls: what they refuse, before any GPU is touched."""
from __future__ import annotations

import ctypes as C
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

P = C.c_void_p


@pytest.fixture(scope="module")
def lib():
    from quiver import _lib

    return _lib


@pytest.fixture(scope="module")
def buf():
    """Host memory that no refused call reads: only its address is looked at."""
    return np.zeros(4096, np.uint8)


def _at(buf, off=0):
    return buf.ctypes.data + off


def test_quantize_refusals(lib, buf):
    f, p = lib.load().qv_quantize_rows, _at(buf)
    ok = dict(x=p, type=lib.QV_FLOAT, n=2, dim=8, xs=8, codes=p, cs=8, scales=p)

    def rc(**change):
        return f(*{**ok, **change}.values(), 0, None)

    for change, text in [(dict(x=None), b"x: null"), (dict(codes=None), b"codes: null"), (dict(scales=None), b"scales: null"),
                         (dict(type=lib.QV_INT8), b"type must be"), (dict(type=9), b"type must be"),
                         (dict(n=-1), b"negative"), (dict(dim=-1), b"negative"), (dict(xs=7), b"x: rows overlap"),
                         (dict(cs=7), b"codes: rows overlap"), (dict(x=p + 2), b"x: not aligned"),
                         (dict(scales=p + 1), b"scales: not aligned")]:
        assert rc(**change) == lib.QV_EINVAL, change
        assert text in lib.load().qv_last_error(), (change, lib.load().qv_last_error())
    assert rc(n=2 ** 31, dim=1, xs=1, cs=1) == lib.QV_EUNSUPPORTED
    assert rc(n=0, x=None, codes=None, scales=None) == lib.QV_OK  # nothing to do, no GPU needed


def test_product_refusals(lib, buf):
    f, p = lib.load().qv_int8_product, _at(buf)
    ok = dict(a=p, astr=8, asc=p, m=2, b=p, bstr=8, bsc=p, bias=None, n=2, k=8, out=p, type=lib.QV_FLOAT, ostr=2)

    def rc(**change):
        return f(*{**ok, **change}.values(), 0, None)

    for change, text in [(dict(a=None), b"a: null"), (dict(b=None), b"b: null"), (dict(out=None), b"out: null"),
                         (dict(asc=None), b"a_scales: null"), (dict(bsc=None), b"b_scales: null"),
                         (dict(type=lib.QV_UINT8), b"type must be"), (dict(m=-1), b"negative"), (dict(n=-1), b"negative"),
                         (dict(k=-1), b"negative"), (dict(astr=7), b"a: rows overlap"), (dict(bstr=7), b"b: rows overlap"),
                         (dict(ostr=1), b"out: rows overlap"), (dict(out=p + 2), b"out: not aligned"),
                         (dict(bias=p + 2), b"bias: not aligned")]:
        assert rc(**change) == lib.QV_EINVAL, change
        assert text in lib.load().qv_last_error(), (change, lib.load().qv_last_error())
    big = lib.QV_PRODUCT_MAX_K + 1
    assert rc(k=big, astr=big, bstr=big) == lib.QV_EUNSUPPORTED
    assert rc(m=0, a=None, asc=None, out=None) == lib.QV_OK
    assert rc(n=0, b=None, bsc=None, out=None) == lib.QV_OK


def test_log_probs_refusals(lib, buf):
    L, p = lib.load(), _at(buf)
    need = L.qv_log_probs_workspace(2, 8, 4)
    assert 0 <= need
    assert L.qv_log_probs_workspace(-1, 8, 4) < 0 and L.qv_log_probs_workspace(1, 8, 65) < 0
    ok = dict(x=p, type=lib.QV_FLOAT, rows=2, cols=8, stride=8, temp=1.0, targets=p, per_row=1, topk=4, target=p,
              entropy=p, lse=p, stats=p, ids=p, top=p, work=p, bytes=max(need, 64))

    def rc(**change):
        return L.qv_log_probs(*{**ok, **change}.values(), 0, None)

    nan, inf = float("nan"), float("inf")
    for change, text in [(dict(x=None), b"logits: null"), (dict(x=p + 1), b"logits: not aligned"),
                         (dict(stride=7), b"logits: rows overlap"), (dict(type=0), b"type must be"),
                         (dict(rows=-1), b"negative"), (dict(cols=-1), b"negative"), (dict(temp=0.0), b"temperature"),
                         (dict(temp=-1.0), b"temperature"), (dict(temp=nan), b"temperature"),
                         (dict(temp=inf), b"temperature"), (dict(temp=1e-45), b"temperature"),
                         (dict(targets=None), b"targets: null"), (dict(target=None), b"target: null"),
                         (dict(per_row=-1), b"targets_per_row"), (dict(topk=-1), b"topk"), (dict(stats=None), b"stats: null"),
                         (dict(ids=None), b"top_ids: null"), (dict(top=None), b"top: null")]:
        assert rc(**change) == lib.QV_EINVAL, change
        assert text in L.qv_last_error(), (change, L.qv_last_error())
    assert rc(topk=65) == lib.QV_EUNSUPPORTED and rc(per_row=65) == lib.QV_EUNSUPPORTED
    assert rc(cols=2 ** 31, stride=2 ** 31) == lib.QV_EUNSUPPORTED
    assert rc(rows=0, x=None, targets=None, target=None, stats=None, ids=None, top=None) == lib.QV_OK
    # a workspace that is needed has to be there, large enough and aligned
    need = L.qv_log_probs_workspace(1, 2 ** 24, 4)
    if need:
        for change, text in [(dict(work=None), b"workspace"), (dict(bytes=need - 1), b"workspace"), (dict(work=p + 8), b"workspace")]:
            assert rc(rows=1, cols=2 ** 24, stride=2 ** 24, **{"bytes": need, **change}) == lib.QV_EINVAL
            assert text in L.qv_last_error(), (change, L.qv_last_error())


def test_gradient_refusals(lib, buf):
    L, p = lib.load(), _at(buf)
    ok = dict(x=p, type=lib.QV_FLOAT, rows=2, cols=8, stride=8, temp=1.0, stats=p, entropy=p, targets=p, per_row=1,
              ids=p, topk=4, gt=p, ge=p, gl=p, gk=p, grad=p, gstride=8)

    def rc(**change):
        return L.qv_log_probs_grad(*{**ok, **change}.values(), 0, None)

    for change, text in [(dict(x=None), b"logits: null"), (dict(grad=None), b"grad: null"), (dict(gstride=7), b"grad: rows overlap"),
                         (dict(stats=None), b"stats: null"), (dict(entropy=None), b"entropy: null"),
                         (dict(targets=None), b"targets: null"), (dict(ids=None), b"top_ids: null"),
                         (dict(temp=0.0), b"temperature"), (dict(grad=p + 2), b"grad: not aligned")]:
        assert rc(**change) == lib.QV_EINVAL, change
        assert text in L.qv_last_error(), (change, L.qv_last_error())
    assert rc(rows=0, x=None, grad=None, stats=None, entropy=None, targets=None, ids=None) == lib.QV_OK
    assert rc(cols=0, stride=0, x=None, grad=None, gstride=0) == lib.QV_OK


def test_python_refusals():
    """Tensors that are not on a GPU, or have another type, shape or layout, are refused by name."""
    from quiver import scoring

    x = torch.zeros(3, 8)
    with pytest.raises(ValueError, match="on the GPU"):
        scoring.quantize_rows(x)
    with pytest.raises(ValueError, match="on the GPU"):
        scoring.log_probs(x)
    codes, scales = torch.zeros(3, 8, dtype=torch.int8), torch.zeros(3)
    with pytest.raises(ValueError, match="on the GPU"):
        scoring.int8_product(codes, scales, codes, scales)
    with pytest.raises(ValueError, match="x has the type"):
        scoring.quantize_rows(x.double())
    with pytest.raises(ValueError, match="two dimensions"):
        scoring.quantize_rows(x[0])
    with pytest.raises(ValueError, match="contiguous along its rows"):
        scoring.quantize_rows(torch.zeros(8, 3).T)
    with pytest.raises(ValueError, match="a has the type"):
        scoring.int8_product(x, scales, codes, scales)
    with pytest.raises(ValueError, match="length of their rows"):
        scoring.int8_product(codes, scales, codes[:, :4], scales)
    with pytest.raises(ValueError, match="a_scales must be"):
        scoring.int8_product(codes, scales[:2], codes, scales)
    with pytest.raises(ValueError, match="bias must be"):
        scoring.int8_product(codes, scales, codes, scales, bias=scales[:2])
    with pytest.raises(ValueError, match="out must have the shape"):
        scoring.int8_product(codes, scales, codes, scales, out=torch.zeros(3, 4))
    with pytest.raises(ValueError, match="dtype must be"):
        scoring.int8_product(codes, scales, codes, scales, dtype=torch.float64)
    with pytest.raises(ValueError, match="targets must be"):
        scoring.log_probs(x, torch.zeros(3, 1, dtype=torch.int64))
    with pytest.raises(ValueError, match="targets must be"):
        scoring.log_probs(x, torch.zeros(2, 1, dtype=torch.int32))
    with pytest.raises(ValueError, match="top_k must be"):
        scoring.log_probs(x, top_k=65)
    with pytest.raises(ValueError, match="targets per row"):
        scoring.log_probs(x, torch.zeros(3, 65, dtype=torch.int32))
    with pytest.raises(ValueError, match="score_bytes"):
        scoring.DenseCatalogue(x, score_bytes=0)


@pytest.mark.parametrize("order, says", [("_lib.load(); from quiver import scoring", "loaded before torch"),
                                         ("from quiver import scoring; _lib.load()", ""),
                                         ("import torch; _lib.load(); from quiver import scoring", "")])
def test_one_hip_runtime(order, says):
    """Loading the library before torch is refused by name, not left to fail as a missing GPU."""
    package = Path(__file__).resolve().parents[1] / "quiver-ae_amd"
    run = subprocess.run([sys.executable, "-c", f"import sys; sys.path.insert(0, {str(package)!r}); from quiver import _lib; "
                          + order], capture_output=True, text=True, timeout=300)
    assert (run.returncode != 0) == bool(says)
    assert says in run.stderr


def test_buffers_refused(lib):
    """What the library refuses to size is its error, not an allocation of a negative size."""
    from quiver import scoring

    with pytest.raises(lib.QuiverError, match="more than 2\\^31 - 1 rows or columns"):
        scoring.LogProbs.empty(1, 2 ** 31, 0, 4, 1.0, torch.device("cuda"))


@pytest.mark.parametrize("temp, fine", [(1.2e-38, True), (1e-30, True), (1e38, True), (4.2e-39, False), (4e-39, False), (3e-39, False)])
def test_temperature_range(lib, buf, temp, fine):
    """A temperature whose reciprocal is finite and log2(e) times it is not would make every row NaN: refused."""
    L, p = lib.load(), _at(buf)
    rcs = [L.qv_log_probs(p, lib.QV_FLOAT, 0, 8, 8, temp, None, 0, 0, None, p, p, p, None, None, p, 64, 0, None),
           L.qv_log_probs_grad(p, lib.QV_FLOAT, 0, 8, 8, temp, p, p, None, 0, None, 0, None, p, None, None, p, 8, 0, None)]
    assert rcs == [lib.QV_OK if fine else lib.QV_EINVAL] * 2
    if not fine:
        assert b"temperature" in L.qv_last_error()


def _calls_without_derivative(wrap):
    """Every call and argument that a derivative would be lost at; `wrap` makes an argument ask for one."""
    from quiver import scoring

    x, codes, scales = torch.zeros(3, 8), torch.zeros(3, 8, dtype=torch.int8), torch.zeros(3)
    empty = torch.zeros(3, 0)
    r = scoring.LogProbs.of(empty, scales, scales, empty.int(), empty, torch.zeros(3, 2), 1.0, torch.zeros(0))
    catalogue = scoring.DenseCatalogue.__new__(scoring.DenseCatalogue)
    catalogue.codes, catalogue.scales, catalogue.bias = codes, scales, None
    catalogue.score_dtype, catalogue.score_bytes = torch.float32, 1
    yield lambda: scoring.quantize_rows(wrap(x))
    yield lambda: scoring.quantize_rows(x, out=(codes, wrap(scales)))
    yield lambda: scoring.int8_product(codes, wrap(scales), codes, scales)
    yield lambda: scoring.int8_product(codes, scales, codes, wrap(scales))
    yield lambda: scoring.int8_product(codes, scales, codes, scales, bias=wrap(scales))
    yield lambda: scoring.int8_product(codes, scales, codes, scales, out=wrap(torch.zeros(3, 3)))
    yield lambda: scoring.log_probs(x, out=scoring.LogProbs.of(empty, wrap(scales), scales, empty.int(), empty,
                                                               torch.zeros(3, 2), 1.0, torch.zeros(0)))
    yield lambda: scoring.log_probs_grad(wrap(x), r)
    yield lambda: scoring.log_probs_grad(x, r, grad_target=wrap(empty))
    yield lambda: scoring.log_probs_grad(x, r, grad_entropy=wrap(scales))
    yield lambda: scoring.log_probs_grad(x, r, grad_logsumexp=wrap(scales))
    yield lambda: scoring.log_probs_grad(x, r, grad_top=wrap(empty))
    yield lambda: scoring.log_probs_grad(x, r, out=wrap(torch.zeros(3, 8)))
    yield lambda: scoring.DenseCatalogue(wrap(x))
    yield lambda: catalogue.scores(wrap(x))
    yield lambda: catalogue.log_probs(wrap(x))


def test_gradients_are_not_lost():
    """A gradient that a call does not have is refused, not left out; under no_grad nobody asks for it."""
    for call in _calls_without_derivative(lambda t: t.clone().requires_grad_()):
        with pytest.raises(ValueError, match="requires a gradient"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="on the GPU"):
            call()


def test_tangents_are_not_lost():
    """Forward-mode derivatives are refused, those of log_probs among them."""
    from torch.autograd import forward_ad

    from quiver import scoring

    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t.clone(), torch.ones_like(t))

        calls = list(_calls_without_derivative(dual))
        calls.append(lambda: scoring.log_probs(dual(torch.zeros(3, 8))))
        calls.append(lambda: scoring.log_probs(dual(torch.zeros(3, 8).requires_grad_())))
        for call in calls:
            with pytest.raises(ValueError, match="has a tangent"):
                call()
        with pytest.raises(ValueError, match="on the GPU"):
            scoring.log_probs(torch.zeros(3, 8))


def test_type_of_out():
    """A type that is asked for beside out= has to be out's; none takes out's."""
    from quiver import scoring

    codes, scales = torch.zeros(3, 8, dtype=torch.int8), torch.zeros(3)
    half = torch.zeros(3, 3, dtype=torch.float16)
    for dtype in (torch.float32, torch.bfloat16, torch.float64):
        with pytest.raises(ValueError, match="out has the type torch.float16"):
            scoring.int8_product(codes, scales, codes, scales, dtype=dtype, out=half)
    for dtype in (None, torch.float16):
        with pytest.raises(ValueError, match="on the GPU"):
            scoring.int8_product(codes, scales, codes, scales, dtype=dtype, out=half)


@pytest.mark.parametrize("rows, shape", [(6, (6, 1)), (6, (6,)), (2, (2, 1)), (4, (4, 1, 1))])
def test_targets_of_a_catalogue(rows, shape):
    """Targets of another number of rows than the queries are refused, however the queries are cut into batches."""
    from quiver import scoring

    catalogue = scoring.DenseCatalogue.__new__(scoring.DenseCatalogue)
    catalogue.codes, catalogue.scales, catalogue.bias = torch.zeros(3, 8, dtype=torch.int8), torch.zeros(3), None
    catalogue.score_dtype = torch.float32
    for catalogue.score_bytes in (24, 1 << 30):  # two queries at a time, all at once
        with pytest.raises(ValueError, match="targets must be"):
            catalogue.log_probs(torch.zeros(4, 8), torch.zeros(shape, dtype=torch.int32))
        with pytest.raises(ValueError, match="on the GPU"):
            catalogue.log_probs(torch.zeros(4, 8), torch.zeros(4, 1, dtype=torch.int32))
