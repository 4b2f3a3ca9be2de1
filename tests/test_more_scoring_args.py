"""4-bit rows, their product and layer norm: what they refuse, before any GPU is touched."""
from __future__ import annotations

import numpy as np
import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from quiver import _lib

    return _lib


@pytest.fixture(scope="module")
def buf():
    """Host memory that no refused call reads: only its address is looked at."""
    return np.zeros(4096, np.uint8)


def _at(buf):
    return buf.ctypes.data + -buf.ctypes.data % 16


def _refused(lib, f, ok, cases):
    for change, text in cases:
        assert f(*{**ok, **change}.values(), 0, None) == lib.QV_EINVAL, change
        assert text in lib.load().qv_last_error(), (change, lib.load().qv_last_error())


def test_rows_refusals(lib, buf):
    L, p = lib.load(), _at(buf)
    ok = dict(x=p, type=lib.QV_FLOAT, n=2, dim=40, xs=40, codes=p, cs=20, scales=p, ss=2)
    _refused(lib, L.qv_quantize_rows_mx4, ok, [
        (dict(x=None), b"x: null"), (dict(codes=None), b"codes: null"), (dict(scales=None), b"scales: null"),
        (dict(type=lib.QV_INT8), b"type must be"), (dict(n=-1), b"negative"), (dict(dim=-1), b"negative"),
        (dict(xs=39), b"x: rows overlap"), (dict(cs=19), b"codes: rows overlap"), (dict(ss=1), b"scales: rows overlap"),
        (dict(x=p + 2), b"x: not aligned")])
    assert L.qv_quantize_rows_mx4(*{**ok, "n": 2 ** 31, "dim": 1}.values(), 0, None) == lib.QV_EUNSUPPORTED
    assert L.qv_quantize_rows_mx4(None, lib.QV_FLOAT, 0, 40, 40, None, 20, None, 2, 0, None) == lib.QV_OK
    assert L.qv_quantize_rows_mx4(None, lib.QV_FLOAT, 3, 0, 0, None, 0, None, 0, 0, None) == lib.QV_OK
    ok = dict(codes=p, cs=20, scales=p, ss=2, n=2, dim=40, out=p, type=lib.QV_FLOAT, os=40)
    _refused(lib, L.qv_mx4_values, ok, [
        (dict(out=None), b"out: null"), (dict(codes=None), b"codes: null"), (dict(scales=None), b"scales: null"),
        (dict(type=0), b"type must be"), (dict(n=-1), b"negative"), (dict(dim=-3), b"negative"),
        (dict(os=39), b"out: rows overlap"), (dict(cs=19), b"codes: rows overlap"), (dict(ss=1), b"scales: rows overlap"),
        (dict(out=p + 1), b"out: not aligned")])


def test_product_refusals(lib, buf):
    L, p = lib.load(), _at(buf)
    ok = dict(a=p, astr=20, asc=p, ass=2, m=2, b=p, bstr=20, bsc=p, bss=2, bias=None, n=2, k=40, out=p, type=lib.QV_FLOAT,
              ostr=2)
    _refused(lib, L.qv_mx4_product, ok, [
        (dict(a=None), b"a: null"), (dict(b=None), b"b: null"), (dict(out=None), b"out: null"),
        (dict(asc=None), b"a_scales: null"), (dict(bsc=None), b"b_scales: null"), (dict(type=lib.QV_UINT8), b"type must be"),
        (dict(m=-1), b"negative"), (dict(n=-1), b"negative"), (dict(k=-2), b"negative"), (dict(k=39), b"k must be even"),
        (dict(astr=19), b"a: rows overlap"), (dict(bstr=19), b"b: rows overlap"), (dict(ass=1), b"a_scales: rows overlap"),
        (dict(bss=1), b"b_scales: rows overlap"), (dict(ostr=1), b"out: rows overlap"), (dict(out=p + 2), b"out: not aligned"),
        (dict(bias=p + 2), b"bias: not aligned")])
    assert L.qv_mx4_product(*{**ok, "m": 0, "a": None, "asc": None, "out": None}.values(), 0, None) == lib.QV_OK
    assert L.qv_mx4_product(*{**ok, "n": 0, "b": None, "bsc": None}.values(), 0, None) == lib.QV_OK


def test_norm_refusals(lib, buf):
    L, p = lib.load(), _at(buf)
    nan, inf = float("nan"), float("inf")
    eps = [(dict(eps=e), b"eps must be") for e in (0.0, -1.0, 1e-40, nan, inf)]
    ok = dict(x=p, type=lib.QV_FLOAT, n=2, dim=8, xs=8, w=p, b=p, params=lib.QV_FLOAT, eps=1e-5, y=p, ys=8)
    _refused(lib, L.qv_layer_norm, ok, eps + [
        (dict(x=None), b"x: null"), (dict(y=None), b"y: null"), (dict(type=0), b"type must be"), (dict(params=9), b"type must be"),
        (dict(n=-1), b"negative"), (dict(dim=-1), b"negative"), (dict(xs=7), b"x: rows overlap"), (dict(ys=7), b"y: rows overlap"),
        (dict(x=p + 2), b"x: not aligned"), (dict(w=p + 2), b"weight: not aligned"), (dict(b=p + 1), b"bias: not aligned")])
    assert L.qv_layer_norm(None, lib.QV_FLOAT, 0, 8, 8, None, None, lib.QV_FLOAT, 1e-5, None, 8, 0, None) == lib.QV_OK
    assert L.qv_layer_norm(*{**ok, "n": 2 ** 31}.values(), 0, None) == lib.QV_EUNSUPPORTED
    need = L.qv_layer_norm_grad_workspace(2, 8)
    assert need > 0 and L.qv_layer_norm_grad_workspace(0, 8) == 0 and L.qv_layer_norm_grad_workspace(-1, 8) == lib.QV_EINVAL
    most = lib.QV_LAYER_NORM_MAX_DIM
    assert L.qv_layer_norm_grad_workspace(1, most + 1) == lib.QV_EUNSUPPORTED and L.qv_layer_norm_grad_workspace(1, most) > 0
    assert L.qv_layer_norm(*{**ok, "dim": most + 1, "xs": most + 1, "ys": most + 1}.values(), 0, None) == lib.QV_EUNSUPPORTED
    ok = dict(x=p, type=lib.QV_FLOAT, n=2, dim=8, xs=8, g=p, gs=8, w=p, params=lib.QV_FLOAT, eps=1e-5, dx=p, dxs=8, dw=p,
              db=p, work=p, bytes=need)
    _refused(lib, L.qv_layer_norm_grad, ok, eps + [
        (dict(x=None), b"x: null"), (dict(g=None), b"grad: null"), (dict(type=0), b"type must be"), (dict(params=9), b"type must be"),
        (dict(n=-1), b"negative"), (dict(dim=-1), b"negative"), (dict(xs=7), b"x: rows overlap"), (dict(gs=7), b"grad: rows overlap"),
        (dict(dxs=7), b"dx: rows overlap"), (dict(dx=p + 2), b"dx: not aligned"), (dict(w=p + 2), b"weight: not aligned"),
        (dict(dw=p + 1), b"dweight: not aligned"), (dict(db=p + 1), b"dbias: not aligned"), (dict(work=None), b"workspace"),
        (dict(work=p + 8), b"workspace"), (dict(bytes=need - 1), b"workspace")])
    nothing = dict(dx=None, dw=None, db=None, work=None, bytes=0)
    assert L.qv_layer_norm_grad(*{**ok, **nothing}.values(), 0, None) == lib.QV_OK


def test_python_refusals(lib):
    """Tensors that are not on a GPU, or have another type, shape or layout, are refused by name."""
    from quiver import scoring

    x = torch.zeros(3, 40)
    codes, scales = torch.zeros(3, 20, dtype=torch.uint8), torch.zeros(3, 2, dtype=torch.uint8)
    rows = codes, scales
    none = torch.zeros(0, dtype=torch.uint8)
    made_for = (3, 40, torch.float32, torch.float32)
    grads = scoring.LayerNormGrad.of(x, x[0], x[0], none, made_for)
    for call, text in [
            (lambda: scoring.quantize_rows_mx4(x), "on the GPU"),
            (lambda: scoring.mx4_values(*rows), "on the GPU"),
            (lambda: scoring.mx4_product(*rows, *rows), "on the GPU"),
            (lambda: scoring.layer_norm(x), "on the GPU"),
            (lambda: scoring.layer_norm(x.clone().requires_grad_()), "on the GPU"),
            (lambda: scoring.layer_norm_grad(x, x), "on the GPU"),
            (lambda: scoring.DenseCatalogue(x, bits=4), "on the GPU"),
            (lambda: scoring.DenseCatalogue(x, bits=5), "bits must be"),
            (lambda: scoring.quantize_rows_mx4(x.double()), "x has the type"),
            (lambda: scoring.quantize_rows_mx4(x[0]), "two dimensions"),
            (lambda: scoring.quantize_rows_mx4(torch.zeros(8, 3).T), "contiguous along its rows"),
            (lambda: scoring.quantize_rows_mx4(x, out=(codes[:, :19], scales)), "codes must have the shape"),
            (lambda: scoring.quantize_rows_mx4(x, out=(codes, scales[:, :1])), "scales must have the shape"),
            (lambda: scoring.quantize_rows_mx4(x, out=(codes.char(), scales)), "codes has the type"),
            (lambda: scoring.mx4_values(codes, scales[:2]), "scales must have the shape"),
            (lambda: scoring.mx4_values(codes, scales, 41), "bytes of codes"),
            (lambda: scoring.mx4_values(codes, scales, 38), "bytes of codes"),
            (lambda: scoring.mx4_values(codes, scales, 39), "on the GPU"),
            (lambda: scoring.mx4_values(codes, scales, dtype=torch.float64), "dtype must be"),
            (lambda: scoring.mx4_values(codes, scales, dtype=torch.float16, out=x), "out has the type"),
            (lambda: scoring.mx4_values(codes, scales, 39, out=x), "out must have the shape"),
            (lambda: scoring.mx4_product(codes, scales[:, :1], *rows), "a_scales must have"),
            (lambda: scoring.mx4_product(*rows, codes, scales.int()), "b_scales has the type"),
            (lambda: scoring.mx4_product(*rows, codes[:, :16], scales[:, :1]), "length of their rows"),
            (lambda: scoring.mx4_product(*rows, *rows, bias=x[0]), "bias must be"),
            (lambda: scoring.mx4_product(*rows, *rows, out=x), "out must have the shape"),
            (lambda: scoring.mx4_product(*rows, *rows, dtype=torch.int8), "dtype must be"),
            (lambda: scoring.mx4_product(*rows, *rows, dtype=torch.float16, out=torch.zeros(3, 3)), "out has the type"),
            (lambda: scoring.layer_norm(x.int()), "x has the type"),
            (lambda: scoring.layer_norm(x[0]), "two dimensions"),
            (lambda: scoring.layer_norm(x, x[0, :39]), "weight must be"),
            (lambda: scoring.layer_norm(x, x[0].double()), "weight has the type"),
            (lambda: scoring.layer_norm(x, x[0], x[0].half()), "weight must be a contiguous torch.float16"),
            (lambda: scoring.layer_norm(x, None, x[0].int()), "bias has the type"),
            (lambda: scoring.layer_norm(x, out=x.half()), "out has the type"),
            (lambda: scoring.layer_norm(x, out=x[:2]), "out and x differ"),
            (lambda: scoring.layer_norm_grad(x, x.half()), "grad has the type"),
            (lambda: scoring.layer_norm_grad(x, x[:2]), "grad and x differ"),
            (lambda: scoring.layer_norm_grad(x, x, x[0, :9]), "weight must be"),
            (lambda: scoring.layer_norm_grad(x[:2], x[:2], out=grads), "another number of rows"),
            (lambda: scoring.layer_norm_grad(x, x, x[0].half(), out=grads), "or other types"),
            (lambda: scoring.layer_norm_grad(x.half(), x.half(), out=grads), "or other types"),
            (lambda: scoring.LayerNormGrad.of(x[:2], None, None, none, made_for), "out.x has another"),
            (lambda: scoring.LayerNormGrad.of(x.half(), None, None, none, made_for), "out.x has the type"),
            (lambda: scoring.LayerNormGrad.of(x, x[0, :9], None, none, made_for), "out.weight must be"),
            (lambda: scoring.LayerNormGrad.of(x, x[0], x[0].half(), none, made_for), "out.bias must be"),
            (lambda: scoring.layer_norm_grad(x, x, wanted=(1, 1, 0), out=grads), "wanted cannot"),
            (lambda: scoring.layer_norm_grad(x, x, out=grads), "on the GPU")]:
        with pytest.raises(ValueError, match=text):
            call()


def _calls_without_derivative(wrap):
    """Every call and argument that a derivative would be lost at; `wrap` makes an argument ask for one."""
    from quiver import scoring

    x, v = torch.zeros(3, 40), torch.zeros(40)
    codes, scales = torch.zeros(3, 20, dtype=torch.uint8), torch.zeros(3, 2, dtype=torch.uint8)
    none = torch.zeros(0, dtype=torch.uint8)
    yield lambda: scoring.quantize_rows_mx4(wrap(x))
    yield lambda: scoring.mx4_values(codes, scales, out=wrap(x))
    yield lambda: scoring.mx4_product(codes, scales, codes, scales, bias=wrap(v[:3]))
    yield lambda: scoring.mx4_product(codes, scales, codes, scales, out=wrap(torch.zeros(3, 3)))
    yield lambda: scoring.layer_norm(x, out=wrap(x))
    yield lambda: scoring.layer_norm_grad(wrap(x), x)
    yield lambda: scoring.layer_norm_grad(x, wrap(x))
    yield lambda: scoring.layer_norm_grad(x, x, wrap(v))
    for at in range(3):
        outs = [wrap(t) if i == at else t for i, t in enumerate((x, v, v))]
        yield lambda outs=outs: scoring.layer_norm_grad(
            x, x, out=scoring.LayerNormGrad.of(*outs, none, (3, 40, torch.float32, torch.float32)))
    yield lambda: scoring.DenseCatalogue(wrap(x), bits=4)


def test_gradients_are_not_lost():
    """A gradient that a call does not have is refused, not left out; under no_grad nobody asks for it."""
    for call in _calls_without_derivative(lambda t: t.clone().requires_grad_()):
        with pytest.raises(ValueError, match="requires a gradient"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="on the GPU"):
            call()


def test_tangents_are_not_lost():
    """Forward-mode derivatives are refused, those of layer_norm among them."""
    from torch.autograd import forward_ad

    from quiver import scoring

    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t.clone(), torch.ones_like(t))

        x, v = torch.zeros(3, 40), torch.zeros(40)
        calls = list(_calls_without_derivative(dual))
        for t in (lambda: dual(x), lambda: dual(x.clone().requires_grad_())):
            calls.append(lambda t=t: scoring.layer_norm(t()))
        calls.append(lambda: scoring.layer_norm(x, dual(v)))
        calls.append(lambda: scoring.layer_norm(x, v, dual(v)))
        for call in calls:
            with pytest.raises(ValueError, match="has a tangent"):
                call()
        with pytest.raises(ValueError, match="on the GPU"):
            scoring.layer_norm(x, v)
