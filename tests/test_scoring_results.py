"""Results that are written again (out=): where a tensor's memory has changed hands, calls write to what it holds now."""
from __future__ import annotations

from dataclasses import replace

import pytest
import torch


class Recorder:
    """In the library's place: takes the addresses that calls pass on."""

    def qv_layer_norm_grad_workspace(self, n, d):
        return 64

    def qv_layer_norm_grad(self, *a):
        self.grad = dict(x=a[10], stride=a[11], weight=a[12], bias=a[13], workspace=a[14])
        return 0

    def qv_log_probs_workspace(self, n, v, k):
        return 64

    def qv_log_probs(self, *a):
        self.log_probs = dict(target=a[9], entropy=a[10], logsumexp=a[11], stats=a[12], top_ids=a[13], top=a[14])
        return 0

    def qv_log_probs_grad(self, *a):
        self.log_probs_grad = dict(stats=a[6], entropy=a[7], top_ids=a[10])
        return 0


@pytest.fixture
def recorder(monkeypatch):
    from quiver import scoring

    r = Recorder()
    monkeypatch.setattr(scoring._lib, "load", lambda: r)
    monkeypatch.setattr(scoring, "_device", lambda first, *others: first.get_device())
    monkeypatch.setattr(scoring, "_raw_stream", lambda device: None)
    return r


N, D = 6, 8


def _gradients():
    from quiver import scoring

    x = torch.zeros(N, D)
    r = scoring.layer_norm_grad(x, x, torch.zeros(D))
    return lambda out=r: scoring.layer_norm_grad(x, x, torch.zeros(D), out=out), r


def _replaced(t, how):
    """Gives `t` other memory of the same shape, as torch lets a program do."""
    if how == "data":
        t.data = torch.ones_like(t)
    elif how == "set_":
        t.set_(torch.ones_like(t))
    elif how == "resize_":
        shape = t.shape
        t.resize_(1000)
        t.resize_(shape)
    elif how == "storage":
        size = t.untyped_storage().nbytes()
        t.untyped_storage().resize_(4 * size)
    elif how == "module":  # a parameter's gradient, whose module is moved there and back
        parameter = torch.nn.Parameter(torch.zeros_like(t))
        parameter.grad = t
        module = torch.nn.Module()
        module.p = parameter
        module.double().float()
        assert parameter.grad is t


@pytest.mark.parametrize("how", ["data", "set_", "resize_", "storage", "module"])
@pytest.mark.parametrize("part", ["x", "weight", "bias"])
def test_gradients_follow_their_memory(recorder, part, how):
    call, r = _gradients()
    old = getattr(r, part)
    kept, at = old.detach(), old.data_ptr()  # kept, so that its address is not given out again
    _replaced(old, how)
    assert call() is r and kept is not None
    for p in ("x", "weight", "bias"):
        assert recorder.grad[p] == getattr(r, p).data_ptr()
    assert recorder.grad[part] != at


def test_gradients_in_wider_rows(recorder):
    """A result of rows inside a wider matrix is written with its own stride."""
    call, r = _gradients()
    r.x.data = torch.zeros(N, 2 * D)[:, 3:3 + D]
    call()
    assert recorder.grad["x"] == r.x.data_ptr() and recorder.grad["stride"] == 2 * D
    r.x.data = torch.zeros(N, D)
    call()
    assert recorder.grad["x"] == r.x.data_ptr() and recorder.grad["stride"] == D
    without = replace(r, x=None)
    call(without)
    assert recorder.grad["x"] is None and recorder.grad["bias"] == r.bias.data_ptr()


@pytest.mark.parametrize("part, change, text", [
    ("weight", lambda t: t.data.half(), "out.weight must be"), ("bias", lambda t: t.data.half(), "out.bias must be"),
    ("x", lambda t: t.data.half(), "out.x has the type"), ("weight", lambda t: t.data[:D - 1], "out.weight must be"),
    ("bias", lambda t: torch.zeros(2 * D)[::2], "out.bias must be"), ("x", lambda t: t.data[:, :D - 1], "out.x has another"),
    ("x", lambda t: t.data[:N - 1], "out.x has another"), ("x", lambda t: t.data.reshape(D, N), "out.x has another"),
    ("x", lambda t: torch.zeros(D, N).T, "out.x must be contiguous"),
    ("weight", lambda t: t.data.view(torch.int32), "out.weight must be")])
def test_gradients_of_another_form_are_refused(recorder, part, change, text):
    call, r = _gradients()
    call()
    del recorder.grad
    t = getattr(r, part)
    t.data = change(t)
    with pytest.raises(ValueError, match=text):
        call()
    assert not hasattr(recorder, "grad")


def test_gradients_of_less_memory_are_refused(recorder):
    call, r = _gradients()
    r.weight.untyped_storage().resize_(8)
    with pytest.raises(ValueError, match="made smaller"):
        call()


PARTS = ("target", "entropy", "logsumexp", "top_ids", "top", "stats")


def _log_probs():
    from quiver import scoring

    new = [torch.zeros(shape, dtype=dtype) for shape, dtype in (
        ((N, 1), torch.float32), ((N,), torch.float32), ((N,), torch.float32), ((N, 2), torch.int32), ((N, 2), torch.float32),
        ((N, 2), torch.float32))]
    r = scoring.LogProbs.of(*new, 1.0, torch.zeros(64, dtype=torch.uint8))
    x, targets = torch.zeros(N, D), torch.zeros(N, 1, dtype=torch.int32)
    return (lambda: scoring.log_probs(x, targets, top_k=2, out=r),
            lambda: scoring.log_probs_grad(x, r, targets, grad_target=torch.ones(N, 1)), r)


@pytest.mark.parametrize("how", ["data", "set_", "resize_", "storage"])
@pytest.mark.parametrize("part", PARTS)
def test_log_probs_follow_their_memory(recorder, part, how):
    """... and their gradient reads what the result holds now."""
    call, gradient, r = _log_probs()
    old = getattr(r, part)
    kept, at = old.detach(), old.data_ptr()
    _replaced(old, how)
    assert call() is r and kept is not None
    for p in PARTS:
        assert recorder.log_probs[p] == getattr(r, p).data_ptr()
    assert recorder.log_probs[part] != at
    gradient()
    for p in ("stats", "entropy", "top_ids"):
        assert recorder.log_probs_grad[p] == getattr(r, p).data_ptr()


@pytest.mark.parametrize("part, change", [
    ("target", lambda t: t.data.half()), ("entropy", lambda t: t.data[:N - 1]), ("logsumexp", lambda t: torch.zeros(2 * N)[::2]),
    ("top_ids", lambda t: t.data.long()), ("top", lambda t: t.data[:, :1]), ("stats", lambda t: torch.zeros(2, N).T),
    ("entropy", lambda t: t.data.view(torch.float16))])
def test_log_probs_of_another_form_are_refused(recorder, part, change):
    call, gradient, r = _log_probs()
    call()
    gradient()
    del recorder.log_probs, recorder.log_probs_grad
    getattr(r, part).data = change(getattr(r, part))
    for f in (call, gradient):
        with pytest.raises(ValueError, match=f"out.{part} must be"):
            f()
    assert not hasattr(recorder, "log_probs") and not hasattr(recorder, "log_probs_grad")


def test_log_probs_of_less_memory_are_refused(recorder):
    call, gradient, r = _log_probs()
    r.stats.untyped_storage().resize_(8)
    for f in (call, gradient):
        with pytest.raises(ValueError, match="made smaller"):
            f()


@pytest.mark.parametrize("workspace", [torch.zeros(1, dtype=torch.uint8).expand(1 << 20), torch.zeros(2, 64, dtype=torch.uint8),
                                       torch.zeros(64, dtype=torch.uint8)[::2]])
def test_workspaces_are_whole(workspace):
    """A workspace is as many bytes as it has elements: none that repeats or skips them."""
    from quiver import scoring

    x = torch.zeros(N, D)
    with pytest.raises(ValueError, match="workspace must be"):
        scoring.LayerNormGrad.of(x, x[0], x[0], workspace, (N, D, torch.float32, torch.float32))
    with pytest.raises(ValueError, match="workspace must be"):
        scoring.LogProbs.of(x[:, :0], x[:, 0].contiguous(), x[:, 0].contiguous(), x[:, :0].int(), x[:, :0],
                            x[:, :2].contiguous(), 1.0, workspace)


def test_lent_buffers(recorder):
    """Buffers of a program's own, without a word of what a workspace is: None takes a new one."""
    from quiver import scoring

    x, weight, bias = torch.zeros(N, D), torch.zeros(D), torch.zeros(D)
    made_for = (N, D, torch.float32, torch.float32)
    for buffers in ((x, weight, bias), (x, None, None), (None, None, bias)):
        r = scoring.LayerNormGrad.of(*buffers, None, made_for)
        assert r._workspace.shape == (64,) and r._workspace.dtype == torch.uint8
        scoring.layer_norm_grad(x, torch.ones_like(x), weight, out=r)
        assert [recorder.grad[p] for p in ("x", "weight", "bias")] == [None if b is None else b.data_ptr() for b in buffers]
        assert recorder.grad["workspace"] == r._workspace.data_ptr()
    assert scoring.LayerNormGrad.workspace(N, D, "cpu").shape == (64,)
    with pytest.raises(ValueError, match="none of the gradients"):
        scoring.LayerNormGrad.of(None, None, None, None, made_for)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dim, other", [(7, 8), (8, 7), (33, 34), (8, 6)])
def test_queries_of_another_length(monkeypatch, bits, dim, other):
    """Rows of 7 values in 4 bits have as many bytes as rows of 8; queries of another length than the vectors' are refused."""
    from quiver import scoring

    def quantized(rows):
        n, d = rows.shape
        if bits == 8:
            return torch.zeros((n, d), dtype=torch.int8), torch.zeros(n)
        return torch.zeros((n, (d + 1) // 2), dtype=torch.uint8), torch.zeros((n, (d + 31) // 32), dtype=torch.uint8)

    monkeypatch.setattr(scoring, "quantize_rows" if bits == 8 else "quantize_rows_mx4", quantized)
    catalogue = scoring.DenseCatalogue(torch.zeros(5, dim), bits=bits)
    for call in (catalogue.scores, catalogue.log_probs):
        with pytest.raises(ValueError, match="dimensions"):
            call(torch.zeros(3, other))
        with pytest.raises(ValueError, match="on the GPU"):
            call(torch.zeros(3, dim))
