"""Dense scores and the distribution over them, on torch tensors of one GPU.

What stands next to a graph search: scoring a whole catalogue (or a linear
layer) by inner products in 8 bits, and what a model's answer or its training
loss takes from scores -- log probabilities of the relevant columns, the
entropy, the best alternatives (a retriever's hard negatives), the gradient.

``quantize_rows``, ``int8_product``, ``log_probs`` and ``log_probs_grad`` are
the C ABI's calls (include/quiver_hip.h) on the current stream of the tensors'
GPU; none of them waits.  ``log_probs`` takes part in autograd.
``DenseCatalogue`` runs them together: a catalogue kept in 8 bits, scored and
normalised for batches of queries.

Results can be handed back through ``out=`` to be written again (a loop then
allocates nothing); a result is ordered with the stream it was made on.  A wrong
argument raises ``ValueError``, a failing call ``QuiverError``; nothing here
falls back to torch.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib

_TYPES = {torch.float32: _lib.QV_FLOAT, torch.bfloat16: _lib.QV_BFLOAT16, torch.float16: _lib.QV_FLOAT16}


def _device(*tensors: torch.Tensor) -> int:
    """The one GPU that every tensor is on."""
    index = None
    for t in tensors:
        if not t.is_cuda:
            raise ValueError("tensors must be on the GPU")
        if index is None:
            index = t.get_device()
        elif t.get_device() != index:
            raise ValueError("tensors must be on one GPU")
    return index


def _stream(device: int) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _matrix(name: str, t: torch.Tensor, types) -> int:
    """Checks a row-major matrix; its row stride."""
    if t.dtype not in types:
        raise ValueError(f"{name} has the type {t.dtype}; " + " or ".join(str(x) for x in types) + " is needed")
    if t.dim() != 2:
        raise ValueError(f"{name} must have two dimensions")
    rows, cols = t.shape
    if cols > 1 and t.stride(1) != 1:
        raise ValueError(f"{name} must be contiguous along its rows")
    # one row, or none, has no stride of its own
    return t.stride(0) if rows > 1 else max(cols, 1)


def _vector(name: str, t: torch.Tensor, shape, dtype=torch.float32) -> int:
    if t.dtype != dtype or tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)}")
    return t.data_ptr()


def quantize_rows(x: torch.Tensor, *, out: tuple[torch.Tensor, torch.Tensor] | None = None):
    """``(codes int8 [n, d], scales float32 [n])`` with ``x[i] ~ codes[i] * scales[i]``.

    scales[i] = max_j |x[i, j]| / 127; codes are rounded to the nearest whole
    number, halves to even.  A row of zeros (below 2^-119) has the scale 0, a
    row with an infinity or a NaN the scale NaN and zero codes.
    """
    stride = _matrix("x", x, _TYPES)
    n, d = x.shape
    if out is None:
        out = (torch.empty((n, d), dtype=torch.int8, device=x.device),
               torch.empty(n, dtype=torch.float32, device=x.device))
    codes, scales = out
    code_stride = _matrix("codes", codes, (torch.int8,))
    if codes.shape != x.shape:
        raise ValueError("codes and x differ in shape")
    at = _vector("scales", scales, (n,))
    device = _device(x, codes, scales)
    _lib.check(_lib.load().qv_quantize_rows(x.data_ptr(), _TYPES[x.dtype], n, d, stride, codes.data_ptr(), code_stride,
                                            at, device, _stream(device)))
    return out


def int8_product(a: torch.Tensor, a_scales: torch.Tensor, b: torch.Tensor, b_scales: torch.Tensor, *,
                 bias: torch.Tensor | None = None, dtype: torch.dtype = torch.float32,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """``(a . b^T) * a_scales[:, None] * b_scales[None, :] + bias`` of int8 ``a`` [m, k] and ``b`` [n, k].

    The sums are exact; the rest is fp32, rounded once to ``dtype``.  A bias of
    -inf takes a column out of ``log_probs``.
    """
    a_stride, b_stride = _matrix("a", a, (torch.int8,)), _matrix("b", b, (torch.int8,))
    (m, k), n = a.shape, b.shape[0]
    if b.shape[1] != k:
        raise ValueError("a and b differ in the length of their rows")
    if out is None:
        if dtype not in _TYPES:
            raise ValueError("dtype must be float32, bfloat16 or float16")
        out = torch.empty((m, n), dtype=dtype, device=a.device)
    out_stride = _matrix("out", out, _TYPES)
    if tuple(out.shape) != (m, n):
        raise ValueError(f"out must have the shape {(m, n)}")
    at_a, at_b = _vector("a_scales", a_scales, (m,)), _vector("b_scales", b_scales, (n,))
    tensors = [a, a_scales, b, b_scales, out]
    at_bias = None
    if bias is not None:
        at_bias = _vector("bias", bias, (n,))
        tensors.append(bias)
    device = _device(*tensors)
    _lib.check(_lib.load().qv_int8_product(a.data_ptr(), a_stride, at_a, m, b.data_ptr(), b_stride, at_b, at_bias, n, k,
                                           out.data_ptr(), _TYPES[out.dtype], out_stride, device, _stream(device)))
    return out


@dataclass
class LogProbs:
    """What ``log_probs`` gives; ``stats`` is what its gradient needs again."""

    target: torch.Tensor     # [n, t] log probabilities of the given columns
    entropy: torch.Tensor    # [n] natural units
    logsumexp: torch.Tensor  # [n] of logits / temperature
    top_ids: torch.Tensor    # [n, k] int32, -1 past the columns above -inf
    top: torch.Tensor        # [n, k] their log probabilities
    stats: torch.Tensor      # [n, 2] largest logit, ln of the sum of exp((x - it) / temperature)
    temperature: float
    _workspace: torch.Tensor


def _given(targets: torch.Tensor | None, rows: int) -> tuple[int | None, int]:
    """(address, columns per row) of int32 targets [n, t] or [n]."""
    if targets is None:
        return None, 0
    per_row = targets.shape[1] if targets.dim() == 2 else 1
    shape = (rows, per_row) if targets.dim() == 2 else (rows,)
    return _vector("targets", targets, shape, torch.int32), per_row


def _forward(logits, targets, top_k, temperature, out) -> LogProbs:
    stride = _matrix("logits", logits, _TYPES)
    n, v = logits.shape
    at_targets, t = _given(targets, n)
    temperature = float(temperature)
    lib = _lib.load()
    if out is None:
        if not 0 <= top_k <= _lib.QV_LOG_PROBS_MAX_TOPK:
            raise ValueError(f"top_k must be in [0, {_lib.QV_LOG_PROBS_MAX_TOPK}]")
        if t > _lib.QV_LOG_PROBS_MAX_TARGETS:
            raise ValueError(f"at most {_lib.QV_LOG_PROBS_MAX_TARGETS} targets per row")

        def empty(*shape, dtype=torch.float32):
            return torch.empty(shape, dtype=dtype, device=logits.device)

        out = LogProbs(empty(n, t), empty(n), empty(n), empty(n, top_k, dtype=torch.int32), empty(n, top_k),
                       empty(n, 2), temperature,
                       empty(lib.qv_log_probs_workspace(n, v, top_k), dtype=torch.uint8))
    out.temperature = temperature
    at_target, at_top = _vector("out.target", out.target, (n, t)), _vector("out.top", out.top, (n, top_k))
    at_ids = _vector("out.top_ids", out.top_ids, (n, top_k), torch.int32)
    at_entropy, at_lse = _vector("out.entropy", out.entropy, (n,)), _vector("out.logsumexp", out.logsumexp, (n,))
    at_stats = _vector("out.stats", out.stats, (n, 2))
    device = _device(logits, out.target, out.entropy, out.logsumexp, out.top, out.top_ids, out.stats, out._workspace,
                     *(() if targets is None else (targets,)))
    _lib.check(lib.qv_log_probs(logits.data_ptr(), _TYPES[logits.dtype], n, v, stride, temperature, at_targets, t,
                                top_k, at_target, at_entropy, at_lse, at_stats, at_ids, at_top,
                                out._workspace.data_ptr(), out._workspace.numel(), device, _stream(device)))
    return out


class _LogProbsFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top_k, temperature):
        r = _forward(logits, targets, top_k, temperature, None)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(r.top_ids, r.stats, r._workspace)
        ctx.save_for_backward(logits, targets, r.stats, r.entropy, r.top_ids)
        return r.target, r.entropy, r.logsumexp, r.top_ids, r.top, r.stats, r._workspace

    @staticmethod
    def backward(ctx, g_target, g_entropy, g_lse, _ids, g_top, _stats, _workspace):
        logits, targets, stats, entropy, top_ids = ctx.saved_tensors

        def plain(g):
            return None if g is None else g.contiguous()

        grad = _gradient(logits, stats, entropy, top_ids, ctx.temperature, targets, plain(g_target),
                         plain(g_entropy), plain(g_lse), plain(g_top), None)
        return grad, None, None, None


def log_probs(logits: torch.Tensor, targets: torch.Tensor | None = None, *, top_k: int = 0, temperature: float = 1.0,
              out: LogProbs | None = None) -> LogProbs:
    """The softmax distribution of each row of ``logits / temperature`` (float32, bfloat16 or float16 [n, v]).

    ``targets``: int32 [n, t] or [n], the columns whose log probabilities are
    wanted; a negative one is absent (0, no gradient), one past the row's end
    gives NaN.  ``top_k`` (up to 64) columns with the largest logits come in
    descending order, the lower column first among equal ones.  -inf takes a
    column out; a row with none left has log probabilities -inf, entropy 0 and
    ids -1, one that holds +inf or NaN has NaN.  With logits that require a
    gradient the results take part in autograd (``out`` is then refused).
    """
    if torch.is_grad_enabled() and logits.requires_grad:
        if out is not None:
            raise ValueError("out= cannot be given for logits that require a gradient")
        target, entropy, lse, ids, top, stats, workspace = _LogProbsFunction.apply(logits, targets, top_k,
                                                                                  float(temperature))
        return LogProbs(target, entropy, lse, ids, top, stats, float(temperature), workspace)
    return _forward(logits, targets, top_k, temperature, out)


def _gradient(logits, stats, entropy, top_ids, temperature, targets, g_target, g_entropy, g_lse, g_top, out):
    stride = _matrix("logits", logits, _TYPES)
    n, v = logits.shape
    at_targets, t = _given(targets, n)
    k = top_ids.shape[1]
    if out is None:
        out = torch.empty((n, v), dtype=logits.dtype, device=logits.device)
    out_stride = _matrix("out", out, (logits.dtype,))
    if out.shape != logits.shape:
        raise ValueError("out and logits differ in shape")
    at_stats, at_entropy = _vector("stats", stats, (n, 2)), _vector("entropy", entropy, (n,))
    at_ids = _vector("top_ids", top_ids, (n, k), torch.int32)
    tensors, given = [logits, out, stats, entropy, top_ids], []
    if targets is not None:
        tensors.append(targets)
    for name, g, shape in (("grad_target", g_target, (n, t)), ("grad_entropy", g_entropy, (n,)),
                           ("grad_logsumexp", g_lse, (n,)), ("grad_top", g_top, (n, k))):
        given.append(None if g is None else _vector(name, g, shape))
        if g is not None:
            tensors.append(g)
    device = _device(*tensors)
    _lib.check(_lib.load().qv_log_probs_grad(logits.data_ptr(), _TYPES[logits.dtype], n, v, stride, temperature,
                                             at_stats, at_entropy, at_targets, t, at_ids, k, *given, out.data_ptr(),
                                             out_stride, device, _stream(device)))
    return out


def log_probs_grad(logits: torch.Tensor, result: LogProbs, targets: torch.Tensor | None = None, *,
                   grad_target: torch.Tensor | None = None, grad_entropy: torch.Tensor | None = None,
                   grad_logsumexp: torch.Tensor | None = None, grad_top: torch.Tensor | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """The gradient of a loss with respect to ``logits``, from its gradients with respect to ``result``'s parts.

    ``result`` and ``targets`` as they were for ``log_probs``; ``out`` may be
    the logits themselves.  What autograd runs, for training loops without it.
    """
    return _gradient(logits, result.stats, result.entropy, result.top_ids, result.temperature, targets, grad_target,
                     grad_entropy, grad_logsumexp, grad_top, out)


class DenseCatalogue:
    """Embedding vectors kept in 8 bits and scored exhaustively.

    ``DenseCatalogue(vectors)`` quantises the rows once.  ``log_probs(queries,
    targets, ...)`` gives each query's distribution over all of them, by inner
    products; the scores exist for one batch of queries at a time, about
    ``score_bytes`` of them.
    """

    def __init__(self, vectors: torch.Tensor, *, bias: torch.Tensor | None = None,
                 score_dtype: torch.dtype = torch.float32, score_bytes: int = 1 << 30) -> None:
        if score_dtype not in _TYPES:
            raise ValueError("score_dtype must be float32, bfloat16 or float16")
        if score_bytes <= 0:
            raise ValueError("score_bytes must be positive")
        self.codes, self.scales = quantize_rows(vectors)
        if bias is not None:
            _vector("bias", bias, (vectors.shape[0],))
        self.bias, self.score_dtype, self.score_bytes = bias, score_dtype, int(score_bytes)

    def __len__(self) -> int:
        return self.codes.shape[0]

    def scores(self, queries: torch.Tensor, *, out: torch.Tensor | None = None) -> torch.Tensor:
        """Inner products of the queries, quantised row by row, with every vector: [n, len(self)]."""
        codes, scales = quantize_rows(queries)
        return int8_product(codes, scales, self.codes, self.scales, bias=self.bias, dtype=self.score_dtype, out=out)

    def log_probs(self, queries: torch.Tensor, targets: torch.Tensor | None = None, *, top_k: int = 0,
                  temperature: float = 1.0) -> LogProbs:
        """``log_probs`` of the scores, batch by batch of the queries."""
        n = queries.shape[0]
        row_bytes = max(1, len(self)) * torch.empty((), dtype=self.score_dtype).element_size()
        step = max(1, min(n, self.score_bytes // row_bytes))
        if n <= step:
            return log_probs(self.scores(queries), targets, top_k=top_k, temperature=temperature)
        scores = torch.empty((step, len(self)), dtype=self.score_dtype, device=queries.device)
        parts = []
        for at in range(0, n, step):
            here = queries[at:at + step]
            s = self.scores(here, out=scores[:here.shape[0]])
            parts.append(log_probs(s, None if targets is None else targets[at:at + step], top_k=top_k,
                                   temperature=temperature))
        joined = [torch.cat([getattr(p, f) for p in parts])
                  for f in ("target", "entropy", "logsumexp", "top_ids", "top", "stats")]
        return LogProbs(*joined, float(temperature), parts[-1]._workspace)
