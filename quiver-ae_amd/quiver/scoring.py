"""Dense scores and the distribution over them, on torch tensors of one GPU.

What stands next to a graph search: scoring a whole catalogue (or a linear
layer) by inner products in 8 bits, and what a model's answer or its training
loss takes from scores -- log probabilities of the relevant columns, the
entropy, the best alternatives (a retriever's hard negatives), the gradient.

``quantize_rows``, ``int8_product``, ``log_probs`` and ``log_probs_grad`` are
the C ABI's calls (include/quiver_hip.h) on the current stream of the tensors'
GPU; none of them waits.  ``log_probs`` takes part in autograd (reverse mode);
where there is no derivative, an argument that asks for one is refused.
``DenseCatalogue`` runs them together: a catalogue kept in 8 bits, scored and
normalised for batches of queries.

Results can be handed back through ``out=`` to be written again (a loop then
allocates nothing); a result is ordered with the stream it was made on.  A wrong
argument raises ``ValueError``, a failing call ``QuiverError``; nothing here
falls back to torch.

torch brings its own HIP runtime, and a process can hold one: import torch or
this module before the library is first called (an index opened earlier has
loaded the system's).
"""
from __future__ import annotations

from dataclasses import dataclass, replace

from . import _lib

if _lib.before_torch:
    raise _lib.QuiverError("libquiver_hip was loaded before torch, so the process would hold two HIP runtimes: "
                           "import torch (or quiver.scoring) before the first call into the library")

import torch  # noqa: E402
from torch.autograd import forward_ad  # noqa: E402

_TYPES = {torch.float32: _lib.QV_FLOAT, torch.bfloat16: _lib.QV_BFLOAT16, torch.float16: _lib.QV_FLOAT16}
_CODES = (torch.int8,)

# These calls take a few microseconds on the GPU for a small batch, so the checks
# below avoid what torch's Python layer is slow at (device objects, stream objects,
# repeated shapes).
_raw_stream = torch._C._cuda_getCurrentRawStream

# For tensors given as out=: autograd then refuses a backward pass that needs what they held.
_written = torch._C._increment_version


def _device(first: torch.Tensor, *others: torch.Tensor) -> int:
    """The one GPU that every tensor is on."""
    index = first.get_device()
    for t in others:
        if t.get_device() != index:
            raise ValueError("tensors must be on one GPU")
    if index < 0:
        raise ValueError("tensors must be on the GPU")
    return index


# The two checks below are called only where an argument requires a gradient or a forward-mode level is
# entered (`forward_ad._current_level >= 0`): reading that is what the other calls pay.
def _has_tangent(*tensors: torch.Tensor | None) -> bool:
    """Whether a forward-mode derivative goes with one of them."""
    if forward_ad._current_level < 0 or not torch._C._is_fwd_grad_enabled():
        return False
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _no_derivative(call: str, *tensors: torch.Tensor | None) -> None:
    """Results are made outside autograd: a derivative that is asked for is refused, not left out."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{call} has no derivative, and an argument requires a gradient: detach it, or call "
                                 "under torch.no_grad()")
    if _has_tangent(*tensors):
        raise ValueError(f"{call} has no forward-mode derivative, and an argument has a tangent")


def _matrix(name: str, t: torch.Tensor, types) -> tuple[int, int, int]:
    """Checks a row-major matrix; its rows, columns and row stride."""
    if t.dtype not in types:
        raise ValueError(f"{name} has the type {t.dtype}; " + " or ".join(str(x) for x in types) + " is needed")
    shape = t.shape
    if len(shape) != 2:
        raise ValueError(f"{name} must have two dimensions")
    rows, cols = shape
    stride, step = t.stride()
    if step != 1 and cols > 1:
        raise ValueError(f"{name} must be contiguous along its rows")
    # one row, or none, has no stride of its own
    return rows, cols, stride if rows > 1 else max(cols, 1)


def _vector(name: str, t: torch.Tensor, shape: tuple, dtype=torch.float32) -> int:
    if t.dtype != dtype or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {shape}")
    return t.data_ptr()


def quantize_rows(x: torch.Tensor, *, out: tuple[torch.Tensor, torch.Tensor] | None = None):
    """``(codes int8 [n, d], scales float32 [n])`` with ``x[i] ~ codes[i] * scales[i]``.

    scales[i] = max_j |x[i, j]| / 127; codes are rounded to the nearest whole
    number, halves to even.  A row of zeros (below 2^-119) has the scale 0, a
    row with an infinity or a NaN the scale NaN and zero codes.
    """
    n, d, stride = _matrix("x", x, _TYPES)
    again = out is not None
    if x.requires_grad or again and out[1].requires_grad or forward_ad._current_level >= 0:
        _no_derivative("quantize_rows", x, out[1] if again else None)
    if not again:
        out = (torch.empty((n, d), dtype=torch.int8, device=x.device),
               torch.empty(n, dtype=torch.float32, device=x.device))
    codes, scales = out
    code_rows, code_cols, code_stride = _matrix("codes", codes, _CODES)
    if code_rows != n or code_cols != d:
        raise ValueError("codes and x differ in shape")
    at = _vector("scales", scales, (n,))
    device = _device(x, codes, scales)
    _lib.check(_lib.load().qv_quantize_rows(x.data_ptr(), _TYPES[x.dtype], n, d, stride, codes.data_ptr(), code_stride,
                                            at, device, _raw_stream(device)))
    if again:
        _written(out)
    return out


def int8_product(a: torch.Tensor, a_scales: torch.Tensor, b: torch.Tensor, b_scales: torch.Tensor, *,
                 bias: torch.Tensor | None = None, dtype: torch.dtype | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """``(a . b^T) * a_scales[:, None] * b_scales[None, :] + bias`` of int8 ``a`` [m, k] and ``b`` [n, k].

    The sums are exact; the rest is fp32, rounded once to ``dtype`` (``out``'s
    type, or float32).  A bias of -inf takes a column out of ``log_probs``.
    """
    m, k, a_stride = _matrix("a", a, _CODES)
    n, k_b, b_stride = _matrix("b", b, _CODES)
    if k_b != k:
        raise ValueError("a and b differ in the length of their rows")
    again = out is not None
    if (a_scales.requires_grad or b_scales.requires_grad or bias is not None and bias.requires_grad
            or again and out.requires_grad or forward_ad._current_level >= 0):
        _no_derivative("int8_product", a_scales, b_scales, bias, out)
    if not again:
        if dtype is None:
            dtype = torch.float32
        elif dtype not in _TYPES:
            raise ValueError("dtype must be float32, bfloat16 or float16")
        out = torch.empty((m, n), dtype=dtype, device=a.device)
    elif dtype is not None and out.dtype != dtype:
        raise ValueError(f"out has the type {out.dtype}, and {dtype} is asked for")
    out_rows, out_cols, out_stride = _matrix("out", out, _TYPES)
    if out_rows != m or out_cols != n:
        raise ValueError(f"out must have the shape {(m, n)}")
    at_a, at_b = _vector("a_scales", a_scales, (m,)), _vector("b_scales", b_scales, (n,))
    if bias is None:
        at_bias, device = None, _device(a, a_scales, b, b_scales, out)
    else:
        at_bias, device = _vector("bias", bias, (n,)), _device(a, a_scales, b, b_scales, out, bias)
    _lib.check(_lib.load().qv_int8_product(a.data_ptr(), a_stride, at_a, m, b.data_ptr(), b_stride, at_b, at_bias, n, k,
                                           out.data_ptr(), _TYPES[out.dtype], out_stride, device, _raw_stream(device)))
    if again:
        _written((out,))
    return out


@dataclass(frozen=True, eq=False)
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
    _device: int
    _parts: tuple            # the buffers in the order above, the workspace last
    _at: tuple               # their addresses
    _size: tuple             # rows, targets and alternatives per row, bytes of the workspace

    @staticmethod
    def empty(n: int, v: int, t: int, k: int, temperature: float, device: torch.device) -> "LogProbs":
        """Buffers for ``log_probs`` of n rows of v columns with t targets and k alternatives."""
        if not 0 <= k <= _lib.QV_LOG_PROBS_MAX_TOPK:
            raise ValueError(f"top_k must be in [0, {_lib.QV_LOG_PROBS_MAX_TOPK}]")
        if t > _lib.QV_LOG_PROBS_MAX_TARGETS:
            raise ValueError(f"at most {_lib.QV_LOG_PROBS_MAX_TARGETS} targets per row")
        if device.type != "cuda":
            raise ValueError("tensors must be on the GPU")

        workspace = _lib.load().qv_log_probs_workspace(n, v, k)
        if workspace < 0:
            _lib.check(workspace)

        def new(*shape, dtype=torch.float32):
            return torch.empty(shape, dtype=dtype, device=device)

        return LogProbs.of(new(n, t), new(n), new(n), new(n, k, dtype=torch.int32), new(n, k), new(n, 2), temperature,
                           new(workspace, dtype=torch.uint8))

    @staticmethod
    def of(target, entropy, logsumexp, top_ids, top, stats, temperature, workspace) -> "LogProbs":
        parts = (target, entropy, logsumexp, top_ids, top, stats, workspace)
        return LogProbs(target, entropy, logsumexp, top_ids, top, stats, temperature, workspace, stats.get_device(),
                        parts, tuple(p.data_ptr() for p in parts), (*target.shape, top.shape[1], workspace.shape[0]))


def _given(targets: torch.Tensor | None, rows: int) -> tuple[int | None, int]:
    """(address, columns per row) of int32 targets [n, t] or [n]."""
    if targets is None:
        return None, 0
    shape = targets.shape
    per_row = shape[1] if len(shape) == 2 else 1
    return _vector("targets", targets, (rows, per_row) if len(shape) == 2 else (rows,), torch.int32), per_row


def _forward(logits, targets, top_k, temperature, out) -> LogProbs:
    n, v, stride = _matrix("logits", logits, _TYPES)
    at_targets, t = _given(targets, n)
    temperature = float(temperature)
    again = out is not None
    if not again:
        out = LogProbs.empty(n, v, t, top_k, temperature, logits.device)
    elif out._size[:3] != (n, t, top_k):
        raise ValueError("out was made for another number of rows, targets or alternatives")
    elif out.temperature != temperature:
        out = replace(out, temperature=temperature)
    device = _device(logits) if targets is None else _device(logits, targets)
    if device != out._device:
        raise ValueError("tensors must be on one GPU")
    at_target, at_entropy, at_lse, at_ids, at_top, at_stats, at_work = out._at
    _lib.check(_lib.load().qv_log_probs(logits.data_ptr(), _TYPES[logits.dtype], n, v, stride, temperature, at_targets,
                                        t, top_k, at_target, at_entropy, at_lse, at_stats, at_ids, at_top, at_work,
                                        out._size[3], device, _raw_stream(device)))
    if again:
        _written(out._parts)
    return out


class _Once(torch.autograd.Function):
    """A gradient made while a graph is recorded: there is no derivative of it, and taking one must not give zeros."""

    @staticmethod
    def forward(ctx, grad, *inputs):
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, _g):
        raise _lib.QuiverError("the gradient of log_probs cannot be differentiated again")


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

        if _has_tangent(g_target, g_entropy, g_lse, g_top):
            raise _lib.QuiverError("the gradient of log_probs has no forward-mode derivative")

        def plain(g):
            return None if g is None else g.contiguous()

        grad = _gradient(logits, stats.data_ptr(), entropy.data_ptr(), top_ids.data_ptr(), top_ids.shape[1],
                         logits.get_device(), ctx.temperature, targets, plain(g_target), plain(g_entropy), plain(g_lse),
                         plain(g_top), None)
        if torch.is_grad_enabled():
            grad = _Once.apply(grad, logits, *(g for g in (g_target, g_entropy, g_lse, g_top) if g is not None))
        return grad, None, None, None


def log_probs(logits: torch.Tensor, targets: torch.Tensor | None = None, *, top_k: int = 0, temperature: float = 1.0,
              out: LogProbs | None = None) -> LogProbs:
    """The softmax distribution of each row of ``logits / temperature`` (float32, bfloat16 or float16 [n, v]).

    ``targets``: int32 [n, t] or [n], the columns whose log probabilities are
    wanted; a negative one is absent (0, no gradient), one past the row's end
    gives NaN (and the row a gradient of NaN unless its weight is 0).  ``top_k``
    (up to 64) columns with the largest logits come in descending order, the
    lower column first among equal ones.  -inf takes a column out; a row with
    none left has log probabilities -inf, entropy 0 and ids -1, one that holds
    +inf or NaN has NaN.  With logits that require a gradient the results take
    part in autograd (``out`` is then refused), once: the gradient has none of
    its own, and there is no forward-mode derivative.
    """
    if logits.requires_grad and torch.is_grad_enabled():
        if out is not None:
            raise ValueError("out= cannot be given for logits that require a gradient")
        if _has_tangent(logits):
            raise ValueError("log_probs has no forward-mode derivative, and logits has a tangent")
        target, entropy, lse, ids, top, stats, workspace = _LogProbsFunction.apply(logits, targets, top_k,
                                                                                  float(temperature))
        return LogProbs.of(target, entropy, lse, ids, top, stats, float(temperature), workspace)
    if out is not None and out.entropy.requires_grad or forward_ad._current_level >= 0:
        _no_derivative("log_probs", logits, None if out is None else out.entropy)
    return _forward(logits, targets, top_k, temperature, out)


def _gradient(logits, at_stats, at_entropy, at_ids, k, device, temperature, targets, g_target, g_entropy, g_lse, g_top,
              out):
    n, v, stride = _matrix("logits", logits, _TYPES)
    at_targets, t = _given(targets, n)
    again = out is not None
    if not again:
        out = torch.empty((n, v), dtype=logits.dtype, device=logits.device)
    out_rows, out_cols, out_stride = _matrix("out", out, (logits.dtype,))
    if out_rows != n or out_cols != v:
        raise ValueError("out and logits differ in shape")
    tensors = [logits, out]
    if targets is not None:
        tensors.append(targets)

    def given(name, g, shape):
        if g is None:
            return None
        tensors.append(g)
        return _vector(name, g, shape)

    at = (given("grad_target", g_target, (n, t)), given("grad_entropy", g_entropy, (n,)),
          given("grad_logsumexp", g_lse, (n,)), given("grad_top", g_top, (n, k)))
    if _device(*tensors) != device:
        raise ValueError("tensors must be on one GPU")
    _lib.check(_lib.load().qv_log_probs_grad(logits.data_ptr(), _TYPES[logits.dtype], n, v, stride, temperature,
                                             at_stats, at_entropy, at_targets, t, at_ids, k, *at, out.data_ptr(),
                                             out_stride, device, _raw_stream(device)))
    if again:
        _written((out,))
    return out


def log_probs_grad(logits: torch.Tensor, result: LogProbs, targets: torch.Tensor | None = None, *,
                   grad_target: torch.Tensor | None = None, grad_entropy: torch.Tensor | None = None,
                   grad_logsumexp: torch.Tensor | None = None, grad_top: torch.Tensor | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """The gradient of a loss with respect to ``logits``, from its gradients with respect to ``result``'s parts.

    ``result`` and ``targets`` as they were for ``log_probs``; ``out`` may be
    the logits themselves.  What autograd runs, for training loops without it
    (so logits that require a gradient come detached, or under
    ``torch.no_grad()``).
    """
    if (logits.requires_grad or grad_target is not None and grad_target.requires_grad
            or grad_entropy is not None and grad_entropy.requires_grad
            or grad_logsumexp is not None and grad_logsumexp.requires_grad
            or grad_top is not None and grad_top.requires_grad or out is not None and out.requires_grad
            or forward_ad._current_level >= 0):
        _no_derivative("log_probs_grad", logits, grad_target, grad_entropy, grad_logsumexp, grad_top, out)
    if result.entropy.shape[0] != logits.shape[0]:
        raise ValueError("result was made for another number of rows")
    _, at_entropy, _, at_ids, _, at_stats, _ = result._at
    return _gradient(logits, at_stats, at_entropy, at_ids, result.top.shape[1], result._device, result.temperature,
                     targets, grad_target, grad_entropy, grad_logsumexp, grad_top, out)


class DenseCatalogue:
    """Embedding vectors kept in 8 bits and scored exhaustively.

    ``DenseCatalogue(vectors)`` quantises the rows once.  ``log_probs(queries,
    targets, ...)`` gives each query's distribution over all of them, by inner
    products; the scores exist for one batch of queries at a time, about
    ``score_bytes`` of them.  Scores have no derivative (vectors, queries or a
    bias that require a gradient are refused).
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
        """Inner products of the queries, quantised row by row, with every vector: [n, len(self)], of ``out``'s type if given."""
        codes, scales = quantize_rows(queries)
        return int8_product(codes, scales, self.codes, self.scales, bias=self.bias,
                            dtype=self.score_dtype if out is None else None, out=out)

    def log_probs(self, queries: torch.Tensor, targets: torch.Tensor | None = None, *, top_k: int = 0,
                  temperature: float = 1.0) -> LogProbs:
        """``log_probs`` of the scores, batch by batch of the queries."""
        n = queries.shape[0]
        _given(targets, n)  # of all batches at once: rows past the queries' would be left out
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
        return LogProbs.of(*joined, float(temperature), parts[-1]._workspace)
