"""Dense scores and the distribution over them, on torch tensors of one GPU.

What stands next to a graph search: scoring a whole catalogue (or a linear
layer) by inner products in 8 bits or in microscaled 4 bits, what a model's
answer or its training loss takes from scores -- log probabilities of the
relevant columns, the entropy, the best alternatives (a retriever's hard
negatives), the gradient -- and the layer norm that embeddings come from.

``quantize_rows``, ``int8_product``, ``quantize_rows_mx4``, ``mx4_values``,
``mx4_product``, ``log_probs``, ``log_probs_grad``, ``layer_norm`` and
``layer_norm_grad`` are the C ABI's calls (include/quiver_hip.h) on the current
stream of the tensors' GPU; none of them waits.  ``log_probs`` and
``layer_norm`` take part in autograd (reverse mode); where there is no
derivative, an argument that asks for one is refused.  ``DenseCatalogue`` runs
them together: a catalogue kept in 8 or 4 bits, scored and normalised for
batches of queries.

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
_PACKED = (torch.uint8,)

# These calls take a few microseconds on the GPU for a small batch, so the checks
# below avoid what torch's Python layer is slow at (device objects, stream objects,
# repeated shapes).
_raw_stream = torch._C._cuda_getCurrentRawStream

# Of results that are kept with their addresses.
_address, _count = torch.Tensor.data_ptr, torch.Tensor.numel

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


def _whole(t: torch.Tensor) -> None:
    """Refuses a tensor whose memory was cut below its elements (``untyped_storage().resize_``)."""
    last = t.storage_offset() + sum((size - 1) * step for size, step in zip(t.shape, t.stride()))
    if t.numel() and (last + 1) * t.element_size() > t.untyped_storage().nbytes():
        raise ValueError("a result's memory was made smaller than the result")


def _bytes(workspace: torch.Tensor) -> None:
    """A workspace's elements are counted as its bytes: they have to be there, one behind the other."""
    if workspace.dim() != 1 or not workspace.is_contiguous():
        raise ValueError("a workspace must be a contiguous vector")


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


def _packed(name: str, codes: torch.Tensor, scales: torch.Tensor, scales_name: str = "scales"):
    """Checks rows of 4-bit codes and their scales: rows, bytes of codes in a row, both row strides."""
    rows, cols, stride = _matrix(name, codes, _PACKED)
    scale_rows, blocks, scale_stride = _matrix(scales_name, scales, _PACKED)
    if scale_rows != rows or blocks != (cols + 15) // 16:
        raise ValueError(f"{scales_name} must have the shape {(rows, (cols + 15) // 16)}, one for each 16 bytes of {name}")
    return rows, cols, stride, scale_stride


def quantize_rows_mx4(x: torch.Tensor, *, out: tuple[torch.Tensor, torch.Tensor] | None = None):
    """``(codes uint8 [n, ceil(d / 2)], scales uint8 [n, ceil(d / 32)])``: rows in microscaled 4-bit floating point.

    Each 32 values of a row share a power of two, 2^(scale - 127), the least of
    which their largest magnitude is 7 times at most; a code is a sign and one of
    0, 0.5, 1, 1.5, 2, 3, 4, 6, the nearest to the scaled value, halves to the even
    code.  Two codes to a byte, the first in its low half; a row of odd length
    ends with a zero code.  Blocks with an infinity or a NaN get the scale 255
    (NaN) and zero codes.
    """
    n, d, stride = _matrix("x", x, _TYPES)
    if x.requires_grad or forward_ad._current_level >= 0:
        _no_derivative("quantize_rows_mx4", x)
    again = out is not None
    if not again:
        out = (torch.empty((n, (d + 1) // 2), dtype=torch.uint8, device=x.device),
               torch.empty((n, (d + 31) // 32), dtype=torch.uint8, device=x.device))
    codes, scales = out
    rows, cols, code_stride, scale_stride = _packed("codes", codes, scales)
    if rows != n or cols != (d + 1) // 2:
        raise ValueError(f"codes must have the shape {(n, (d + 1) // 2)}")
    device = _device(x, codes, scales)
    _lib.check(_lib.load().qv_quantize_rows_mx4(x.data_ptr(), _TYPES[x.dtype], n, d, stride, codes.data_ptr(), code_stride,
                                                scales.data_ptr(), scale_stride, device, _raw_stream(device)))
    if again:
        _written(out)
    return out


def _result(name: str, rows: int, cols: int, dtype: torch.dtype | None, out: torch.Tensor | None, device) -> torch.Tensor:
    """``out``, which has to be of the type asked for, or a new matrix of it (float32 without)."""
    if out is None:
        if dtype is None:
            dtype = torch.float32
        elif dtype not in _TYPES:
            raise ValueError("dtype must be float32, bfloat16 or float16")
        return torch.empty((rows, cols), dtype=dtype, device=device)
    if dtype is not None and out.dtype != dtype:
        raise ValueError(f"{name} has the type {out.dtype}, and {dtype} is asked for")
    return out


def mx4_values(codes: torch.Tensor, scales: torch.Tensor, dim: int | None = None, *, dtype: torch.dtype | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """What ``quantize_rows_mx4``'s rows stand for, [n, dim] of ``dtype`` (``out``'s type, or float32).

    ``dim``: the rows' length, twice the bytes of their codes if it is not given.
    """
    n, cols, code_stride, scale_stride = _packed("codes", codes, scales)
    if dim is None:
        dim = 2 * cols
    elif (dim + 1) // 2 != cols:
        raise ValueError(f"rows of {dim} values have {(dim + 1) // 2} bytes of codes, not {cols}")
    if out is not None and out.requires_grad or forward_ad._current_level >= 0:
        _no_derivative("mx4_values", out)
    again = out is not None
    out = _result("out", n, dim, dtype, out, codes.device)
    rows, columns, stride = _matrix("out", out, _TYPES)
    if rows != n or columns != dim:
        raise ValueError(f"out must have the shape {(n, dim)}")
    device = _device(codes, scales, out)
    _lib.check(_lib.load().qv_mx4_values(codes.data_ptr(), code_stride, scales.data_ptr(), scale_stride, n, dim,
                                         out.data_ptr(), _TYPES[out.dtype], stride, device, _raw_stream(device)))
    if again:
        _written((out,))
    return out


def mx4_product(a: torch.Tensor, a_scales: torch.Tensor, b: torch.Tensor, b_scales: torch.Tensor, *,
                bias: torch.Tensor | None = None, dtype: torch.dtype | None = None,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """``A . B^T + bias`` of the rows that ``a`` and ``b`` stand for (``quantize_rows_mx4``).

    Products are exact, their sums and the bias fp32, rounded once to ``dtype``
    (``out``'s type, or float32).  A bias of -inf takes a column out of ``log_probs``.
    """
    m, cols, a_stride, a_scale_stride = _packed("a", a, a_scales, "a_scales")
    n, b_cols, b_stride, b_scale_stride = _packed("b", b, b_scales, "b_scales")
    if b_cols != cols:
        raise ValueError("a and b differ in the length of their rows")
    again = out is not None
    if bias is not None and bias.requires_grad or again and out.requires_grad or forward_ad._current_level >= 0:
        _no_derivative("mx4_product", bias, out)
    out = _result("out", m, n, dtype, out, a.device)
    out_rows, out_cols, out_stride = _matrix("out", out, _TYPES)
    if out_rows != m or out_cols != n:
        raise ValueError(f"out must have the shape {(m, n)}")
    if bias is None:
        at_bias, device = None, _device(a, a_scales, b, b_scales, out)
    else:
        at_bias, device = _vector("bias", bias, (n,)), _device(a, a_scales, b, b_scales, out, bias)
    _lib.check(_lib.load().qv_mx4_product(a.data_ptr(), a_stride, a_scales.data_ptr(), a_scale_stride, m, b.data_ptr(),
                                          b_stride, b_scales.data_ptr(), b_scale_stride, at_bias, n, 2 * cols,
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
    _at: tuple               # addresses of the buffers in the order above, the workspace last
    _counts: tuple           # of their elements, but the workspace's
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
        _bytes(workspace)
        return LogProbs(*parts[:-1], temperature, workspace, stats.get_device(), tuple(map(_address, parts)),
                        tuple(map(_count, parts[:-1])), (*target.shape, top.shape[1], workspace.shape[0]))

    def _parts(self) -> tuple:
        return self.target, self.entropy, self.logsumexp, self.top_ids, self.top, self.stats, self._workspace

    def _now(self) -> tuple:
        """(addresses, device), taken again where a tensor is no longer what they were taken of: its memory can be
        another's after ``t.data = ...``, ``set_`` or ``resize_``."""
        a, b, c, d, e, f, g = parts = self._parts()
        if ((a.data_ptr(), b.data_ptr(), c.data_ptr(), d.data_ptr(), e.data_ptr(), f.data_ptr(), g.data_ptr()) == self._at
                and (a.numel(), b.numel(), c.numel(), d.numel(), e.numel(), f.numel()) == self._counts):
            return self._at, self._device
        n, t, k, nbytes = self._size
        ids, number = torch.int32, torch.float32
        for name, part, shape, dtype in zip(("target", "entropy", "logsumexp", "top_ids", "top", "stats", "workspace"), parts,
                                            ((n, t), (n,), (n,), (n, k), (n, k), (n, 2), (nbytes,)),
                                            (number, number, number, ids, number, number, self._workspace.dtype)):
            _vector(f"out.{name}", part, shape, dtype)
            _whole(part)
            if part.get_device() != parts[0].get_device():
                raise ValueError("tensors must be on one GPU")
        return tuple(map(_address, parts)), parts[0].get_device()


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
    at, made_on = out._now() if again else (out._at, out._device)
    if device != made_on:
        raise ValueError("tensors must be on one GPU")
    at_target, at_entropy, at_lse, at_ids, at_top, at_stats, at_work = at
    _lib.check(_lib.load().qv_log_probs(logits.data_ptr(), _TYPES[logits.dtype], n, v, stride, temperature, at_targets,
                                        t, top_k, at_target, at_entropy, at_lse, at_stats, at_ids, at_top, at_work,
                                        out._size[3], device, _raw_stream(device)))
    if again:
        _written(out._parts())
    return out


class _Once(torch.autograd.Function):
    """A gradient made while a graph is recorded: there is no derivative of it, and taking one must not give zeros."""

    @staticmethod
    def forward(ctx, call, grad, *inputs):
        ctx.call = call
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, _g):
        raise _lib.QuiverError(f"the gradient of {ctx.call} cannot be differentiated again")


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
            grad = _Once.apply("log_probs", grad, logits, *(g for g in (g_target, g_entropy, g_lse, g_top) if g is not None))
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
    if result._size[0] != logits.shape[0]:
        raise ValueError("result was made for another number of rows")
    (_, at_entropy, _, at_ids, _, at_stats, _), device = result._now()
    return _gradient(logits, at_stats, at_entropy, at_ids, result._size[2], device, result.temperature, targets,
                     grad_target, grad_entropy, grad_logsumexp, grad_top, out)


def _param(name: str, p: torch.Tensor, dim: int, dtype: torch.dtype | None) -> int:
    """The address of a weight or bias, of ``dtype`` if that is known already."""
    if p.dtype not in _TYPES:
        raise ValueError(f"{name} has the type {p.dtype}; " + " or ".join(str(x) for x in _TYPES) + " is needed")
    return _vector(name, p, (dim,), p.dtype if dtype is None else dtype)


def _norm(x, weight, bias, eps, out):
    n, d, stride = _matrix("x", x, _TYPES)
    dtype = at_weight = at_bias = None
    if bias is not None:
        dtype, at_bias = bias.dtype, _param("bias", bias, d, None)
    if weight is not None:
        dtype, at_weight = weight.dtype if dtype is None else dtype, _param("weight", weight, d, dtype)
    again = out is not None
    if not again:
        out, out_stride = torch.empty((n, d), dtype=x.dtype, device=x.device), max(d, 1)
    else:
        rows, cols, out_stride = _matrix("out", out, (x.dtype,))
        if rows != n or cols != d:
            raise ValueError("out and x differ in shape")
    if weight is None:
        device = _device(x, out) if bias is None else _device(x, out, bias)
    else:
        device = _device(x, out, weight) if bias is None else _device(x, out, weight, bias)
    _lib.check(_lib.load().qv_layer_norm(x.data_ptr(), _TYPES[x.dtype], n, d, stride, at_weight, at_bias,
                                         _lib.QV_FLOAT if dtype is None else _TYPES[dtype], eps, out.data_ptr(), out_stride,
                                         device, _raw_stream(device)))
    if again:
        _written((out,))
    return out


@dataclass(frozen=True, eq=False)
class LayerNormGrad:
    """What ``layer_norm_grad`` gives; None for what was not wanted."""

    x: torch.Tensor | None       # [n, d] of x's type
    weight: torch.Tensor | None  # [d] of the weight's type
    bias: torch.Tensor | None    # [d] of the weight's type
    _workspace: torch.Tensor
    _made_for: tuple             # rows, columns, types of x and weight
    _at: tuple                   # addresses of the first three (and x's row stride), the workspace and its bytes
    _strides: tuple | None       # of x
    _device: int

    @staticmethod
    def empty(n: int, d: int, dtype: torch.dtype, param_dtype: torch.dtype, wanted: tuple, device) -> "LayerNormGrad":
        """Buffers for the gradients that are wanted, of n rows of d values."""
        def new(want, shape, type_):
            return torch.empty(shape, dtype=type_, device=device) if want else None

        return LayerNormGrad.of(new(wanted[0], (n, d), dtype), new(wanted[1], d, param_dtype), new(wanted[2], d, param_dtype),
                                LayerNormGrad.workspace(n, d, device), (n, d, dtype, param_dtype))

    @staticmethod
    def workspace(n: int, d: int, device) -> torch.Tensor:
        """What the gradients of n rows of d values need beside their buffers; several results may share one on a stream."""
        size = _lib.load().qv_layer_norm_grad_workspace(n, d)
        if size < 0:
            _lib.check(size)
        return torch.empty(size, dtype=torch.uint8, device=device)

    @staticmethod
    def of(x, weight, bias, workspace, made_for: tuple) -> "LayerNormGrad":
        """Given buffers (None: not wanted; a gradient's own or x's memory may be its ``x``), a workspace (None: a new one),
        and what they are ``made_for``: rows, columns, types of x and of the weight."""
        n, d, dtype, param_dtype = made_for
        if workspace is None:
            there = [t for t in (x, weight, bias) if t is not None]
            if not there:
                raise ValueError("buffers for none of the gradients are given")
            workspace = LayerNormGrad.workspace(n, d, there[0].device)
        at_x, stride = None, d
        if x is not None:
            rows, cols, stride = _matrix("out.x", x, (dtype,))
            if rows != n or cols != d:
                raise ValueError("out.x has another number of rows or columns")
            at_x = x.data_ptr()
        at_weight, at_bias = (None if p is None else _vector(name, p, (d,), param_dtype)
                              for name, p in (("out.weight", weight), ("out.bias", bias)))
        _bytes(workspace)
        device = workspace.get_device()
        if any(t is not None and t.get_device() != device for t in (x, weight, bias)):
            raise ValueError("tensors must be on one GPU")
        return LayerNormGrad(x, weight, bias, workspace, made_for,
                             (at_x, stride, at_weight, at_bias, workspace.data_ptr(), workspace.shape[0]),
                             None if x is None else x.stride(), device)

    def _now(self) -> tuple:
        """(addresses, device), taken again where a tensor is no longer what they were taken of: its memory can be
        another's after ``t.data = ...``, ``set_`` or ``resize_`` (as ``Module.to`` does to a parameter's gradient)."""
        x, weight, bias, (n, d, dtype, param_dtype) = self.x, self.weight, self.bias, self._made_for
        at_x, _, at_weight, at_bias, at_work, _ = self._at
        if ((at_x is None if x is None else x.data_ptr() == at_x and x.shape == (n, d) and x.stride() == self._strides
             and x.dtype is dtype)
                and (at_weight is None if weight is None else weight.data_ptr() == at_weight and weight.numel() == d
                     and weight.is_contiguous() and weight.dtype is param_dtype)
                and (at_bias is None if bias is None else bias.data_ptr() == at_bias and bias.numel() == d
                     and bias.is_contiguous() and bias.dtype is param_dtype)
                and self._workspace.data_ptr() == at_work):
            return self._at, self._device
        for t in (x, weight, bias, self._workspace):
            if t is not None:
                _whole(t)
        same = LayerNormGrad.of(x, weight, bias, self._workspace, self._made_for)
        return same._at, same._device


def _norm_grad(x, grad, weight, eps, dtype, wanted, out) -> LayerNormGrad:
    n, d, stride = _matrix("x", x, _TYPES)
    grad_rows, grad_cols, grad_stride = _matrix("grad", grad, (x.dtype,))
    if grad_rows != n or grad_cols != d:
        raise ValueError("grad and x differ in shape")
    if weight is None:
        at_weight = None
    elif weight.numel() == d and weight.dim() == 1 and weight.is_contiguous() and weight.dtype in _TYPES:
        at_weight = weight.data_ptr()
    else:
        at_weight = _param("weight", weight, d, None)
    again = out is not None
    if again and out._made_for != (n, d, x.dtype, dtype):
        raise ValueError("out was made for another number of rows or columns, or other types")
    device = _device(x, grad) if weight is None else _device(x, grad, weight)
    if not again:
        out = LayerNormGrad.empty(n, d, x.dtype, dtype, wanted, x.device)
        at = out._at
    else:
        at, made_on = out._now()
        if made_on != device:
            raise ValueError("tensors must be on one GPU")
    _lib.check(_lib.load().qv_layer_norm_grad(x.data_ptr(), _TYPES[x.dtype], n, d, stride, grad.data_ptr(), grad_stride,
                                              at_weight, _TYPES[dtype], eps, *at, device, _raw_stream(device)))
    if again:
        to = (out.x, out.weight, out.bias)
        if to[0] is None or to[1] is None or to[2] is None:
            to = [t for t in to if t is not None]
        _written(to)
    return out


class _LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y = _norm(x, weight, bias, eps, None)
        ctx.eps = eps
        ctx.dtype = torch.float32 if weight is None and bias is None else (bias if weight is None else weight).dtype
        ctx.save_for_backward(x, weight)
        return y

    @staticmethod
    def backward(ctx, g):
        x, weight = ctx.saved_tensors
        if _has_tangent(g):
            raise _lib.QuiverError("the gradient of layer_norm has no forward-mode derivative")
        r = _norm_grad(x, g.contiguous(), weight, ctx.eps, ctx.dtype, ctx.needs_input_grad[:3], None)
        grads = (r.x, r.weight, r.bias)
        if torch.is_grad_enabled():
            inputs = [t for t in (g, x, weight) if t is not None]
            grads = tuple(None if t is None else _Once.apply("layer_norm", t, *inputs) for t in grads)
        return (*grads, None)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *, eps: float = 1e-5,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over each row of ``x`` (float32, bfloat16 or float16 [n, d]).

    Mean and variance (over d) in fp32; the result has x's type, rounded once.
    ``weight`` and ``bias`` [d] are of one type, x's or another of the three.
    ``eps``: positive (a normal float).  ``out`` may be ``x``.  A row that holds an
    infinity or a NaN gives NaN.  With arguments that require a gradient the
    result takes part in autograd (``out`` is then refused), once: the gradient
    has none of its own, and there is no forward-mode derivative.
    """
    if (x.requires_grad or weight is not None and weight.requires_grad
            or bias is not None and bias.requires_grad) and torch.is_grad_enabled():
        if out is not None:
            raise ValueError("out= cannot be given for arguments that require a gradient")
        if _has_tangent(x, weight, bias):
            raise ValueError("layer_norm has no forward-mode derivative, and an argument has a tangent")
        return _LayerNormFunction.apply(x, weight, bias, float(eps))
    if out is not None and out.requires_grad or forward_ad._current_level >= 0:
        _no_derivative("layer_norm", x, weight, bias, out)
    return _norm(x, weight, bias, eps, out)


def layer_norm_grad(x: torch.Tensor, grad: torch.Tensor, weight: torch.Tensor | None = None, *, eps: float = 1e-5,
                    wanted: tuple[bool, bool, bool] | None = None, out: LayerNormGrad | None = None) -> LayerNormGrad:
    """The gradients of x, weight and bias from that of ``layer_norm``'s result.

    ``x``, ``weight`` and ``eps`` as they were for ``layer_norm``, ``grad`` of
    x's type.  The weight's and bias's come in the weight's type (float32
    without one).  ``wanted``: which of the three (all of them); ``out``: an
    earlier result, to be written again.  What autograd runs, for training loops
    without it (so arguments that require a gradient come detached, or under
    ``torch.no_grad()``).
    """
    again = out is not None
    to = (out.x, out.weight, out.bias) if again else (None, None, None)
    if (x.requires_grad or grad.requires_grad or weight is not None and weight.requires_grad
            or forward_ad._current_level >= 0 or to[0] is not None and to[0].requires_grad
            or to[1] is not None and to[1].requires_grad or to[2] is not None and to[2].requires_grad):
        _no_derivative("layer_norm_grad", x, grad, weight, *to)
    if wanted is None:
        wanted = (True, True, True)
    elif again:
        raise ValueError("wanted cannot be given beside out=, which has what is wanted")
    return _norm_grad(x, grad, weight, eps, torch.float32 if weight is None else weight.dtype, wanted, out)


class DenseCatalogue:
    """Embedding vectors kept in 8 bits, or in microscaled 4 bits, and scored exhaustively.

    ``DenseCatalogue(vectors)`` quantises the rows once, ``bits=4`` to half the
    bytes and 15 to 18 times the error of an inner product, as their queries.  ``log_probs(queries,
    targets, ...)`` gives each query's distribution over all of them, by inner
    products; the scores exist for one batch of queries at a time, about
    ``score_bytes`` of them.  Scores have no derivative (vectors, queries or a
    bias that require a gradient are refused).
    """

    bits = 8
    dim = None  # of the vectors: in 4 bits an odd one has as many bytes as the next

    def __init__(self, vectors: torch.Tensor, *, bias: torch.Tensor | None = None,
                 score_dtype: torch.dtype = torch.float32, score_bytes: int = 1 << 30, bits: int = 8) -> None:
        if bits not in (8, 4):
            raise ValueError("bits must be 8 or 4")
        if score_dtype not in _TYPES:
            raise ValueError("score_dtype must be float32, bfloat16 or float16")
        if score_bytes <= 0:
            raise ValueError("score_bytes must be positive")
        self.bits = bits
        self.codes, self.scales = self._quantize(vectors)
        self.dim = vectors.shape[1]
        if bias is not None:
            _vector("bias", bias, (vectors.shape[0],))
        self.bias, self.score_dtype, self.score_bytes = bias, score_dtype, int(score_bytes)

    def __len__(self) -> int:
        return self.codes.shape[0]

    def _quantize(self, rows: torch.Tensor):
        return quantize_rows(rows) if self.bits == 8 else quantize_rows_mx4(rows)

    def scores(self, queries: torch.Tensor, *, out: torch.Tensor | None = None) -> torch.Tensor:
        """Inner products of the queries, quantised row by row, with every vector: [n, len(self)], of ``out``'s type if given."""
        codes, scales = self._quantize(queries)
        if self.dim is not None and queries.shape[1] != self.dim:
            raise ValueError(f"queries have {queries.shape[1]} dimensions, the catalogue's vectors {self.dim}")
        product = int8_product if self.bits == 8 else mx4_product
        return product(codes, scales, self.codes, self.scales, bias=self.bias,
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
