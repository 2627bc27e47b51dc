"""Orthogonalised updates: the Newton-Schulz iteration on a batch of matrices and the optimiser
step around it.

``orthogonalize(x)`` replaces each matrix of a batch by an approximation of its polar factor
(all singular values moved towards 1), the direction of an orthogonalised-momentum optimiser:

    X = x / (||x||_F + eps);  per step  X <- a X + (b A + c A^2) X,  A = X X^T

``muon_update_`` is one whole step of that optimiser: momentum, direction, weights, in place.
It takes a batch, so the matrices of one shape (the projections of every layer, or the experts'
matrices whose gradient ``grouped.grouped_outer`` returns as one ``(experts, k, n)`` tensor, passed as
its ``.mT`` view) go through one call.

Both run the hand-written sm_100a products of ``libchol_b200.so`` (include/linalg_b200.h). CPU
tensors raise ``TypeError`` as in ``cholesky.custom_kernel``: there is no CPU path. The reference
project has no counterpart.
"""

from __future__ import annotations

import array
import functools
import math
from collections.abc import Sequence

import torch
from torch.autograd import forward_ad

from . import _lib

__all__ = ["orthogonalize", "muon_update_", "DEFAULT_COEFFICIENTS"]

#: Quintic with the steepest slope at zero that keeps every singular value near 1.
DEFAULT_COEFFICIENTS = (3.4445, -4.7750, 2.0315)

_TYPES = {torch.bfloat16: _lib.LINALG_BF16, torch.float16: _lib.LINALG_FP16,
          torch.float32: _lib.LINALG_FP32}
_PRECISIONS = {None: _lib.LINALG_PRECISION_AUTO, "half": _lib.LINALG_PRECISION_HALF,
               "full": _lib.LINALG_PRECISION_FULL}


def _check_tensor(t, name: str) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise TypeError(f"{name} must be on a CUDA device (this build has no CPU fallback)")
    if t.dtype not in _TYPES:
        raise TypeError(f"{name} must be bfloat16, float16 or float32, got {t.dtype}")
    if t.dim() < 2:
        raise ValueError(f"{name} must be (..., m, n), got shape {tuple(t.shape)}")


def _dual_level() -> bool:
    """Whether a forward_ad.dual_level is open (forward-mode derivatives ask for no requires_grad)."""
    return getattr(forward_ad, "_current_level", 0) >= 0


def _refuse_tangents(where: str, *tensors) -> None:
    """A result without the tangent that its inputs carry would read as a zero derivative."""
    if _dual_level() and torch._C._is_fwd_grad_enabled():
        for t in tensors:
            if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{where} has no forward-mode derivative: call it on a detached "
                                   "tensor")


def _batch_stride(t: torch.Tensor) -> int | None:
    """The distance of consecutive matrices, None when the leading dimensions have no single one."""
    step = None
    size = 1
    for d in range(t.dim() - 3, -1, -1):
        if t.shape[d] == 1:
            continue
        if step is None:
            step = t.stride(d)
        elif t.stride(d) != step * size:
            return None
        size *= t.shape[d]
    return 0 if step is None else step


def _is_rows(t: torch.Tensor, writable: bool) -> bool:
    """Whether the C ABI can address ``t``: contiguous rows, one row and one matrix stride."""
    if t.is_contiguous():
        return True
    m, n = t.shape[-2:]
    step = _batch_stride(t)
    if step is None or (n > 1 and t.stride(-1) != 1) or (m > 1 and t.stride(-2) < n):
        return False
    batch = t.numel() // (m * n) if m * n else 0
    if batch > 1 and not (writable is False and step == 0):
        return step >= (m - 1) * (t.stride(-2) if m > 1 else n) + n
    return True


def _is_transposed(t: torch.Tensor) -> bool:
    """Columns contiguous and rows not: the matrix is the transpose of a row-major one."""
    return t.shape[-1] > 1 and t.shape[-2] > 1 and t.stride(-1) != 1 and t.stride(-2) == 1


def _matrix(t: torch.Tensor) -> tuple[int, int, int, int]:
    m, n = t.shape[-2:]
    if t.is_contiguous():
        return t.data_ptr(), n, m * n, _TYPES[t.dtype]
    return t.data_ptr(), (t.stride(-2) if m > 1 else n), _batch_stride(t), _TYPES[t.dtype]


@functools.lru_cache(maxsize=64)
def _coefficients(coefficients: tuple, steps: int) -> array.array:
    rows = coefficients if isinstance(coefficients[0], tuple) else (coefficients,) * steps
    if len(rows) != steps or any(len(r) != 3 for r in rows):
        raise ValueError("coefficients must be (a, b, c), or one such triple for each step")
    flat = array.array("f", [float(c) for r in rows for c in r])
    if not all(math.isfinite(c) for c in flat):
        raise ValueError("coefficients must be finite")
    return flat


def _check_iteration(steps, coefficients, eps, precision):
    if not isinstance(steps, int) or not 1 <= steps <= _lib.LINALG_MAX_STEPS:
        raise ValueError(f"steps must be a whole number from 1 to {_lib.LINALG_MAX_STEPS}")
    if not 0 <= eps <= torch.finfo(torch.float32).max:
        raise ValueError("eps must be a 32-bit number and not negative")
    if precision not in _PRECISIONS:
        raise ValueError("precision must be None, 'half' or 'full'")
    if type(coefficients) is not tuple or any(type(c) is list for c in coefficients):
        if not isinstance(coefficients, Sequence) or not len(coefficients):
            raise ValueError("coefficients must be (a, b, c), or one such triple for each step")
        coefficients = tuple(tuple(c) if isinstance(c, Sequence) else c for c in coefficients)
    if not coefficients:
        raise ValueError("coefficients must be (a, b, c), or one such triple for each step")
    return _coefficients(coefficients, steps)


def _workspace(batch, m, n, precision, dtype, device):
    if precision is None:
        precision = "half" if dtype is torch.bfloat16 else "full"
    need = _workspace_bytes(batch, m, n, _PRECISIONS[precision])
    return (torch.empty(need, dtype=torch.uint8, device=device) if need else None), need


def _same_memory(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.data_ptr() == b.data_ptr() and a.stride() == b.stride() and a.dtype == b.dtype


def _ends(t: torch.Tensor) -> tuple[int, int]:
    if t.is_contiguous():
        start = t.data_ptr()
        return start, start + t.numel() * t.element_size()
    last = sum((s - 1) * st for s, st in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    (a0, a1), (b0, b1) = _ends(a), _ends(b)
    return a0 < b1 and b0 < a1


@functools.lru_cache(maxsize=256)
def _workspace_bytes(batch: int, m: int, n: int, precision: int) -> int:
    """A function of its arguments alone (no library option changes it)."""
    return int(_lib.load().linalg_orthogonalize_workspace(batch, m, n, precision))


_plain: dict = {}  # (steps, coefficients, eps, precision) of earlier calls -> checked arguments
_call = None       # the binding, once loaded


def _contiguous_call(x, steps, coefficients, eps, precision):
    """The common call (contiguous input, fresh output, one GPU) with arguments that an earlier call
    has checked: the host path paces calls of a few microseconds. None: not that case."""
    if type(x) is not torch.Tensor or not x.is_cuda or not x.is_contiguous() or \
            x.dim() not in (2, 3) or (x.requires_grad and torch.is_grad_enabled()) or \
            _dual_level() or x.is_neg():
        return None
    kind = _TYPES.get(x.dtype)
    try:  # (5.0 would find the plan of 5, and is refused)
        plan = _plain.get((steps, coefficients, eps, precision)) if type(steps) is int else None
    except TypeError:  # coefficients as lists
        return None
    if kind is None or plan is None or _call is None:
        return None
    shape = x.shape
    m, n = shape[-2], shape[-1]
    batch = shape[0] if len(shape) == 3 else 1
    size = m * n
    if not size or not batch:
        return None
    coef, code = plan
    out = torch.empty_like(x)
    need = _workspace_bytes(batch, m, n, code or (1 if kind == 0 else 2))
    ws = torch.empty(need, dtype=torch.uint8, device=x.device).data_ptr() if need else 0
    _lib.check(_call(x.data_ptr(), n, size, kind, out.data_ptr(), n, size, kind, batch, m, n, steps,
                     code, ws, need, _lib.current_queue(x.device.index), eps, coef),
               "linalg_orthogonalize")
    return out


def orthogonalize(x: torch.Tensor, steps: int = 5, *,
                  coefficients: Sequence = DEFAULT_COEFFICIENTS, eps: float = 1e-7,
                  precision: str | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Newton-Schulz approximation of the polar factor of each matrix of ``x``.

    x: ``(..., m, n)`` CUDA tensor, bfloat16, float16 or float32; any strides (a layout without
    contiguous rows or columns is copied first). coefficients: ``(a, b, c)``, or one triple for
    each of the ``steps``. The norm's squares are summed in 32 bits by eights and in 64 bits from there.
    precision: ``"half"`` works in fp16 with FP32 sums, an error of 0.5e-3 to 1.3e-3 of the result's
    norm on random matrices, below bfloat16's own rounding (1.7e-3); up to 2.6e-3 where one side is
    at most ~64 and the other above 4096. On matrices of low rank the roundings' noise is raised
    with the small singular values: 2.4e-2 at rank 64 of 1024, 7e-2 at rank 4, 0.15 at rank 1 (the
    first step on an expert's gradient from few rows, for example); ``"full"`` keeps those right.
    It works in split fp16, about as FP32 products would (1e-6 to 3.3e-6, 2e-4 at rank 1), at three
    times the products; so do matrices with a side above 2^18, whichever is given. None takes ``"half"`` for bfloat16 and ``"full"`` otherwise. out: written and
    returned instead of a new tensor; may be ``x`` itself.

    A matrix whose norm is well below eps gives a small result, ``norm / eps`` times the product of the
    steps' a, in fp16's smallest numbers: the error is then up to 1e-5 (``"full"``) of sqrt of the
    smaller side, what a matrix of full norm would have, and no longer of the result's norm (for
    1024 x 1024 at norm = eps / 1000, where the result's norm is 0.5: 1.4e-3 and 3e-4 of it).

    The iterates are fp16 numbers: coefficients with which some matrix could leave their range (singular
    values above ~8 in ``"half"``, ~4 in ``"full"``, where also ``|b s^2 + c s^4|`` stays below 32; a
    product of the steps' ``|a|`` below 1/4, ``a = 0`` among them) raise ``CholeskyError``;
    include/linalg_b200.h has the bounds.

    A zero matrix gives zeros (with eps > 0); a matrix with a NaN or an infinity gives NaN and leaves the
    others of the batch alone. It has no derivative, in either mode: call it under ``torch.no_grad()``
    or on a detached tensor (forward-mode tangents pass ``no_grad``; they raise).
    """
    if out is None and _one_device():
        out = _contiguous_call(x, steps, coefficients, eps, precision)
        if out is not None:
            return out
    _check_tensor(x, "x")
    coef = _check_iteration(steps, coefficients, eps, precision)
    _remember(steps, coefficients, eps, precision, coef)
    if torch.is_grad_enabled() and (x.requires_grad or (out is not None and out.requires_grad)):
        raise RuntimeError("orthogonalize has no derivative: call it under torch.no_grad()")
    _refuse_tangents("orthogonalize", x, out)
    given = out is not None
    if not given:
        out = (torch.empty_like(x.transpose(-2, -1), memory_format=torch.contiguous_format)
               .transpose(-2, -1) if _is_transposed(x)
               else torch.empty_like(x, memory_format=torch.contiguous_format))
    else:
        _check_tensor(out, "out")
        if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
            raise ValueError("out must have x's shape, type and device")
        if out.is_neg():
            raise ValueError("out must not be a lazy negation")
    if x.numel() == 0:
        return out
    source, target = x.resolve_neg(), out  # (a lazy negation's sign is not in memory yet)
    if _is_transposed(target):
        source, target = source.transpose(-2, -1), target.transpose(-2, -1)
    if not _is_rows(target, True):
        raise ValueError("out must have contiguous rows or columns and one stride between matrices")
    if not _same_memory(source, target) and _overlap(source, target):
        source = source.clone(memory_format=torch.contiguous_format)
    if not _is_rows(source, False):
        source = source.contiguous()
    m, n = source.shape[-2:]
    batch = source.numel() // (m * n)

    def call():
        ws, need = _workspace(batch, m, n, precision, x.dtype, x.device)
        return _lib.linalg().orthogonalize(
            *_matrix(source), *_matrix(target), batch, m, n, steps, _PRECISIONS[precision],
            ws.data_ptr() if need else 0, need, _lib.current_queue(x.device), eps, coef)

    _lib.check(_on_device(x, call), "linalg_orthogonalize")
    if given:
        _written(out)
    return out


def _written(*tensors: torch.Tensor) -> None:
    """Tells autograd that they were written in place (inference tensors keep no versions)."""
    tracked = [t for t in tensors if not t.is_inference()]
    if tracked:
        torch.autograd.graph.increment_version(tracked)


_single: bool | None = None


def _one_device() -> bool:
    """A single visible GPU: no call ever needs a device switch."""
    global _single
    if _single is None:
        _single = torch.cuda.device_count() == 1
    return _single


def _remember(steps, coefficients, eps, precision, coef) -> None:
    global _call
    _call = _lib.linalg().orthogonalize
    if isinstance(coefficients, tuple) and len(_plain) < 64:
        try:
            _plain[(steps, coefficients, eps, precision)] = coef, _PRECISIONS[precision]
        except TypeError:
            pass


def _on_device(t: torch.Tensor, call):
    if t.device.index == torch.cuda.current_device():
        return call()
    with torch.cuda.device(t.device):
        return call()


def muon_update_(param: torch.Tensor, grad: torch.Tensor, momentum: torch.Tensor, *, lr: float,
                 beta: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0,
                 steps: int = 5, coefficients: Sequence = DEFAULT_COEFFICIENTS,
                 eps: float = 1e-7, scale: float | None = None,
                 precision: str | None = None) -> torch.Tensor:
    """One optimiser step on a batch of weight matrices, in place; returns ``param``.

        momentum <- beta * momentum + (1 - beta) * grad
        u        =  beta * momentum + (1 - beta) * grad   if nesterov else   momentum
        param    <- (1 - lr * weight_decay) * param - lr * scale * orthogonalize(u)

    param, grad, momentum: ``(..., m, n)`` CUDA tensors of one shape, each bfloat16, float16 or
    float32, not overlapping. param and momentum need contiguous rows (or columns, both then)
    and one stride between matrices. scale: ``sqrt(max(1, m / n))`` when None, the usual
    ``sqrt(max(1, out / in))`` for weights of ``(out, in)``. Weights of ``(in, out)``, as
    ``grouped.grouped_matmul`` takes them, go in as views, ``w.mT`` with ``w.grad.mT`` and
    ``momentum.mT`` (worked on as they lie), or with their scale. precision: as in
    ``orthogonalize``, by param's type when None; a float32 param whose update may carry an error
    as ``orthogonalize`` gives for it takes ``"half"``, at a third of the work. u is taken from the momentum as
    stored. Call it under ``torch.no_grad()``.
    """
    for t, name in ((param, "param"), (grad, "grad"), (momentum, "momentum")):
        _check_tensor(t, name)
        if t.shape != param.shape or t.device != param.device:
            raise ValueError("param, grad and momentum must have one shape and device")
        if name != "grad" and t.is_neg():
            raise ValueError(f"{name} must not be a lazy negation")
        if name != "grad" and torch.is_grad_enabled() and t.requires_grad:
            raise RuntimeError(f"{name} requires grad: call muon_update_ under torch.no_grad()")
    _refuse_tangents("muon_update_", param, grad, momentum)
    coef = _check_iteration(steps, coefficients, eps, precision)
    for v, name in ((lr, "lr"), (beta, "beta"), (weight_decay, "weight_decay")):
        if not math.isfinite(v):
            raise ValueError(f"{name} must be finite")
    if param.numel() == 0:
        return param
    if scale is None:
        scale = math.sqrt(max(1.0, param.shape[-2] / param.shape[-1]))
    elif not math.isfinite(scale):
        raise ValueError("scale must be finite")
    p, g, mo = param, grad.resolve_neg(), momentum
    if _is_transposed(p):
        p, g, mo = p.transpose(-2, -1), g.transpose(-2, -1), mo.transpose(-2, -1)
    if not _is_rows(p, True) or not _is_rows(mo, True):
        raise ValueError("param and momentum must both have contiguous rows, or both contiguous "
                         "columns, and one stride between matrices")
    (p0, p1), (g0, g1), (m0, m1) = _ends(p), _ends(g), _ends(mo)
    if (p0 < m1 and m0 < p1) or (p0 < g1 and g0 < p1) or (m0 < g1 and g0 < m1):
        raise ValueError("param, grad and momentum must not overlap")
    if not _is_rows(g, False):
        g = g.contiguous()
    m, n = p.shape[-2:]
    batch = p.numel() // (m * n)

    def call():
        ws, need = _workspace(batch, m, n, precision, param.dtype, param.device)
        return _lib.linalg().muon_update(
            *_matrix(p), *_matrix(g), *_matrix(mo), batch, m, n, int(bool(nesterov)), steps,
            _PRECISIONS[precision], ws.data_ptr() if need else 0, need, _lib.current_queue(param.device), beta,
            1.0 - lr * weight_decay, lr * scale, eps, coef)

    _lib.check(_on_device(param, call), "linalg_muon_update")
    _written(param, momentum)
    return param
