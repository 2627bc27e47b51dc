"""Products of rows grouped by an index, each group with its own matrix: the expert products of
a routed layer, with their gradients.

    y[r]  = x[r] @ w[e]                       for offsets[e] <= r < offsets[e + 1]
    dx[r] = dy[r] @ w[e]^T
    dw[e] = sum of outer(x[r], dy[r]) over the group

``grouped_matmul`` is differentiable in x and w; ``grouped_outer`` is its weight gradient alone.
The offsets stay on the device: no call waits for the GPU, and calls can be captured into a CUDA
graph whose replays see other group sizes. The kernels are the tensor-core products of
``libchol_b200.so`` (include/linalg_b200.h); CPU tensors raise ``TypeError``, as everywhere in
this package. The reference project has no counterpart.
"""

from __future__ import annotations

import torch

from . import _lib
from .orthogonal import _refuse_tangents, _written

__all__ = ["grouped_matmul", "grouped_outer"]

_TYPES = {torch.bfloat16: _lib.LINALG_BF16, torch.float16: _lib.LINALG_FP16}


def _check(t, name: str, dim: int, like: torch.Tensor | None = None) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise TypeError(f"{name} must be on a CUDA device (this build has no CPU fallback)")
    if t.dtype not in _TYPES:
        raise TypeError(f"{name} must be bfloat16 or float16, got {t.dtype}")
    if t.dim() != dim:
        raise ValueError(f"{name} must have {dim} dimensions, got shape {tuple(t.shape)}")
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        raise ValueError(f"{name} must have the other operand's type and device")


def _check_offsets(offsets, like: torch.Tensor, groups: int | None = None) -> int:
    if not isinstance(offsets, torch.Tensor) or offsets.dtype not in (torch.int32, torch.int64):
        raise TypeError("offsets must be an int32 or int64 tensor")
    if offsets.device != like.device:
        raise ValueError("offsets must be on the operands' device")
    if offsets.dim() != 1 or offsets.numel() < 1 or not offsets.is_contiguous():
        raise ValueError("offsets must be contiguous, (groups + 1,)")
    n = offsets.numel() - 1
    if groups is not None and n != groups:
        raise ValueError(f"offsets must have {groups + 1} entries, one more than w has matrices")
    if n > _lib.LINALG_MAX_GROUPS:
        raise ValueError(f"at most {_lib.LINALG_MAX_GROUPS} groups, got {n}")
    return n


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """``t`` with contiguous rows that start on 16-byte boundaries (as the bulk copies need), a
    copy with padded rows where it has not."""
    if t.is_neg():  # a lazy negation (imag of a conjugate): the sign is not in memory yet
        t = t.resolve_neg()
    shape, stride = t.shape, t.stride()
    rows, cols, ld = shape[-2], shape[-1], stride[-2]
    if stride[-1] == 1 and not ld & 7 and ld >= cols and not t.data_ptr() & 15 and (
            len(shape) < 3 or (not stride[0] & 7 and stride[0] >= cols + (rows - 1) * ld)):
        return t
    padded = t.new_empty(*shape[:-1], (cols + 7) // 8 * 8)[..., :cols]
    return padded.copy_(t.detach())


def _aligned_weights(w: torch.Tensor) -> torch.Tensor:
    """The same for (groups, k, n) weights, in the order in which they lie in memory."""
    if _stored_transposed(w):
        lies = w.transpose(1, 2)
        rows = _aligned(lies)
        return w if rows is lies else rows.transpose(1, 2)
    return _aligned(w)


def _stored_transposed(w: torch.Tensor) -> bool:
    return w.stride(1) == 1 and w.stride(2) != 1


_call = None  # the binding's (grouped_matmul, grouped_outer), once loaded


def _binding():
    global _call
    if _call is None:
        lib = _lib.linalg()
        _call = lib.grouped_matmul, lib.grouped_outer
    return _call


def _matmul(x, w, offsets, out=None):
    """x and w aligned (_aligned, _aligned_weights); on x's device."""
    rows, k = x.shape
    groups, _, n = w.shape
    fill = out is None
    if fill:
        out = x.new_empty(rows, n)
    if rows == 0 or n == 0:
        return out
    if k == 0 or groups == 0:
        if groups and not fill:
            raise ValueError("out needs k > 0")
        return out.zero_() if fill else out
    transposed = _stored_transposed(w)
    stride = w.stride()
    kind = _TYPES[x.dtype]
    status = (_call or _binding())[0](
        x.data_ptr(), x.stride(0), 0, kind, w.data_ptr(), stride[2 if transposed else 1], stride[0],
        kind, out.data_ptr(), out.stride(0), 0, kind, not transposed, offsets.data_ptr(),
        offsets.dtype is torch.int64, groups, rows, k, n, fill, _lib.current_queue(x.device.index))
    if status:
        _lib.check(status, "linalg_grouped_matmul")
    return out


def _outer(a, b, offsets, groups, out=None):
    """a and b aligned; on a's device."""
    rows, k = a.shape
    n = b.shape[1]
    if out is None:
        out = a.new_empty(groups, k, n)
    if out.numel() == 0:
        return out
    if rows == 0:
        return out.zero_()
    kind = _TYPES[a.dtype]
    status = (_call or _binding())[1](
        a.data_ptr(), a.stride(0), 0, kind, b.data_ptr(), b.stride(0), 0, kind, out.data_ptr(),
        out.stride(1), out.stride(0), kind, offsets.data_ptr(), offsets.dtype is torch.int64, groups,
        rows, k, n, _lib.current_queue(a.device.index))
    if status:
        _lib.check(status, "linalg_grouped_outer")
    return out


_single: bool | None = None


def _on_device(t: torch.Tensor, call):
    """Runs ``call`` with t's device current."""
    global _single
    if _single is None:
        _single = torch.cuda.device_count() == 1
    if _single or t.device.index == torch.cuda.current_device():
        return call()
    with torch.cuda.device(t.device):
        return call()


class _GroupedMatmul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, offsets, aligned):
        # the aligned operands serve the backward pass too: a copy is made once
        ax, aw, ctx.links = aligned
        ctx.save_for_backward(ax, aw, offsets)
        return _matmul(ax, aw, offsets)

    @staticmethod
    def backward(ctx, dy):  # (autograd has made the device current)
        _refuse_tangents("grouped_matmul's backward pass", dy)
        x, w, offsets = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dw = None
        with torch.no_grad():
            rows = _aligned(dy)
            if need[0]:
                dx = _matmul(rows, w.transpose(1, 2), offsets)
            if need[1]:
                if _stored_transposed(w):  # stored (groups, n, k): so is its gradient
                    dw = _outer(rows, x, offsets, w.shape[0]).transpose(1, 2)
                else:
                    dw = _outer(x, rows, offsets, w.shape[0])
        if torch.is_grad_enabled():  # create_graph: dx hangs on w and dy, dw on x and dy
            if dx is not None:
                dx = _Once.apply(dx, dy, _origin(ctx, 1, w))
            if dw is not None:
                dw = _Once.apply(dw, dy, _origin(ctx, 0, x))
        return dx, dw, None, None


class _Once(torch.autograd.Function):
    """A gradient and what it hangs on. It has no derivative: asking for one raises, where a detached
    tensor would read as a constant. (torch's once_differentiable marks gradients only where dy
    requires grad, and hangs them on nothing.)"""

    @staticmethod
    def forward(ctx, t, *on):
        return t.view_as(t)

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError("grouped_matmul has no second derivative")


def _differentiable(x, w, offsets):
    ax, aw = _aligned(x), _aligned_weights(w)
    return _GroupedMatmul.apply(x, w, offsets, (ax, aw, (_link(x, ax), _link(w, aw))))


def _link(t: torch.Tensor, aligned: torch.Tensor) -> torch.Tensor | None:
    """An empty tensor with t's place in the graph, where the backward pass keeps a copy of t instead."""
    return t[:0].clone() if aligned is not t and t.grad_fn is not None else None


def _origin(ctx, i: int, saved: torch.Tensor):
    """A tensor with operand i's place in the graph, None for one that requires no grad."""
    node = ctx.next_functions[i][0]
    if node is None or saved.requires_grad:
        return saved if node is not None else None
    leaf = getattr(node, "variable", None)
    return leaf if leaf is not None else ctx.links[i]


def _check_out(out, shape, like, name, others):
    _check(out, name, len(shape), like)
    if out.is_neg():
        raise ValueError(f"{name} must not be a lazy negation")
    if tuple(out.shape) != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(out.shape)}")
    if out.numel() == 0:
        return
    rows, cols = shape[-2:]
    ld = out.stride(-2)
    if out.stride(-1) != 1 or ld < cols or (
            len(shape) == 3 and out.stride(0) < (rows - 1) * ld + cols):
        raise ValueError(f"{name} must have contiguous, separate rows")
    if torch.is_grad_enabled() and (out.requires_grad or any(o.requires_grad for o in others)):
        raise RuntimeError(f"{name}= is not differentiable: call it under torch.no_grad()")

    def ends(t):
        last = sum((s - 1) * st for s, st in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()

    o0, o1 = ends(out)
    for t in others:
        if t.numel():
            t0, t1 = ends(t)
            if o0 < t1 and t0 < o1:
                raise ValueError(f"{name} must not overlap the operands")


def grouped_matmul(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, *,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """``y[r] = x[r] @ w[e]`` for the rows ``offsets[e] <= r < offsets[e + 1]`` of each group.

    x: ``(rows, k)``, w: ``(groups, k, n)``, bfloat16 or float16 CUDA tensors of one type; sums in
    FP32, rounded once (the tensor core rounds its sums towards zero every 16 terms: at most
    ``(terms / 16 + 2) * 2**-22`` of the sum of the terms' magnitudes, ~1e-3 for 2^16 terms of one
    sign). w may be the transposed view of ``(groups, n, k)`` weights, read as it lies. Rows that do
    not start on 16-byte boundaries (k or n not a multiple of 8) and other layouts are copied first.
    offsets: ``(groups + 1,)`` int32 or int64 on the device, non-decreasing within ``[0, rows]``
    (values that are not are clamped: no row outside x is touched); groups may be empty. Rows of no
    group (padding in front of offsets[0] or behind offsets[-1]) are zero in the result; with
    ``out`` given they stay as they were. At most 1024 groups. ``out`` needs k > 0 and contiguous
    rows, at any distance; nothing between them is written.

    Differentiable in x and w (without ``out``): the gradient of a group without rows, and of rows
    of no group, is zero; dy's rows of no group are not read. Forward-mode tangents and second
    derivatives raise. Runs on the current queue of x's device.
    """
    _check(x, "x", 2)
    _check(w, "w", 3, x)
    if w.shape[1] != x.shape[1]:
        raise ValueError(f"w must be (groups, {x.shape[1]}, n), got {tuple(w.shape)}")
    _check_offsets(offsets, x, w.shape[0])
    _refuse_tangents("grouped_matmul", x, w, out)
    if out is not None:
        _check_out(out, (x.shape[0], w.shape[2]), x, "out", (x, w))
        _on_device(x, lambda: _matmul(_aligned(x), _aligned_weights(w), offsets, out))
        _written(out)
        return out
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad):
        return _on_device(x, lambda: _differentiable(x, w, offsets))
    return _on_device(x, lambda: _matmul(_aligned(x), _aligned_weights(w), offsets))


def grouped_outer(a: torch.Tensor, b: torch.Tensor, offsets: torch.Tensor, *,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """``dw[e] = a[i:j].T @ b[i:j]`` with ``i, j = offsets[e], offsets[e + 1]``: the weight gradient
    of ``grouped_matmul``, ``(groups, k, n)`` for a ``(rows, k)`` and b ``(rows, n)``.

    Types, layouts and offsets as in ``grouped_matmul``. A group without rows gives zeros. Rows
    of no group are never read into a result, whatever they hold. Not differentiable.
    """
    _check(a, "a", 2)
    _check(b, "b", 2, a)
    if a.shape[0] != b.shape[0]:
        raise ValueError(f"a and b must have the same rows, got {a.shape[0]} and {b.shape[0]}")
    groups = _check_offsets(offsets, a)
    if torch.is_grad_enabled() and (a.requires_grad or b.requires_grad):
        raise RuntimeError("grouped_outer has no derivative: call it under torch.no_grad()")
    _refuse_tangents("grouped_outer", a, b, out)
    if out is not None:
        _check_out(out, (groups, a.shape[1], b.shape[1]), a, "out", (a, b))
    result = _on_device(a, lambda: _outer(_aligned(a), _aligned(b), offsets, groups, out))
    if out is not None:
        _written(out)
    return result
