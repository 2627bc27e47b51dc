"""GPU: grouped_matmul's gradients have no derivative, and say so whichever operand requires grad."""

import pytest
import torch

from linalg_kernels_b200.grouped import grouped_matmul

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _problem(k, n, transposed):
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(6, k, device=DEV, generator=g).bfloat16()
    w = torch.randn(2, *((n, k) if transposed else (k, n)), device=DEV, generator=g).bfloat16()
    dy = torch.randn(6, n, device=DEV, generator=g).bfloat16()
    return x, w, dy, torch.tensor([0, 2, 6], device=DEV)


# aligned operands are kept as they are for the backward pass, others as padded copies
@pytest.mark.parametrize("k,n", [(8, 16), (9, 13)])
@pytest.mark.parametrize("transposed", [False, True])
def test_second_derivatives_raise(k, n, transposed):
    x, w, dy, offsets = _problem(k, n, transposed)

    def grads(gx, gw, gdy):
        xx, ww, dd = x.clone().requires_grad_(gx), w.clone().requires_grad_(gw), dy.clone().requires_grad_(gdy)
        y = grouped_matmul(xx, ww.mT if transposed else ww, offsets)
        leaves = [t for t, r in ((xx, gx), (ww, gw)) if r]
        first = torch.autograd.grad(y, leaves, dd, create_graph=True)
        y = grouped_matmul(xx, ww.mT if transposed else ww, offsets)
        plain = torch.autograd.grad(y, leaves, dd)
        for a, b in zip(first, plain):
            assert torch.equal(a, b) and not b.requires_grad
        return first, (xx, ww, dd)

    (dx, dw), (xx, ww, dd) = grads(True, True, False)
    for g, leaf in ((dx, ww), (dw, xx)):
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(g.sum(), leaf, retain_graph=True)
    # a penalty on the gradient beside another term
    loss = ww.square().sum() + dx.square().sum()
    for call in (lambda: torch.autograd.grad(loss, ww, retain_graph=True),
                 lambda: torch.autograd.grad(loss, ww, retain_graph=True, allow_unused=True),
                 loss.backward):
        with pytest.raises(RuntimeError, match="second derivative"):
            call()
    for gx, gw in ((True, False), (False, True)):
        (g,), _ = grads(gx, gw, False)
        assert not g.requires_grad  # linear in the one that requires grad: a constant
        (g,), (xx, ww, dd) = grads(gx, gw, True)
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(g.sum(), dd)


@pytest.mark.parametrize("k,n", [(8, 16), (9, 13)])
@pytest.mark.parametrize("transposed", [False, True])
def test_operands_inside_a_graph(k, n, transposed):
    """Neither operand a leaf; the gradients hang on what the operands were made of."""
    x, w, dy, offsets = _problem(k, n, transposed)
    x.requires_grad_(), w.requires_grad_()

    def first(create_graph):
        xx, ww = x * 2, w * 0.5
        y = grouped_matmul(xx, ww.mT if transposed else ww, offsets)
        return torch.autograd.grad(y, (xx, ww), dy, create_graph=create_graph)

    dx, dw = first(True)
    for a, b in zip((dx, dw), first(False)):
        assert torch.equal(a, b)
    for g, leaf in ((dx, w), (dw, x)):
        for unused in (False, True):
            with pytest.raises(RuntimeError, match="second derivative"):
                torch.autograd.grad(g.sum(), leaf, retain_graph=True, allow_unused=unused)


def test_gradients_accumulate_with_create_graph():
    x, w, dy, offsets = _problem(8, 16, False)
    x.requires_grad_(), w.requires_grad_()
    grouped_matmul(x, w, offsets).backward(dy, create_graph=True)
    first = x.grad.detach().clone(), w.grad.detach().clone()
    x.grad = w.grad = None
    grouped_matmul(x, w, offsets).backward(dy)
    assert torch.equal(x.grad, first[0]) and torch.equal(w.grad, first[1])
    assert not x.grad.requires_grad


def test_forward_over_reverse():
    from torch.autograd import forward_ad

    x, w, dy, offsets = _problem(8, 16, False)
    x.requires_grad_()
    with forward_ad.dual_level():
        y = grouped_matmul(x, w, offsets)
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(y, x, forward_ad.make_dual(dy, torch.ones_like(dy)))
