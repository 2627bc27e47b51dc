"""GPU: the operators in a row, as a routed layer's training step uses them: the expert products of a
two-layer block, their gradients, and the orthogonalised update of all experts' matrices in one
call each, against the same step in 64 bits.

Tolerance. Every bf16 tensor of the step (hidden rows, result, gradients) is a rounding of at most
2^-8 of each value; a tensor computed from rounded ones carries their errors on, so a relative
2-norm error of at most (number of roundings on its longest path) * 2^-8 plus FP32 sums
((K / 16) 2^-23 each) is allowed. The weights then move by lr * scale * direction: the direction
of a perturbed gradient is compared through the weights with the direction's own sensitivity left
out, so the update is checked from the step's own gradients (as the optimiser receives them), with
the tolerance of the optimiser's tests: the fp16 iteration's error twice, and half a bf16 step.
"""

import pytest
import torch

from linalg_kernels_b200.grouped import grouped_matmul
from linalg_kernels_b200.orthogonal import muon_update_
from tests.test_orthogonal_gpu import _tolerance

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _rel(a, b):
    return ((a.double() - b).norm() / b.norm()).item()


@pytest.mark.parametrize("rows,experts,d,h,transposed", [(700, 5, 256, 384, False),
                                                         (96, 8, 160, 264, True)])
def test_expert_training_step(rows, experts, d, h, transposed):
    g = torch.Generator(device=DEV).manual_seed(rows)

    def randn(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    share = torch.rand(experts, generator=torch.Generator().manual_seed(1))
    share[1] = 0  # an expert without rows
    ends = (share.cumsum(0) / share.sum() * rows).round().int()
    offsets = torch.cat([torch.zeros(1, dtype=torch.int32), ends]).to(DEV)
    off = offsets.tolist()
    x = randn(rows, d).bfloat16()

    def weights(k, n):
        w = (randn(experts, n, k) if transposed else randn(experts, k, n)) / k ** 0.5
        w = w.bfloat16().requires_grad_()
        return w, (w.transpose(1, 2) if transposed else w)

    (w1, w1_view), (w2, w2_view) = weights(d, h), weights(h, d)
    x = x.requires_grad_()
    hidden = grouped_matmul(x, w1_view, offsets)
    act = torch.nn.functional.silu(hidden)
    y = grouped_matmul(act, w2_view, offsets)
    target = randn(rows, d).bfloat16()
    ((y.float() - target.float()).square().sum() / rows).backward()

    # the same in 64 bits
    x64 = x.detach().double().requires_grad_()
    v1, v2 = (w.detach().double().requires_grad_() for w in (w1, w2))
    parts = []
    for e in range(experts):
        a = v1[e].T if transposed else v1[e]
        b = v2[e].T if transposed else v2[e]
        parts.append(torch.nn.functional.silu(x64[off[e]:off[e + 1]] @ a) @ b)
    y64 = torch.cat(parts)
    ((y64 - target.double()).square().sum() / rows).backward()
    sums = (max(d, h, rows) / 16 + 2) * 2.0 ** -22
    assert _rel(y, y64.detach()) <= 4 * 2.0 ** -8 + 2 * sums       # hidden, silu, y
    assert _rel(w2.grad, v2.grad) <= 6 * 2.0 ** -8 + 3 * sums      # + dy, dw
    assert _rel(w1.grad, v1.grad) <= 9 * 2.0 ** -8 + 4 * sums      # + dact, silu's, dhidden, dw
    assert _rel(x.grad, x64.grad) <= 9 * 2.0 ** -8 + 4 * sums
    for w in (w1, w2):
        assert not w.grad[1].any()  # no rows, no gradient

    for w in (w1, w2):
        momentum = torch.zeros(w.shape, device=DEV)
        before, grad = w.detach().double(), w.grad.clone()
        with torch.no_grad():
            muon_update_(w, grad, momentum, lr=0.02, weight_decay=0.1)
        m64 = 0.05 * grad.double()
        assert ((momentum.double() - m64).abs() <= m64.abs() * 2.0 ** -22).all()
        u = 0.95 * momentum.double() + 0.05 * grad.double()
        scale = max(1.0, w.shape[-2] / w.shape[-1]) ** 0.5
        live = [e for e in range(experts) if off[e + 1] > off[e]]
        o, tol = _tolerance(u[live], torch.float32, True)
        want = (1 - 0.002) * before[live] - 0.02 * scale * o
        off_by = (w.detach()[live].double() - want).square().sum((-2, -1)).sqrt()
        allowed = (2.0 ** -8 + 3 * 2.0 ** -24) * want.square().sum((-2, -1)).sqrt() + \
            0.02 * scale * tol * o.square().sum((-2, -1)).sqrt()
        assert (off_by <= allowed).all()
        # the expert without rows: momentum and direction are zero, only the decay acts
        decayed = (1 - 0.002) * before[1]
        assert ((w.detach()[1].double() - decayed).abs() <= decayed.abs() * 2.0 ** -8 + 1e-30).all()
