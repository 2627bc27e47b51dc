"""GPU: the training step of the integration notes, run as it stands there: a layer whose weights are stored
(groups, in, out) gets the update of the same layer stored (groups, out, in).

Tolerance: test_expert_step_gpu.py's, from each side's own gradient.
"""

from pathlib import Path

import pytest
import torch

from linalg_kernels_b200.grouped import grouped_matmul
from linalg_kernels_b200.orthogonal import muon_update_
from tests.test_orthogonal_gpu import _tolerance

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _example():
    text = (Path(__file__).resolve().parents[1] / "INTEGRATION.md").read_text()
    text = text[text.index("## Orthogonalised updates and grouped products"):]
    return text.split("```python\n")[1].split("```")[0]


@pytest.mark.parametrize("k,n", [(64, 256), (256, 64), (200, 336), (136, 136)])
def test_both_storage_orders_get_one_update(k, n):
    g = torch.Generator(device=DEV).manual_seed(k)

    def randn(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    start = (randn(3, k, n) / k ** 0.5).bfloat16()
    x, dy = randn(500, k).bfloat16(), randn(500, n).bfloat16()
    offsets = torch.tensor([0, 100, 350, 500], device=DEV)
    w = start.clone().requires_grad_()
    momentum = torch.zeros(3, k, n, device=DEV)
    exec(_example(), dict(torch=torch, x=x, w=w, offsets=offsets, dy=dy, momentum=momentum, g=start))
    v = start.mT.contiguous().requires_grad_()  # (groups, out, in)
    other = torch.zeros(3, n, k, device=DEV)
    grouped_matmul(x, v.mT, offsets).backward(dy)
    with torch.no_grad():
        muon_update_(v, v.grad, other, lr=0.02, weight_decay=0.1)
    rate = 0.02 * max(1.0, n / k) ** 0.5
    for weights, grad, mom in ((w, w.grad, momentum), (v.mT, v.grad.mT, other.mT)):
        u = 0.95 * mom.double() + 0.05 * grad.double()
        o, tol = _tolerance(u, torch.float32, True)
        want = (1 - 0.002) * start.double() - rate * o
        off = (weights.detach().double() - want).square().sum((-2, -1)).sqrt()
        allowed = (2.0 ** -8 + 3 * 2.0 ** -24) * want.square().sum((-2, -1)).sqrt() + \
            rate * tol * o.square().sum((-2, -1)).sqrt()
        assert (off <= allowed).all(), (off, allowed)
