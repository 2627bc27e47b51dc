"""GPU: coefficients with zeros among them, as the cubic iteration X <- 1.5 X - 0.5 X X^T X has.

Tolerances: test_orthogonal_gpu.py's.
"""

import pytest
import torch

from linalg_kernels_b200.orthogonal import muon_update_, orthogonalize
from tests.test_orthogonal_gpu import _far, _input, _tolerance

pytestmark = pytest.mark.gpu

# on chip (one CTA, a cluster, a CTA pair in half precision), by products in both orders
SHAPES = [(3, 64, 64), (2, 100, 30), (1, 100, 1500), (2, 200, 250), (1, 300, 260), (1, 260, 300),
          (2, 129, 700), (3, 700, 140)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("coefs", [(1.5, -0.5, 0.0), (1.875, 0.0, -0.875), (2.0, 0.0, 0.0)])
def test_zero_coefficients(shape, dtype, coefs):
    x = _input(sum(shape), shape, dtype)
    steps = 5 if coefs[0] == 1.5 else 2
    exact, tol = _tolerance(x, dtype, dtype is torch.bfloat16, steps=steps, coefs=coefs)
    got = orthogonalize(x, steps, coefficients=coefs)
    assert _far(got, exact) <= tol
    if dtype is torch.float32:
        momentum, param = torch.zeros_like(x), torch.zeros_like(x)
        muon_update_(param, x, momentum, lr=1.0, beta=0.0, nesterov=False, scale=1.0, steps=steps,
                     coefficients=coefs)
        assert torch.equal(param, -got)
