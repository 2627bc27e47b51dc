"""GPU: half precision on matrices so long that the tensor core's sums, rounded towards zero every 16
terms, would fall short. Tolerances: test_orthogonal_gpu.py's for half precision, which know of no
such loss."""

import pytest
import torch

from linalg_kernels_b200 import _lib
from linalg_kernels_b200.orthogonal import muon_update_, orthogonalize
from tests.test_orthogonal_gpu import _far, _input, _tolerance

pytestmark = pytest.mark.gpu
LONG = 1 << 20


@pytest.mark.parametrize("shape", [(1, 16, LONG), (1, LONG, 16), (2, 1, LONG + 5), (1, 4, LONG * 4),
                                   (1, 16, (1 << 18) + 8), (1, 256, (1 << 18) + 8)])
def test_long(shape):
    x = _input(sum(shape), shape, torch.bfloat16)
    exact, tol = _tolerance(x, x.dtype, True)
    assert _far(orthogonalize(x), exact) <= tol
    exact, tol = _tolerance(x, torch.float32, True)
    assert _far(orthogonalize(x.float(), precision="half"), exact) <= tol
    param, momentum = torch.zeros_like(x), torch.zeros_like(x)
    muon_update_(param, x, momentum, lr=1.0, beta=0.0, nesterov=False, scale=1.0)
    assert torch.equal(param, -orthogonalize(x))


def test_workspace_of_long_matrices():
    f = _lib.load().linalg_orthogonalize_workspace
    half, full = _lib.LINALG_PRECISION_HALF, _lib.LINALG_PRECISION_FULL
    for m, n in ((16, 1 << 18), (1 << 18, 16)):
        assert f(1, m, n, half) < f(1, m, n, full)
        assert f(1, m + (m > n), n + (m < n), half) == f(1, m + (m > n), n + (m < n), full)
