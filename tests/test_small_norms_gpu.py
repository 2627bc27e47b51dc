"""GPU: the zero matrix gives zeros for every positive eps, those below FP32's smallest number among
them, and an eps that FP32 does not hold is refused."""

import pytest
import torch

from linalg_kernels_b200.orthogonal import muon_update_, orthogonalize

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("shape", [(2, 64, 64), (1, 100, 1500), (2, 200, 250), (2, 300, 260)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("eps", [1e-7, 1e-44, 1e-46, 1e-300])
def test_zero_matrix(shape, dtype, eps):
    zero = torch.zeros(shape, device=DEV, dtype=dtype)
    for _ in range(2):  # (the second call takes the short host path)
        assert orthogonalize(zero, eps=eps).eq(0).all()
    param = torch.ones_like(zero)
    muon_update_(param, zero, zero.clone(), lr=0.5, eps=eps)
    assert (param == 1).all()


def test_eps_out_of_range():
    x = torch.ones(3, 8, 8, device=DEV)
    for eps in (1e39, float("inf"), float("nan"), -1e-300):
        with pytest.raises(ValueError):
            orthogonalize(x, eps=eps)
