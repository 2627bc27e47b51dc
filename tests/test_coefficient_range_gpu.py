"""GPU: results at the edge of the range that the coefficients may use.

A matrix with a single entry 1 takes the largest singular value there is, in one entry of X, G and B.
The numbers below are fp16 numbers at every step (61504 = 1922 * 32, 64992 = 2031 * 32, 64512 =
2016 * 32, 15376 = 1922 * 8, 31.03125 = 1986 / 64, and 7.75, 3.875 times a power of two), and the
sums have one term, so the results are exact.
"""

import pytest
import torch

from linalg_kernels_b200 import _lib
from linalg_kernels_b200.orthogonal import muon_update_, orthogonalize

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

# on chip (one CTA, a cluster, a CTA pair in half precision), by products
SHAPES = [(3, 64, 64), (2, 40, 30), (1, 100, 1500), (1, 700, 100), (2, 200, 250), (1, 300, 260),
          (2, 129, 700)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("precision,coefs,want", [
    # s = 7.75, G = 60.0625 * 1024; then B = 1 + 60.0625 / 2
    ("half", ((7.75, 0.0, 0.0), (1.0, 0.5, 0.0)), 7.75 * 31.03125),
    ("half", ((64992.0, 0.0, 0.0),), 64992.0),
    # s = 3.875, G = 15.015625 * 4096; then b G = 7.5078125, times 2048
    ("full", ((3.875, 0.0, 0.0), (1.0, 0.5, 0.0)), 3.875 * 8.5078125),
    ("full", ((1.0, 31.5, 0.0),), 32.5)])
def test_largest_values(shape, precision, coefs, want):
    x = torch.zeros(shape, device=DEV)
    x[:, 3, 5] = 1.0
    got = orthogonalize(x, len(coefs), coefficients=coefs, eps=0.0, precision=precision)
    assert torch.equal(got, x * want)
    param, momentum = torch.zeros_like(x), torch.zeros_like(x)
    muon_update_(param, x, momentum, lr=1.0, beta=0.0, nesterov=False, scale=1.0, steps=len(coefs),
                 coefficients=coefs, eps=0.0, precision=precision)
    assert torch.equal(param, x * -want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_beyond_is_refused(dtype):
    x = torch.zeros(2, 64, 64, device=DEV, dtype=dtype)
    coefs = ((9.0, 0.0, 0.0), (1.0, 0.5, 0.0))
    momentum = torch.ones_like(x)
    for _ in range(2):
        with pytest.raises(_lib.CholeskyError):
            orthogonalize(x, 2, coefficients=coefs)
        with pytest.raises(_lib.CholeskyError):
            muon_update_(x, torch.ones_like(x), momentum, lr=0.1, steps=2, coefficients=coefs)
    assert not x.any() and (momentum == 1).all()


def test_shrinking_is_refused():
    x = torch.ones(1, 100, 1500, device=DEV, dtype=torch.bfloat16)
    with pytest.raises(_lib.CholeskyError):
        orthogonalize(x, 2, coefficients=(0.0, 2.0, -1.0))
    for t in (x, x[:, :, :90], torch.ones(2, 260, 300, device=DEV)):
        assert not orthogonalize(t, 2, coefficients=(0.0, 0.0, 0.0)).any()
