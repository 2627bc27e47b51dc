"""GPU: sums so long that one tile takes more than the 2 s a wait may take otherwise. A 64-wide block of the
summed index takes ~356 ns where its loads' latency paces it, so 420 million terms take ~2.3 s.

All but a few terms are zeros, and what is left is exact: sums of a few small whole numbers.
"""

import ctypes

import pytest
import torch

from linalg_kernels_b200 import _lib
from linalg_kernels_b200.grouped import grouped_matmul, grouped_outer

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
LONG = 420_000_005  # ends inside a 16-wide slab


def _status():
    return _lib.load().chol_status_check(ctypes.c_void_p(_lib.current_queue(torch.device(DEV))))


def _small(*shape):
    g = torch.Generator(device=DEV).manual_seed(sum(shape))
    return torch.randint(-4, 5, shape, device=DEV, generator=g).bfloat16()


def test_outer_of_many_rows():
    a, b = (torch.zeros(LONG, 8, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    first, last = (_small(20, 8), _small(21, 8)), (_small(22, 8), _small(23, 8)[:22])
    for t, f, e in ((a, first[0], last[0]), (b, first[1][:20], last[1])):
        t[:20], t[-22:] = f, e
    dw = grouped_outer(a, b, torch.tensor([0, LONG], device=DEV))
    want = first[0].double().T @ first[1][:20].double() + last[0].double().T @ last[1].double()
    assert torch.equal(dw[0].double(), want.bfloat16().double())
    # with a group before it that takes no time
    dw = grouped_outer(a, b, torch.tensor([0, 16, LONG], device=DEV))
    assert torch.equal(dw[0].double(), (a[:16].double().T @ b[:16].double()).bfloat16().double())
    assert _status() == _lib.CHOL_OK


@pytest.mark.parametrize("rows", [1, 33])  # tiles of few rows, and of 256
def test_long_rows(rows):
    k = LONG + 3
    x = torch.zeros(rows, k, device=DEV, dtype=torch.bfloat16)
    w = torch.zeros(1, 8, k, device=DEV, dtype=torch.bfloat16)
    for t in (x, w[0]):
        t[:, :20], t[:, -22:] = _small(t.shape[0], 20), _small(t.shape[0], 22)
    y = grouped_matmul(x, w.mT, torch.tensor([0, rows], device=DEV))
    want = sum(x[:, i].double() @ w[0, :, i].double().T for i in (slice(0, 20), slice(k - 22, k)))
    assert torch.equal(y.double(), want.bfloat16().double())
    assert _status() == _lib.CHOL_OK
