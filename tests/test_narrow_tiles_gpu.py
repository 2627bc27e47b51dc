"""GPU: products on 128-wide tiles, many of them per CTA pair and with a short summed index, so that
a tile's results are stored while the next one's are being rounded into the same staging buffer.
Compared over the whole result, several times over.

Tolerance: test_grouped_gpu.py's (half a step of the result's type and the FP32 sum's error).
"""

import pytest
import torch

from linalg_kernels_b200.grouped import grouped_matmul, grouped_outer
from linalg_kernels_b200.orthogonal import muon_update_, orthogonalize
from tests.test_grouped_gpu import _close, _problem, _randn, _reference, _reference_outer
from tests.test_orthogonal_gpu import _far, _input, _tolerance

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("rows,groups,k,n", [(65536, 8, 64, 128),   # y on 128-wide tiles
                                             (65536, 8, 128, 64),   # dx too
                                             (60001, 7, 72, 120),
                                             (2304, 1, 64, 2048)])  # too few 256-wide tiles
@pytest.mark.parametrize("transposed", [False, True])
def test_rows(rows, groups, k, n, transposed):
    counts = [rows // groups] * groups
    counts[-1] += rows - sum(counts)
    x, w, off, rows, k, n = _problem((counts, 0, 0, k, n), torch.bfloat16, transposed)
    offsets = torch.tensor(off, device=DEV)
    x.requires_grad_()
    w.requires_grad_()
    y = grouped_matmul(x, w, offsets)
    dy = _randn(3, rows, n)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    x, w, y = x.detach(), w.detach(), y.detach()
    for got, (want, size), terms in ((y, _reference(x, w, off), k),
                                     (dx, _reference(dy, w.transpose(1, 2), off), n),
                                     (dw, _reference_outer(x, dy, off), max(counts))):
        _close(got, want, size, terms)
    for _ in range(8):
        assert torch.equal(grouped_matmul(x, w, offsets), y)


def test_rows_of_no_group():
    """Tiles of zeros have no product to wait for: only the stores pace them."""
    rows, k, n = 65536, 64, 128
    x, w = _randn(1, rows, k), _randn(2, 2, k, n)
    offsets = torch.tensor([30000, 30100, 30300], device=DEV)
    y = grouped_matmul(x, w, offsets)
    want, size = _reference(x, w, offsets.tolist())
    _close(y, want, size, k)
    assert not y[:30000].any() and not y[30300:].any()


@pytest.mark.parametrize("k,n", [(64, 128), (256, 128), (1024, 120)])
def test_outer(k, n):
    groups, each = 600, 16
    a, b = _randn(1, groups * each, k), _randn(2, groups * each, n)
    off = list(range(0, groups * each + 1, each))
    offsets = torch.tensor(off, device=DEV)
    dw = grouped_outer(a, b, offsets)
    want, size = _reference_outer(a, b, off)
    _close(dw, want, size, each)
    for _ in range(8):
        assert torch.equal(grouped_outer(a, b, offsets), dw)


@pytest.mark.parametrize("shape", [(4, 8192, 128), (4, 128, 8192), (3, 9000, 100), (40, 200, 300)])
def test_orthogonalize(shape):
    x = _input(sum(shape), shape, torch.bfloat16, 1e-3)
    exact, tol = _tolerance(x, x.dtype, True)
    got = orthogonalize(x)
    assert _far(got, exact) <= tol
    for _ in range(4):
        assert torch.equal(orthogonalize(x), got)


@pytest.mark.parametrize("shape", [(40, 300, 521), (30, 521, 300), (40, 300, 520)])
def test_full_precision_to_unaligned_rows(shape):
    """Several tiles per pair whose results go to the caller's rows through the buffers that the next
    tile's old X is copied into."""
    x = _input(sum(shape), shape)
    exact, tol = _tolerance(x, x.dtype, False)
    got = orthogonalize(x)
    assert _far(got, exact) <= tol
    for _ in range(4):
        assert torch.equal(orthogonalize(x), got)
    momentum, param = torch.zeros_like(x), torch.zeros_like(x)
    muon_update_(param, x, momentum, lr=1.0, beta=0.0, nesterov=False, scale=1.0)
    assert torch.equal(momentum, x)  # 0 * 0 + 1 * x
    # 0 * 1 - 1 * 1 * o, every step exact but o
    assert torch.equal(param, -got)
