"""GPU: nothing beside a given result is written, whatever its width and pitch. (A bulk store of a box
ends on a 16-byte chunk, not on the last column.)

The values are compared with the call's own fresh result, whose rows are packed.
"""

import pytest
import torch

from linalg_kernels_b200.grouped import grouped_matmul, grouped_outer
from linalg_kernels_b200.orthogonal import muon_update_, orthogonalize

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
MARK = 7.0


def _rand(*shape, dtype=torch.bfloat16):
    g = torch.Generator(device=DEV).manual_seed(sum(shape))
    return torch.randn(*shape, device=DEV, generator=g).to(dtype)


def _frame(shape, dtype, start):
    """A view of `shape` in a larger array of MARK, its rows 16-byte aligned where `start` is."""
    m, n = shape[-2:]
    pitch = (start + n + 7) // 8 * 8 + 8
    big = torch.full((*shape[:-2], m + 3, pitch), MARK, device=DEV, dtype=dtype)
    return big, big[..., :m, start:start + n]


def _untouched(big, view):
    rest = big.clone()
    m, n = view.shape[-2:]
    start = (view.data_ptr() - big.data_ptr()) // big.element_size()
    rest[..., :m, start:start + n] = MARK
    return bool((rest == MARK).all())


@pytest.mark.parametrize("n", [1, 2, 5, 7, 8, 9, 31, 63, 65, 127, 131, 255, 257, 511, 516, 1027, 2050])
@pytest.mark.parametrize("start", [0, 8, 3])
@pytest.mark.parametrize("rows", [20, 1300])  # tiles of few rows, and of 256
def test_grouped_matmul(n, start, rows):
    k, off = 64, [3, rows // 3, rows // 3, rows - 5]
    x, w = _rand(rows, k), _rand(3, k, n)
    offsets = torch.tensor(off, device=DEV)
    want = grouped_matmul(x, w, offsets)
    big, out = _frame((rows, n), x.dtype, start)
    grouped_matmul(x, w, offsets, out=out)
    assert torch.equal(out[3:rows - 5], want[3:rows - 5])
    assert (out[:3] == MARK).all() and (out[rows - 5:] == MARK).all()
    assert _untouched(big, out)


@pytest.mark.parametrize("k,n", [(1, 1), (40, 5), (131, 9), (300, 255), (257, 516), (100, 1027)])
@pytest.mark.parametrize("start", [0, 8, 3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_grouped_outer(k, n, start, dtype):
    a, b = _rand(700, k, dtype=dtype), _rand(700, n, dtype=dtype)
    offsets = torch.tensor([0, 100, 100, 690], device=DEV)
    want = grouped_outer(a, b, offsets)
    big, out = _frame((3, k, n), dtype, start)
    grouped_outer(a, b, offsets, out=out)
    assert torch.equal(out, want) and _untouched(big, out)


def test_wide_tiles():
    """512-wide tiles, in all three."""
    x, w = _rand(6000, 1100), _rand(2, 1100, 2501)
    offsets = torch.tensor([0, 2600, 6000], device=DEV)
    want = grouped_matmul(x, w, offsets)
    big, out = _frame((6000, 2501), x.dtype, 0)
    grouped_matmul(x, w, offsets, out=out)
    assert torch.equal(out, want) and _untouched(big, out)
    want_w = grouped_outer(x, want, offsets)
    big, out = _frame((2, 1100, 2501), x.dtype, 8)
    grouped_outer(x, want, offsets, out=out)
    assert torch.equal(out, want_w) and _untouched(big, out)
    m = _rand(1, 2601, 2701)
    big, out = _frame(m.shape, m.dtype, 0)
    orthogonalize(m, 2, out=out)
    assert torch.equal(out, orthogonalize(m, 2)) and _untouched(big, out)


@pytest.mark.parametrize("m,n", [(5, 3), (64, 61), (100, 1501), (1501, 100), (200, 251), (251, 200),
                                 (300, 257), (257, 300), (257, 301), (129, 700), (700, 131)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("precision", ["half", "full"])
@pytest.mark.parametrize("start", [0, 8, 3])
def test_orthogonalize_and_step(m, n, dtype, precision, start):
    x = _rand(2, m, n, dtype=dtype)
    want = orthogonalize(x, 2, precision=precision)
    big, out = _frame(x.shape, dtype, start)
    orthogonalize(x, 2, precision=precision, out=out)
    assert torch.equal(out, want) and _untouched(big, out)
    args = dict(lr=0.5, steps=2, precision=precision, scale=1.0)
    p, mom = _rand(2, m, n, dtype=dtype), torch.ones(2, m, n, device=DEV)
    big_p, param = _frame(x.shape, dtype, start)
    big_m, momentum = _frame(x.shape, torch.float32, start)
    param.copy_(p), momentum.copy_(mom)
    muon_update_(param, x, momentum, **args)
    muon_update_(p, x, mom, **args)
    assert torch.equal(param, p) and torch.equal(momentum, mom)
    assert _untouched(big_p, param) and _untouched(big_m, momentum)
