"""GPU: the grouped products and their gradients against 64-bit products, group by group.

Tolerance per element: half a step of the result's type, |y| eps / 2, plus the FP32 sum's error.
The sum takes K / 16 steps of 16 products, each rounded towards zero (2^-23 of the partial
sum) after an exact product sum; a partial sum is at most sum |x| |w|, so the error is at most
(K / 16 + 2) 2^-22 sum |x| |w|; and fp16's smallest step.
"""

import pytest
import torch

from linalg_kernels_b200 import _lib
from linalg_kernels_b200.grouped import grouped_matmul, grouped_outer

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _randn(seed, *shape, dtype=torch.bfloat16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, device=DEV, generator=g).to(dtype)


def _close(got, want, size, terms, where=""):
    eps = torch.finfo(got.dtype).eps
    bound = want.abs() * eps / 2 + size * (terms / 16 + 2) * 2.0 ** -22 + 2.0 ** -24
    off = (got.double() - want).abs()
    assert (off <= bound).all(), (where, (off / bound).max().item())


def _reference(x, w, off):
    y = torch.zeros(x.shape[0], w.shape[2], dtype=torch.float64, device=x.device)
    size = torch.zeros_like(y)
    for e in range(len(off) - 1):
        i, j = off[e], off[e + 1]
        y[i:j] = x[i:j].double() @ w[e].double()
        size[i:j] = x[i:j].double().abs() @ w[e].double().abs()
    return y, size


def _reference_outer(a, b, off):
    dw = torch.zeros(len(off) - 1, a.shape[1], b.shape[1], dtype=torch.float64, device=a.device)
    size = torch.zeros_like(dw)
    for e in range(len(off) - 1):
        i, j = off[e], off[e + 1]
        dw[e] = a[i:j].double().T @ b[i:j].double()
        size[e] = a[i:j].double().abs().T @ b[i:j].double().abs()
    return dw, size


# rows of the groups, rows in front of them, rows behind them, k, n
CASES = [
    ([256, 256], 0, 0, 64, 256),
    ([128], 0, 0, 64, 128),
    ([1], 0, 0, 8, 8),
    ([1, 0, 2, 0], 0, 3, 64, 72),
    ([0, 0, 5], 2, 0, 128, 256),
    ([0, 0], 4, 5, 72, 64),
    ([300, 1, 17, 255, 257, 0, 33], 0, 0, 200, 520),
    ([63, 64, 65, 15, 16, 17], 1, 70, 256, 384),
    ([700, 3, 900], 0, 11, 1024, 640),
    ([5] * 40 + [0] * 30, 0, 0, 512, 1024),
    ([37, 80], 3, 2, 77, 131),
    ([1000, 20], 0, 0, 129, 64),
    ([2] * 1000 + [0] * 24, 0, 6, 64, 64),
    ([2500, 1500, 96], 0, 0, 2048, 1024),
]


def _problem(case, dtype, transposed, seed=0):
    counts, front, behind, k, n = case
    off = [front]
    for c in counts:
        off.append(off[-1] + c)
    rows = off[-1] + behind
    x = _randn(seed + 1, rows, k, dtype=dtype)
    w = _randn(seed + 2, len(counts), *((n, k) if transposed else (k, n)), dtype=dtype)
    w = w.transpose(1, 2) if transposed else w
    return x, w, off, rows, k, n


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"g{len(c[0])}r{sum(c[0])}k{c[3]}n{c[4]}")
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("transposed", [False, True])
def test_forward_and_gradients(case, dtype, transposed):
    x, w, off, rows, k, n = _problem(case, dtype, transposed)
    offsets = torch.tensor(off, device=DEV, dtype=torch.int64 if transposed else torch.int32)
    y = grouped_matmul(x, w, offsets)
    want, size = _reference(x, w, off)
    _close(y, want, size, k, "y")
    x.requires_grad_()
    w.requires_grad_()
    y2 = grouped_matmul(x, w, offsets)
    assert torch.equal(y2, y)
    dy = _randn(3, rows, n, dtype=dtype)
    dx, dw = torch.autograd.grad(y2, (x, w), dy)
    want, size = _reference(dy, w.detach().transpose(1, 2), off)
    _close(dx, want, size, n, "dx")
    want, size = _reference_outer(x.detach(), dy, off)
    _close(dw, want, size, max(case[0]), "dw")
    assert dx.shape == x.shape and dw.shape == w.shape
    with torch.no_grad():
        again = grouped_outer(x, dy, offsets)
    _close(again, want, size, max(case[0]), "outer")


def test_gradients_against_differences():
    """d sum(y * r) along a direction, against the exact difference: y is linear in x and in w."""
    x, w, off, rows, k, n = _problem(([30, 0, 45], 0, 0, 64, 72), torch.float16, False)
    offsets = torch.tensor(off, device=DEV)
    r = _randn(5, rows, n, dtype=torch.float16)
    x.requires_grad_(), w.requires_grad_()
    dx, dw = torch.autograd.grad(grouped_matmul(x, w, offsets), (x, w), r)
    hx, hw = _randn(6, rows, k, dtype=torch.float16), _randn(7, *w.shape, dtype=torch.float16)
    for grad, a, b in ((dx, hx, w), (dw, x, hw)):
        y, size = _reference(a.detach(), b.detach(), off)
        h = hx if grad is dx else hw
        want = (y * r.double()).sum().item()
        got = (grad.double() * h.double()).sum().item()
        # each gradient element is off by half an fp16 step of itself (+ its FP32 sum)
        bound = (grad.double().abs() * h.double().abs()).sum().item() * 2.0 ** -11 + \
            (size * r.double().abs()).sum().item() * 16 * 2.0 ** -22
        assert abs(got - want) <= bound


def test_rows_of_no_group():
    """Zero in a fresh result, untouched in a given one; what lies there reaches no result."""
    counts, k, n = [70, 0, 90], 96, 200
    off = [5, 75, 75, 165]
    rows = 180
    x, dy = _randn(1, rows, k), _randn(2, rows, n)
    w = _randn(3, 3, k, n)
    offsets = torch.tensor(off, device=DEV)
    clean_y, clean_dw = grouped_matmul(x, w, offsets), grouped_outer(x, dy, offsets)
    for t in (x, dy):
        t[:5] = float("nan")
        t[165:] = float("inf")
    y = grouped_matmul(x, w, offsets)
    assert torch.equal(y, clean_y) and not y[:5].any() and not y[165:].any()
    out = torch.full((rows, n), 3.0, device=DEV, dtype=torch.bfloat16)
    assert grouped_matmul(x, w, offsets, out=out) is out
    assert torch.equal(out[5:165], clean_y[5:165])
    assert (out[:5] == 3).all() and (out[165:] == 3).all()
    assert torch.equal(grouped_outer(x, dy, offsets), clean_dw)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_non_finite_rows_stay_in_their_group(bad):
    off = [0, 37, 101, 230]
    x, dy, w = _randn(1, 230, 64), _randn(2, 230, 136), _randn(3, 3, 64, 136)
    offsets = torch.tensor(off, device=DEV)
    y, dw = grouped_matmul(x, w, offsets), grouped_outer(x, dy, offsets)
    x[37:101] = bad
    dy[37:101] = bad
    y2, dw2 = grouped_matmul(x, w, offsets), grouped_outer(x, dy, offsets)
    keep = [0, 2]
    assert torch.equal(dw2[keep], dw[keep])
    assert torch.equal(y2[:37], y[:37]) and torch.equal(y2[101:], y[101:])
    assert not torch.isfinite(dw2[1]).any()


def test_offsets_that_are_not_valid_are_clamped():
    """Decreasing, negative and too large offsets: no row outside x is touched, no fault."""
    x, dy, w = _randn(1, 100, 64), _randn(2, 100, 72), _randn(3, 4, 64, 72)
    offsets = torch.tensor([-7, 40, 20, 70, 1 << 40], device=DEV)
    off = [0, 40, 40, 70, 100]
    want, size = _reference(x, w, off)
    _close(grouped_matmul(x, w, offsets), want, size, 64)
    want, size = _reference_outer(x, dy, off)
    _close(grouped_outer(x, dy, offsets), want, size, 40)


def test_layouts():
    """Pitched rows, unaligned bases, transposed and strided operands, an expanded gradient."""
    off = [0, 33, 100]
    offsets = torch.tensor(off, device=DEV)
    base, wbase = _randn(1, 101, 150), _randn(2, 2, 70, 90)
    for x in (base[1:, :64], base[:100, 3:67], base[:100, ::2][:, :64],
              _randn(4, 64, 100).T):
        for w in (wbase[:, :64, :80], wbase[:, 3:67, 5:85], wbase.transpose(1, 2)[:, :64, :],
                  wbase[:, :64, ::2], wbase[:1, :64].expand(2, 64, 90)):
            got = grouped_matmul(x, w, offsets)
            assert torch.equal(got, grouped_matmul(x.contiguous(), w.contiguous(), offsets))
    x = base[:100, :64].contiguous().requires_grad_()
    w = wbase[:, :64, :80].contiguous().requires_grad_()
    grouped_matmul(x, w, offsets).sum().backward()  # a gradient of strides (0, 0)
    ones = torch.ones(100, 80, device=DEV, dtype=torch.bfloat16)
    assert torch.equal(w.grad, grouped_outer(x.detach(), ones, offsets))
    shared = wbase[:1, :64, :80].clone().requires_grad_()  # one matrix for every group
    y = grouped_matmul(x.detach(), shared.expand(2, 64, 80), offsets)
    y.backward(ones)
    each = grouped_outer(x.detach(), ones, offsets).double().sum(0)
    assert ((shared.grad[0].double() - each).abs() <= each.abs() * 2.0 ** -8 + 1e-6).all()
    out = torch.full((100, 88), 2.0, device=DEV, dtype=torch.bfloat16)
    with torch.no_grad():
        got = grouped_matmul(x, w, offsets, out=out[:, 4:84])
        assert torch.equal(got, grouped_matmul(x, w, offsets))
        assert (out[:, :4] == 2).all() and (out[:, 84:] == 2).all()
        big = torch.full((2, 66, 83), 2.0, device=DEV, dtype=torch.bfloat16)
        got = grouped_outer(x, ones, offsets, out=big[:, 1:65, 2:82])
        assert torch.equal(got, grouped_outer(x, ones, offsets))
        assert (big[:, 0] == 2).all() and (big[:, 65] == 2).all() and (big[:, :, 82:] == 2).all()


def test_empty():
    offsets = torch.zeros(4, device=DEV, dtype=torch.int32)
    w = _randn(1, 3, 64, 72)
    assert grouped_matmul(_randn(2, 0, 64), w, offsets).shape == (0, 72)
    assert not grouped_outer(_randn(2, 0, 64), _randn(3, 0, 72), offsets).any()
    assert grouped_matmul(_randn(2, 5, 64), _randn(1, 3, 64, 0), offsets).shape == (5, 0)
    assert not grouped_matmul(_randn(2, 5, 0), _randn(1, 3, 0, 8), offsets).any()
    assert not grouped_matmul(_randn(2, 5, 64), _randn(1, 0, 64, 8), offsets[:1]).any()
    x, ww = _randn(2, 5, 64).requires_grad_(), w.clone().requires_grad_()
    grouped_matmul(x, ww, offsets).sum().backward()
    assert not x.grad.any() and not ww.grad.any()


def test_long_offsets_past_32_bits():
    """Rows behind 2^31 elements of x and of the result are addressed as themselves."""
    k = n = 1024
    rows = (1 << 31) // k + 300
    x = torch.zeros(rows, k, device=DEV, dtype=torch.bfloat16)
    tail = _randn(1, 200, k)
    x[-200:].copy_(tail)
    w = _randn(2, 2, k, n)
    offsets = torch.tensor([0, rows - 200, rows], device=DEV)
    y = grouped_matmul(x, w, offsets)
    assert not y[:-200].any()
    want = grouped_matmul(tail, w[1:], torch.tensor([0, 200], device=DEV))
    assert torch.equal(y[-200:], want)
    dw = grouped_outer(x, y, offsets)
    assert not dw[0].any()
    assert torch.equal(dw[1], grouped_outer(tail, want, torch.tensor([0, 200], device=DEV))[0])


def test_many_matrices_past_32_bits():
    groups, k, n = 520, 2048, 2056
    w = torch.zeros(groups, k, n, device=DEV, dtype=torch.bfloat16)
    w[-1].copy_(_randn(1, k, n))
    x = _randn(2, 40, k)
    off = torch.zeros(groups + 1, device=DEV, dtype=torch.int32)
    off[1:] = 10
    off[-1] = 40
    y = grouped_matmul(x, w, off)
    assert not y[:10].any()
    assert torch.equal(y[10:], grouped_matmul(x[10:], w[-1:], off[-1:].new_tensor([0, 30])))


def test_graph_replays_other_group_sizes():
    """Captured with its backward pass; the replay sees the new offsets."""
    rows, k, n = 300, 128, 192
    x, w, dy = _randn(1, rows, k), _randn(2, 4, k, n), _randn(3, rows, n)
    offsets = torch.tensor([0, 100, 100, 250, 300], device=DEV)
    grouped_matmul(x, w, offsets)
    torch.cuda.synchronize()
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = grouped_matmul(xs, ws, offsets)
        dx, dw = torch.autograd.grad(y, (xs, ws), dy)
    offsets.copy_(torch.tensor([3, 20, 180, 180, 290], device=DEV))
    graph.replay()
    torch.cuda.synchronize()
    off = offsets.tolist()
    want, size = _reference(x, w, off)
    _close(y.detach(), want, size, k)
    want, size = _reference(dy, w.transpose(1, 2), off)
    _close(dx, want, size, n)
    want, size = _reference_outer(x, dy, off)
    _close(dw, want, size, 160)


def test_capture_with_few_rows_and_inference_mode():
    x, w = _randn(1, 40, 128), _randn(2, 8, 128, 192)
    offsets = torch.tensor([0, 3, 3, 10, 12, 20, 25, 30, 38], device=DEV, dtype=torch.int32)
    grouped_matmul(x, w, offsets)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = grouped_matmul(x, w, offsets)
    offsets.copy_(torch.tensor([1, 1, 2, 30, 31, 31, 32, 39, 40], device=DEV))
    x.mul_(2)
    graph.replay()
    want, size = _reference(x, w, offsets.tolist())
    _close(y, want, size, 128)
    with torch.inference_mode():
        out = torch.empty(40, 192, device=DEV, dtype=torch.bfloat16)
        grouped_matmul(x, w, offsets, out=out)
        assert torch.equal(grouped_matmul(x, w, offsets)[1:], out[1:])
        grouped_outer(x, out, offsets, out=torch.empty(8, 128, 192, device=DEV, dtype=torch.bfloat16))


def test_two_queues():
    x, w = _randn(1, 900, 256), _randn(2, 6, 256, 512)
    offs = [torch.tensor(o, device=DEV) for o in ([0, 5, 300, 300, 600, 880, 900],
                                                  [0, 500, 501, 502, 700, 800, 850])]
    want = [grouped_matmul(x, w, o) for o in offs]
    torch.cuda.synchronize()
    queues = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i in (0, 1):
            with torch.cuda.stream(queues[i]):
                got[i].append(grouped_matmul(x, w, offs[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(y, want[i]) for y in got[i])


# pairs' tiles of 512 columns: of the rows' products, of their gradients and of the matrices'
LARGE = [
    ([3000, 1, 0, 4000, 4999], 0, 0, 1111, 1300),
    ([2600, 2600], 0, 0, 1100, 2500),
    ([1500, 3670], 7, 23, 1100, 2500),
    ([4001, 3999], 0, 0, 1200, 2568),
    ([1000] * 15 + [0], 130, 254, 2048, 2056),
    ([3000, 1, 0, 4000, 4999], 3, 6, 2001, 2037),
    ([3000, 1, 0, 4000, 4999], 300, 6, 2000, 2040),
]


@pytest.mark.parametrize("case", LARGE, ids=lambda c: f"g{len(c[0])}r{sum(c[0])}k{c[3]}n{c[4]}")
@pytest.mark.parametrize("transposed", [False, True])
def test_large(case, transposed):
    x, w, off, rows, k, n = _problem(case, torch.bfloat16, transposed)
    offsets = torch.tensor(off, device=DEV)
    x.requires_grad_()
    w.requires_grad_()
    y = grouped_matmul(x, w, offsets)
    dy = _randn(3, rows, n)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    x, w, y = x.detach(), w.detach(), y.detach()
    want, size = _reference(x, w, off)
    _close(y, want, size, k, "y")
    want, size = _reference(dy, w.transpose(1, 2), off)
    _close(dx, want, size, n, "dx")
    want, size = _reference_outer(x, dy, off)
    _close(dw, want, size, max(case[0]), "dw")
    # given results of unaligned rows: not by boxes
    out = torch.full((rows, n + 3), 2.0, device=DEV, dtype=torch.bfloat16)
    grouped_matmul(x, w, offsets, out=out[:, 1:n + 1])
    assert torch.equal(out[off[0]:off[-1], 1:n + 1], y[off[0]:off[-1]])
    assert (out[:, 0] == 2).all() and (out[:, n + 1:] == 2).all()
    assert (out[:off[0]] == 2).all() and (out[off[-1]:] == 2).all()
    big = torch.full((len(off) - 1, k + 1, n + 3), 2.0, device=DEV, dtype=torch.bfloat16)
    grouped_outer(x, dy, offsets, out=big[:, :k, 1:n + 1])
    assert torch.equal(big[:, :k, 1:n + 1], dw)
    assert (big[:, k] == 2).all() and (big[:, :, 0] == 2).all() and (big[:, :, n + 1:] == 2).all()


def test_status_word_is_clear():
    import ctypes
    assert _lib.load().chol_status_check(
        ctypes.c_void_p(_lib.current_queue(torch.device(DEV)))) == _lib.CHOL_OK
