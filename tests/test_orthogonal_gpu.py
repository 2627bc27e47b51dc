"""GPU: orthogonalize and muon_update_ against the same iteration in 64 bits.

Tolerance. The half-precision iteration rounds X, G and B of every step to fp16. `_model` runs
the iteration in 64 bits with exactly these roundings; its distance to the unrounded iteration is
the error the number format brings for this input. The kernel's sums differ from the model's in
their last FP32 bits, which moves some roundings to the neighbouring fp16 number: other roundings
of the same size, independent of the model's, so its error is allowed twice the model's (plus
half a step of the result's type). The full-precision iteration keeps 22 bits and FP32 sums; its
model is the iteration in FP32 (torch), and four times that error is allowed: two roundings
towards zero (2^-23 each) per FP32 rounding to nearest (2^-24).
"""

import math

import pytest
import torch

from linalg_kernels_b200 import _lib
from linalg_kernels_b200.orthogonal import DEFAULT_COEFFICIENTS, muon_update_, orthogonalize

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _input(seed, shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, device=DEV, generator=g) * scale).to(dtype)


def _iterate(x, steps, coefs, eps, work, keep):
    """The iteration in type `work`; keep(t) rounds what the kernel stores."""
    x = x.to(work)
    x = keep(x / (x.double().square().sum((-2, -1), keepdim=True).sqrt().to(work) + eps))
    wide = x.shape[-2] <= x.shape[-1]
    for k in range(steps):
        a, b, c = coefs[k] if isinstance(coefs[0], tuple) else coefs
        g = keep(x @ x.mT if wide else x.mT @ x)
        p = keep(b * g + c * (g @ g))
        y = a * x + (p @ x if wide else x @ p)
        x = keep(y) if k + 1 < steps else y
    return x


def _exact(x, steps=5, coefs=DEFAULT_COEFFICIENTS, eps=1e-7):
    return _iterate(x, steps, coefs, eps, torch.float64, lambda t: t)


def _model(x, half, steps=5, coefs=DEFAULT_COEFFICIENTS, eps=1e-7):
    if half:
        return _iterate(x, steps, coefs, eps, torch.float64,
                        lambda t: (t * 1024).half().double() / 1024)
    return _iterate(x, steps, coefs, eps, torch.float32, lambda t: t).double()


def _far(a, b):
    return ((a.double() - b).square().sum((-2, -1)).sqrt() / b.square().sum((-2, -1)).sqrt()
            ).max().item()


def _tolerance(x, dtype, half, **kw):
    exact = _exact(x, **kw)
    model = _far(_model(x, half, **kw), exact)
    return exact, (2 if half else 4) * model + torch.finfo(dtype).eps / 2


SHAPES = [(1, 128, 128), (3, 64, 64), (2, 256, 256), (1, 512, 512), (2, 200, 328), (2, 328, 200),
          (1, 1000, 601), (1, 601, 1000), (5, 33, 17), (5, 17, 33), (2, 1, 40), (2, 40, 1),
          (3, 1, 1), (1, 2048, 130), (1, 130, 2048), (4, 65, 1025), (300, 16, 24), (1, 768, 1536),
          # on chip: one matrix or several per tile, split over 2, 4 and 8 CTAs, odd sizes
          (1, 128, 512), (2, 128, 513), (1, 100, 700), (2, 700, 100), (1, 90, 1537), (1, 4096, 128),
          (1, 127, 4096), (5, 1, 3000), (6, 43, 64), (9, 31, 1), (7, 64, 129), (130, 1, 5),
          (3, 1536, 20),
          # on chip over two CTAs, odd edges, both ways; and just beyond
          (1, 256, 256), (3, 130, 190), (80, 256, 256), (2, 200, 256), (2, 256, 200), (1, 129, 129),
          (3, 255, 131), (3, 131, 255), (2, 257, 256), (150, 129, 257), (5, 512, 512), (40, 300, 520)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float16])
def test_orthogonalize(shape, dtype):
    x = _input(sum(shape), shape, dtype, 1e-3 if dtype is not torch.float16 else 1.0)
    exact, tol = _tolerance(x, dtype, dtype is torch.bfloat16)
    before = x.clone()
    got = orthogonalize(x)
    assert got.dtype == dtype and got.shape == x.shape
    assert torch.equal(x, before)
    far = _far(got, exact)
    assert far <= tol, (far, tol)
    assert torch.equal(got, orthogonalize(x))  # the same bits every time


@pytest.mark.parametrize("dtype,precision", [(torch.float32, "half"), (torch.bfloat16, "full")])
@pytest.mark.parametrize("shape", [(2, 96, 200), (1, 300, 140)])
def test_precision_argument(dtype, precision, shape):
    x = _input(5, shape, dtype)
    exact, tol = _tolerance(x, dtype, precision == "half")
    assert _far(orthogonalize(x, precision=precision), exact) <= tol


@pytest.mark.parametrize("steps", [1, 2, 8])
def test_steps_and_coefficients(steps):
    x = _input(steps, (2, 100, 150), torch.bfloat16)
    coefs = tuple((3.0 - 0.1 * k, -3.2, 1.2 + 0.05 * k) for k in range(steps))
    exact, tol = _tolerance(x, x.dtype, True, steps=steps, coefs=coefs)
    assert _far(orthogonalize(x, steps, coefficients=coefs), exact) <= tol
    assert torch.equal(orthogonalize(x, steps, coefficients=[list(c) for c in coefs]),
                       orthogonalize(x, steps, coefficients=coefs))


def test_singular_values_move_to_one():
    x = _input(11, (1, 512, 512), torch.float32)
    s = torch.linalg.svdvals(orthogonalize(x).double())[0]
    start = torch.linalg.svdvals(x.double())[0] / x.double().norm()
    # values above 1e-2 of the norm reach the band that these coefficients keep, [0.67, 1.21]
    big = s[start > 1e-2]
    assert big.min() > 0.6 and s.max() < 1.3


@pytest.mark.parametrize("magnitude", [1e-30, 1e-12, 1e12, 1e30])
def test_magnitudes(magnitude):
    """The norm is taken in 64 bits, so neither its squares nor the start value leave the range."""
    x = (_input(2, (2, 80, 120)).double() * magnitude).to(torch.bfloat16)
    got = orthogonalize(x, eps=0.0)
    exact, tol = _tolerance(x.double() / magnitude, x.dtype, True, eps=0.0)
    assert _far(got, exact) <= tol


@pytest.mark.parametrize("m,n", [(48, 80), (10, 30), (30, 10), (128, 128), (60, 900), (200, 250), (300, 260)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_zero_and_non_finite_matrices(m, n, dtype):
    """(Matrices of 48 x 80 and 10 x 30 share a tile.)"""
    x = _input(3, (5, m, n), dtype)
    x[1] = 0
    x[2, 5, 7] = float("nan")
    x[3, 0, 0] = float("inf")
    got = orthogonalize(x)
    assert torch.equal(got[1], torch.zeros_like(got[1]))
    assert got[2].isnan().all() and got[3].isnan().all()
    clean = orthogonalize(x[[0, 4]])
    assert torch.equal(got[[0, 4]], clean)


@pytest.mark.parametrize("m,n", [(60, 100), (100, 60), (260, 140)])
def test_layouts(m, n):
    """Pitched, transposed, strided and expanded inputs; results equal the contiguous call's."""
    dtype = torch.bfloat16
    base = _input(7, (2, 3, m + 3, n + 5), dtype)
    want = orthogonalize(base[..., 1:m + 1, 2:n + 2].contiguous())
    got = orthogonalize(base[..., 1:m + 1, 2:n + 2])
    assert torch.equal(got, want) and got.is_contiguous()
    t = base[..., 1:m + 1, 2:n + 2].contiguous().mT  # columns contiguous: worked on as it lies
    got = orthogonalize(t)
    assert torch.equal(got, want.mT) and got.stride() == t.stride()
    wide = _input(8, (2, m, 2 * n), dtype)[..., ::2]
    assert torch.equal(orthogonalize(wide), orthogonalize(wide.contiguous()))
    one = _input(9, (m, n), dtype)
    assert torch.equal(orthogonalize(one.expand(3, m, n)), orthogonalize(one).expand(3, m, n))
    swapped = _input(10, (2, 3, m, n), dtype).transpose(0, 1)
    assert torch.equal(orthogonalize(swapped), orthogonalize(swapped.contiguous()))


def test_out():
    x = _input(12, (3, 70, 90), torch.float32)
    want = orthogonalize(x)
    out = torch.full((3, 75, 99), 7.0, device=DEV)
    got = orthogonalize(x, out=out[:, 2:72, 4:94])
    assert got.data_ptr() == out[:, 2:72, 4:94].data_ptr() and torch.equal(got, want)
    rest = out.clone()
    rest[:, 2:72, 4:94] = 7.0
    assert (rest == 7.0).all()  # nothing around it is written
    same = x.clone()
    assert orthogonalize(same, out=same) is same and torch.equal(same, want)
    shifted = torch.empty(3 * 70 * 90 + 90, device=DEV)
    src, dst = shifted[:18900].view(3, 70, 90), shifted[90:].view(3, 70, 90)
    src.copy_(x)
    assert torch.equal(orthogonalize(src, out=dst), want)  # overlapping: as if from a copy
    t = torch.empty(3, 90, 70, device=DEV).mT
    assert torch.equal(orthogonalize(x, out=t), orthogonalize(x.mT.contiguous()).mT)


def test_empty():
    for shape in ((0, 4, 4), (2, 0, 5), (2, 5, 0), (0, 0)):
        x = torch.empty(*shape, device=DEV, dtype=torch.bfloat16)
        assert orthogonalize(x).shape == x.shape


@pytest.mark.parametrize("shape", [(1, 128, 128), (2, 256, 512), (3, 200, 100), (2, 200, 230),
                                   (3, 251, 145)])
@pytest.mark.parametrize("types", [(torch.bfloat16, torch.bfloat16, torch.float32),
                                   (torch.float32, torch.float32, torch.float32),
                                   (torch.float32, torch.bfloat16, torch.bfloat16),
                                   (torch.float16, torch.float16, torch.float32)])
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_update(shape, types, nesterov):
    pt, gt, mt = types
    lr, beta, decay = 0.05, 0.9, 0.2
    param = _input(1, shape, pt, shape[-1] ** -0.5)
    grad, momentum = _input(2, shape, gt, 1e-3 if gt is not torch.float16 else 1.0), _input(3, shape, mt, 1e-3)
    p64, g64, m64 = param.double(), grad.double(), momentum.double()
    new_m = beta * m64 + (1 - beta) * g64
    version = param._version
    assert muon_update_(param, grad, momentum, lr=lr, beta=beta, nesterov=nesterov,
                        weight_decay=decay) is param
    assert param._version > version
    # momentum: two products and a sum in FP32 (3 half steps of 2^-24), then its own rounding
    size = beta * m64.abs() + (1 - beta) * g64.abs()
    bound = size * 3 * 2.0 ** -24 + new_m.abs() * torch.finfo(mt).eps / 2
    assert ((momentum.double() - new_m).abs() <= bound + 1e-45).all()
    # the direction is taken from the momentum as stored
    stored = momentum.double()
    u = beta * stored + (1 - beta) * g64 if nesterov else stored
    scale = math.sqrt(max(1.0, shape[-2] / shape[-1]))
    o, tol = _tolerance(u, torch.float32, pt is torch.bfloat16)
    want = (1 - lr * decay) * p64 - lr * scale * o
    off = (param.double() - want).square().sum((-2, -1)).sqrt()
    allowed = (torch.finfo(pt).eps / 2 + 3 * 2.0 ** -24) * want.square().sum((-2, -1)).sqrt() + \
        lr * scale * tol * o.square().sum((-2, -1)).sqrt()
    assert (off <= allowed).all(), (off, allowed)


@pytest.mark.parametrize("m,n", [(6, 8), (40, 30), (150, 140)])
def test_smallest_and_largest_norms(m, n):
    """FP32 subnormals and values whose squares pass FP32's range."""
    base = _input(6, (3, m, n))
    want = orthogonalize(base, eps=0.0)
    for power in (-146 if m < 100 else -140, 120):
        x = torch.ldexp(base.double(), torch.tensor(float(power), device=DEV)).float()
        exact, tol = _tolerance(x.double() * 2.0 ** -power, torch.float32, False, eps=0.0)
        assert _far(orthogonalize(x, eps=0.0), exact) <= tol
    assert want.isfinite().all()
    assert orthogonalize(torch.zeros_like(base)).eq(0).all()


def test_muon_layouts_and_scale():
    """A transposed weight (its gradient row-major), a pitched one, and an explicit scale."""
    m, n = 96, 160
    args = dict(lr=0.1, beta=0.5, weight_decay=0.1)
    p, g, mo = (_input(i, (2, m, n), torch.float32, 0.1) for i in (1, 2, 3))
    want_p, want_m = p.clone(), mo.clone()
    muon_update_(want_p, g, want_m, **args, scale=1.5)
    big = torch.zeros(2, m, n + 4, device=DEV)
    pp = big[..., :n]
    pp.copy_(p)
    mm = mo.clone()
    muon_update_(pp, g, mm, **args, scale=1.5)
    assert torch.equal(pp, want_p) and torch.equal(mm, want_m) and (big[..., n:] == 0).all()
    pt, mt = p.mT.contiguous().mT, mo.mT.contiguous().mT
    muon_update_(pt, g, mt, **args, scale=1.5)
    assert torch.allclose(pt, want_p, rtol=0, atol=1e-5) and torch.equal(mt, want_m)


def test_two_queues_and_graph():
    """Each call owns its workspace: calls on two queues at once do not mix, and a captured call
    replays on new contents."""
    a, b = _input(1, (4, 300, 260), torch.bfloat16), _input(2, (4, 300, 260), torch.bfloat16)
    want_a, want_b = orthogonalize(a), orthogonalize(b)
    torch.cuda.synchronize()
    queues = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for i, x in enumerate((a, b)):
            with torch.cuda.stream(queues[i]):
                got[i].append(orthogonalize(x))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want_a) for y in got[0])
    assert all(torch.equal(y, want_b) for y in got[1])

    x = a.clone()
    param, grad, mom = b.clone(), a.clone(), torch.zeros(4, 300, 260, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = orthogonalize(x)
        muon_update_(param, grad, mom, lr=0.1)
    x.copy_(b)
    ref, ref_m = b.clone(), torch.zeros_like(mom)
    graph.replay()
    muon_update_(ref, grad, ref_m, lr=0.1)
    assert torch.equal(y, want_b) and torch.equal(param, ref) and torch.equal(mom, ref_m)
    graph.replay()
    muon_update_(ref, grad, ref_m, lr=0.1)
    torch.cuda.synchronize()
    assert torch.equal(param, ref) and torch.equal(mom, ref_m)


@pytest.mark.parametrize("shape", [(3, 64, 64), (2, 100, 900), (2, 200, 256), (2, 300, 260)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_capture_of_every_kernel(shape, dtype):
    """One launch per tile, clusters, pairs and the products, captured and replayed twice."""
    x, other = _input(1, shape, dtype), _input(2, shape, dtype)
    want = orthogonalize(other)
    static = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = orthogonalize(static)
    static.copy_(other)
    for _ in range(2):
        y.zero_()
        graph.replay()
        assert torch.equal(y, want)


def test_inference_mode():
    with torch.inference_mode():
        x = _input(1, (2, 60, 70), torch.bfloat16)
        y = orthogonalize(x)
        assert torch.equal(orthogonalize(x, out=torch.empty_like(x)), y)
        p, m = x.clone(), torch.zeros(2, 60, 70, device=DEV)
        muon_update_(p, x, m, lr=0.1)


def test_large_batch_past_32_bit_offsets():
    """The last matrix of an input longer than 2^31 elements gets its own result."""
    batch, m, n = 130, 2048, 8200
    x = torch.zeros(batch, m, n, device=DEV, dtype=torch.bfloat16)
    one = _input(4, (m, n), torch.bfloat16)
    x[-1].copy_(one)
    got = orthogonalize(x, 1, out=x)
    assert torch.equal(got[-1], orthogonalize(one, 1))
    assert not got[:-1].any()


# pairs' tiles of 512 columns: of X X^T, of X^T X, of P X and of X P; ragged edges, a last column tile
# that lies half outside, odd numbers of row tiles
LARGE = [(2, 2304, 2600), (2, 2600, 2304), (1, 2600, 2700), (1, 2700, 2600), (7, 1290, 1400),
         (7, 1400, 1290)]


@pytest.mark.parametrize("shape", LARGE)
def test_large(shape):
    x = _input(sum(shape), shape, torch.bfloat16, 1e-3)
    exact, tol = _tolerance(x, x.dtype, True)
    got = orthogonalize(x)
    assert _far(got, exact) <= tol
    assert torch.equal(got, orthogonalize(x))


def test_large_in_half_precision_to_float32():
    x = _input(4, (1, 2600, 2701))
    exact, tol = _tolerance(x, x.dtype, True)
    assert _far(orthogonalize(x, precision="half"), exact) <= tol


@pytest.mark.parametrize("shape", [(1, 2600, 2700), (1, 2700, 2600)])
def test_large_update(shape):
    param = _input(1, shape, torch.bfloat16, 0.02)
    grad, momentum = _input(2, shape, torch.bfloat16, 1e-3), _input(3, shape, torch.float32, 1e-3)
    p64, g64 = param.double(), grad.double()
    muon_update_(param, grad, momentum, lr=0.05, beta=0.9, nesterov=True, weight_decay=0.1)
    o, tol = _tolerance(0.9 * momentum.double() + 0.1 * g64, torch.float32, True)
    rate = 0.05 * math.sqrt(max(1.0, shape[-2] / shape[-1]))
    want = (1 - 0.05 * 0.1) * p64 - rate * o
    off = (param.double() - want).norm()
    assert off <= (2.0 ** -8 + 3 * 2.0 ** -24) * want.norm() + rate * tol * o.norm()


def test_status_word_is_clear():
    import ctypes
    assert _lib.load().chol_status_check(
        ctypes.c_void_p(_lib.current_queue(torch.device(DEV)))) == _lib.CHOL_OK
