"""GPU: what orthogonalize, muon_update_, grouped_matmul and grouped_outer refuse once their arguments are
on the device."""

import pytest
import torch
from torch.autograd import forward_ad

from linalg_kernels_b200.grouped import grouped_matmul, grouped_outer
from linalg_kernels_b200.orthogonal import muon_update_, orthogonalize

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _ones(*shape, dtype=torch.bfloat16):
    return torch.ones(*shape, device=DEV, dtype=dtype)


def test_forward_mode_tangents():
    """A result without its tangent would read as a zero derivative."""
    x, w, dy = _ones(6, 8), _ones(2, 8, 16), _ones(6, 16)
    offsets = torch.tensor([0, 2, 6], device=DEV)
    orthogonalize(x)
    for _ in range(2):
        with forward_ad.dual_level():
            def dual(t):
                return forward_ad.make_dual(t, torch.ones_like(t))

            for call in (lambda: grouped_matmul(dual(x), w, offsets),
                         lambda: grouped_matmul(x, dual(w), offsets),
                         lambda: grouped_matmul(x, dual(w).mT.contiguous().mT, offsets),
                         lambda: grouped_matmul(dual(x), w, offsets, out=_ones(6, 16)),
                         lambda: grouped_outer(dual(x), dy, offsets),
                         lambda: grouped_outer(x, dual(dy), offsets),
                         lambda: orthogonalize(dual(x)),
                         lambda: orthogonalize(dual(x), out=_ones(6, 8)),
                         lambda: muon_update_(dual(_ones(6, 8)), _ones(6, 8), _ones(6, 8), lr=0.1),
                         lambda: muon_update_(_ones(6, 8), dual(_ones(6, 8)), _ones(6, 8), lr=0.1),
                         lambda: muon_update_(_ones(6, 8), _ones(6, 8), dual(_ones(6, 8)), lr=0.1)):
                for mode in (torch.enable_grad, torch.no_grad):
                    with mode(), pytest.raises(RuntimeError, match="forward-mode"):
                        call()
            # without a tangent, the same as outside
            assert torch.equal(orthogonalize(x), orthogonalize(dual(x).detach()))
            grouped_matmul(x, w, offsets)
    x.requires_grad_()
    grouped_matmul(x, w, offsets).sum().backward()
    assert x.grad is not None


def test_iteration_arguments_every_time():
    """The second call takes the short host path: it refuses the same."""
    x = _ones(3, 8, 8)
    for _ in range(2):
        orthogonalize(x, 5)
        orthogonalize(x, 1)
        for steps in (5.0, 0, 33, "5", None, 1.0):
            with pytest.raises(ValueError, match="steps"):
                orthogonalize(x, steps)
        for coefs in ((1.0, 2.0), (), None, 5, ((1.0, 2.0, 3.0),) * 3, (float("inf"), 0.0, 0.0)):
            with pytest.raises(ValueError, match="coefficients"):
                orthogonalize(x, 5, coefficients=coefs)
        with pytest.raises(ValueError, match="precision"):
            orthogonalize(x, precision="double")


def test_orthogonalize_tensors():
    x = _ones(3, 8, 12)
    for t in (x.to(torch.float64), x.int(), x.cfloat()):
        with pytest.raises(TypeError):
            orthogonalize(t)
    with pytest.raises(ValueError):
        orthogonalize(x[0, 0])
    with pytest.raises(TypeError):
        orthogonalize(x, out=torch.empty(3, 8, 12, dtype=torch.bfloat16))
    for out in (_ones(3, 8, 13), _ones(3, 12, 8), _ones(2, 8, 12), _ones(3, 8, 12, dtype=torch.float32)):
        with pytest.raises(ValueError, match="shape, type"):
            orthogonalize(x, out=out)
    for out in (_ones(1, 8, 12).expand(3, 8, 12), _ones(3, 8, 24)[..., ::2], _ones(3, 1, 12).expand(3, 8, 12),
                _ones(3, 8, 1).expand(3, 8, 12)):
        with pytest.raises(ValueError, match="contiguous"):
            orthogonalize(x, out=out)
    for grad in (x.clone().requires_grad_(), torch.nn.Parameter(x.clone())):
        with pytest.raises(RuntimeError, match="derivative"):
            orthogonalize(grad)
        with pytest.raises(RuntimeError, match="derivative"):
            orthogonalize(x, out=grad)
        with torch.no_grad():
            assert torch.equal(orthogonalize(grad), orthogonalize(x))


def test_muon_tensors():
    p, g, m = _ones(2, 8, 12), _ones(2, 8, 12), _ones(2, 8, 12, dtype=torch.float32)
    kept = [t.clone() for t in (p, g, m)]

    def refused(error, match, *tensors, **kw):
        with pytest.raises(error, match=match):
            muon_update_(*tensors, **{"lr": 0.1, **kw})

    refused(TypeError, "grad", p, g.double(), m)
    refused(TypeError, "momentum", p, g, m.cpu())
    refused(ValueError, "one shape", p, g[:1], m)
    refused(ValueError, "one shape", p, g, m.mT.contiguous())
    refused(ValueError, "columns", p, g, m.mT.contiguous().mT)  # rows and columns
    refused(ValueError, "columns", p.mT.contiguous().mT, g, m)
    refused(ValueError, "columns", p[:1].expand(2, 8, 12), g, m)
    refused(ValueError, "overlap", p, p, m)
    refused(ValueError, "overlap", p, g, p)
    refused(ValueError, "overlap", p, g, g)
    refused(ValueError, "overlap", m, p, m)
    wide = _ones(3, 8, 12)
    refused(ValueError, "overlap", wide[:2], wide[1:], m)
    refused(RuntimeError, "param", p.clone().requires_grad_(), g, m)
    refused(RuntimeError, "momentum", p, g, m.clone().requires_grad_())
    for name in ("lr", "beta", "weight_decay", "scale"):
        for bad in (float("nan"), float("inf")):
            refused(ValueError, name, p, g, m, **{name: bad})
    refused(ValueError, "steps", p, g, m, steps=0)
    refused(ValueError, "eps", p, g, m, eps=-1.0)
    refused(ValueError, "precision", p, g, m, precision="best")
    for t, k in zip((p, g, m), kept):
        assert torch.equal(t, k)
    # a gradient that requires grad is read alone; parameters under no_grad are written
    param = torch.nn.Parameter(p.clone())
    with torch.no_grad():
        muon_update_(param, g, m.clone(), lr=0.1)
    muon_update_(p, g.clone().requires_grad_(), m, lr=0.1)
    assert torch.equal(param.detach(), p)


def test_grouped_tensors():
    x, w, dy = _ones(6, 8), _ones(2, 8, 16), _ones(6, 16)
    offsets = torch.tensor([0, 2, 6], device=DEV)

    def refused(error, match, call, *args, **kw):
        with pytest.raises(error, match=match):
            call(*args, **kw)

    for call, a, b in ((grouped_matmul, x, w), (grouped_outer, x, dy)):
        refused(TypeError, "float16", call, a.float(), b.float(), offsets)
        refused(ValueError, "type", call, a, b.half(), offsets)
        refused(TypeError, "CUDA", call, a, b.cpu(), offsets)
        refused(ValueError, "dimensions", call, a[None], b, offsets)
        refused(ValueError, "dimensions", call, a, b[None], offsets)
        refused(TypeError, "offsets", call, a, b, [0, 2, 6])
        refused(TypeError, "offsets", call, a, b, offsets.float())
        refused(TypeError, "offsets", call, a, b, offsets.short())
        refused(ValueError, "device", call, a, b, offsets.cpu())
        refused(ValueError, "contiguous", call, a, b, offsets[None])
        refused(ValueError, "contiguous", call, a, b, offsets.repeat_interleave(2)[::2])
        refused(ValueError, "contiguous", call, a, b, offsets[:0])
    refused(ValueError, "3 entries", grouped_matmul, x, w, offsets[:2])
    refused(ValueError, "w must be", grouped_matmul, x, w.mT, offsets)
    refused(ValueError, "same rows", grouped_outer, x, dy[:5], offsets)
    many = torch.zeros(1026, device=DEV, dtype=torch.int32)
    refused(ValueError, "1024", grouped_matmul, x, w[:1].expand(1025, 8, 16), many)
    refused(ValueError, "1024", grouped_outer, x, dy, many)
    for out in (_ones(6, 17), _ones(7, 16), _ones(16, 6)):
        refused(ValueError, "shape", grouped_matmul, x, w, offsets, out=out)
    refused(ValueError, "type", grouped_matmul, x, w, offsets, out=_ones(6, 16, dtype=torch.float16))
    refused(ValueError, "dimensions", grouped_matmul, x, w, offsets, out=_ones(1, 6, 16))
    refused(ValueError, "rows", grouped_matmul, x, w, offsets, out=_ones(16, 6).T)
    refused(ValueError, "rows", grouped_matmul, x, w, offsets, out=_ones(1, 16).expand(6, 16))
    refused(ValueError, "rows", grouped_outer, x, dy, offsets, out=_ones(1, 8, 16).expand(2, 8, 16))
    square = _ones(2, 6, 6)
    refused(ValueError, "overlap", grouped_matmul, square[0], square, offsets, out=square[0])
    refused(ValueError, "overlap", grouped_matmul, square[0].clone(), square, offsets, out=square[1])
    big = _ones(40, 8)
    refused(ValueError, "overlap", grouped_outer, big[:6], big[6:12], offsets,
            out=big.view(-1)[64:192].view(2, 8, 8))
    refused(ValueError, "k > 0", grouped_matmul, x[:, :0], w[:, :0], offsets, out=_ones(6, 16))
    for a, b in ((x.clone().requires_grad_(), w), (x, w.clone().requires_grad_())):
        refused(RuntimeError, "no_grad", grouped_matmul, a, b, offsets, out=_ones(6, 16))
        with torch.no_grad():
            grouped_matmul(a, b, offsets, out=_ones(6, 16))
    refused(RuntimeError, "no_grad", grouped_matmul, x, w, offsets, out=_ones(6, 16).requires_grad_())
    refused(RuntimeError, "no_grad", grouped_outer, x.clone().requires_grad_(), dy, offsets)
    refused(RuntimeError, "no_grad", grouped_outer, x, dy, offsets, out=_ones(2, 8, 16).requires_grad_())
    # operands changed between the passes
    xx, ww = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = grouped_matmul(xx, ww, offsets)
    with torch.no_grad():
        ww.mul_(2)
    refused(RuntimeError, "modified", y.sum().backward)
    y = grouped_matmul(xx, ww, offsets)
    with torch.no_grad():
        muon_update_(ww, _ones(2, 8, 16), _ones(2, 8, 16), lr=0.1)
    refused(RuntimeError, "modified", y.sum().backward)


@pytest.mark.parametrize("precision", ["half", "full"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_muon_precision_argument(precision, dtype):
    from tests.test_orthogonal_gpu import _input, _tolerance

    for shape in ((2, 96, 200), (2, 300, 260)):
        grad, momentum = _input(1, shape), torch.zeros(shape, device=DEV)
        param = torch.zeros(shape, device=DEV, dtype=dtype)
        muon_update_(param, grad, momentum, lr=1.0, beta=0.0, nesterov=False, scale=1.0,
                     precision=precision)
        exact, tol = _tolerance(grad, dtype, precision == "half")
        off = (param.double() + exact).square().sum((-2, -1)).sqrt()
        assert (off <= (tol + 3 * 2.0 ** -24) * exact.square().sum((-2, -1)).sqrt()).all()


def test_lazy_negations():
    """The imaginary part of a conjugate is a view whose sign is not in memory: inputs are resolved, results
    refused."""
    g = torch.Generator(device=DEV).manual_seed(1)
    z = torch.randn(2, 40, 1, dtype=torch.complex64, device=DEV, generator=g)
    v = z.conj().imag
    assert v.is_neg()
    for _ in range(2):
        assert torch.equal(orthogonalize(v), orthogonalize(-z.imag))
        t = torch._neg_view(_ones(2, 8, 12))
        assert torch.equal(orthogonalize(t), -orthogonalize(_ones(2, 8, 12)))
    p, m = _ones(2, 8, 12), _ones(2, 8, 12)
    q, n = p.clone(), m.clone()
    muon_update_(p, torch._neg_view(_ones(2, 8, 12)), m, lr=0.1)
    muon_update_(q, -_ones(2, 8, 12), n, lr=0.1)
    assert torch.equal(p, q) and torch.equal(m, n)
    x, w, dy = _ones(6, 8), _ones(2, 8, 16), _ones(6, 16)
    offsets = torch.tensor([0, 2, 6], device=DEV)
    neg = torch._neg_view
    y = grouped_matmul(x, w, offsets)
    for a, b in ((neg(x), w), (x, neg(w)), (x, neg(w.mT.contiguous()).mT), (neg(x)[:, ::1], w)):
        assert torch.equal(grouped_matmul(a, b, offsets), -y)
    dw = grouped_outer(x, dy, offsets)
    assert torch.equal(grouped_outer(neg(x), dy, offsets), -dw)
    xx, ww = x.clone().requires_grad_(), w.clone().requires_grad_()
    for d in torch.autograd.grad(grouped_matmul(xx, ww, offsets), (xx, ww), neg(dy)):
        assert (d < 0).all()
    for call in (lambda: orthogonalize(p, out=neg(q)), lambda: muon_update_(neg(p), q, n, lr=0.1),
                 lambda: muon_update_(p, q, neg(n), lr=0.1),
                 lambda: grouped_matmul(x, w, offsets, out=neg(dy)),
                 lambda: grouped_outer(x, dy, offsets, out=neg(_ones(2, 8, 16)))):
        with pytest.raises(ValueError, match="negation"):
            call()
