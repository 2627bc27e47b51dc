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
