"""CPU: the check for forward-mode tangents, which the wrappers make before any device call."""

import pytest
import torch
from torch.autograd import forward_ad

from linalg_kernels_b200 import orthogonal


def test_tangents_are_refused():
    x = torch.ones(3, 4)
    orthogonal._refuse_tangents("here", x, None)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(3, 4))
        orthogonal._refuse_tangents("here", x, None, dual.detach())
        for t in (dual, dual.mT, dual * 2):
            with pytest.raises(RuntimeError, match="here"):
                orthogonal._refuse_tangents("here", x, t)
            with torch.no_grad(), pytest.raises(RuntimeError):  # tangents pass no_grad
                orthogonal._refuse_tangents("here", t)
    orthogonal._refuse_tangents("here", dual)
