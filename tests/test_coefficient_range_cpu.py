"""CPU: the coefficients whose iterates could leave fp16's range are refused by the C entries' host
checks."""

import ctypes

from linalg_kernels_b200 import _lib, orthogonal
from tests.test_linalg_cpu import SPACE, TOO_BIG, _floats, _m, _orth


def test_coefficients_that_could_leave_fp16():
    """Singular values start at 1 at most: G = s^2 has 65504 / 32^2 = 63.97 (half) or 65504 / 64^2 =
    15.99 (full), B 65504 or 65504 / 2048 = 31.98."""
    def orth(coef, prec):  # (a workspace that is too small: what passes the check answers SPACE)
        return _orth(x=_m(ld=300), out=_m(1 << 20, ld=300), m=200, n=300, steps=len(coef) // 3,
                     coef=coef, prec=prec, size=100)

    one, (a, b, c) = (1.0, 0.0, 0.0), orthogonal.DEFAULT_COEFFICIENTS
    for prec in (1, 2, 0):
        assert orth((a, b, c) * 32, prec) == SPACE
        assert orth((3.0, -3.2, 1.2) * 8, prec) == SPACE
        assert orth((1.5, -0.5, 0.0) * 32, prec) == SPACE
        # a shrinks the small singular values
        assert orth((0.0, 2.0, -1.0), prec) == TOO_BIG
        assert orth((0.0, 0.0, 0.0), prec) == SPACE  # zeros, exactly
        assert orth((0.25, 1.0, 0.0), prec) == SPACE and orth((0.2, 1.0, 0.0), prec) == TOO_BIG
        assert orth((0.6, 0.0, 0.0) * 2, prec) == SPACE and orth((0.6, 0.0, 0.0) * 3, prec) == TOO_BIG
        assert orth((2.0, 0.0, 0.0, 0.2, 0.0, 0.0), prec) == SPACE
        assert orth((1e30, 0.0, 0.0) + one, prec) == TOO_BIG
        assert orth((3e38, -3e38, 3e38) * 2, prec) == TOO_BIG
    # the last step's s is not stored, the others' are
    for prec, most in ((1, 7.75), (2, 3.875)):
        assert orth((most, 0.0, 0.0) + one, prec) == SPACE
        assert orth((-most, 0.0, 0.0) + one, prec) == SPACE
        assert orth((most * 1.05, 0.0, 0.0) + one, prec) == TOO_BIG
        assert orth(one + (most * 1.05, 0.0, 0.0), prec) == SPACE
        # growth over the steps, and an extremum inside the range: t - t^5 is 0 at 0 and 1, largest
        # 0.535 between (t^4 = 1/5)
        assert orth((1.5, 0.0, 0.0) * 9, prec) == TOO_BIG
        assert orth((most * 1.8, 0.0, -most * 1.8) + one, prec) == SPACE
        assert orth((most * 2.0, 0.0, -most * 2.0) + one, prec) == TOO_BIG
        # and 3 b t^2 = -a alone: t - t^3, 0.385
        assert orth((most * 2.5, -most * 2.5, 0.0) + one, prec) == SPACE
        assert orth((most * 2.7, -most * 2.7, 0.0) + one, prec) == TOO_BIG
    assert orth((64992.0, 0.0, 0.0), 1) == SPACE and orth((65600.0, 0.0, 0.0), 1) == TOO_BIG
    assert orth((65600.0, -65600.0, 0.0), 1) == TOO_BIG  # a alone, at zero singular values
    assert orth((1.0, 31.5, 0.0), 2) == SPACE and orth((1.0, 32.1, 0.0), 2) == TOO_BIG
    assert orth((1.0, 120.0, -120.0), 2) == SPACE  # b t^2 + c t^4: 30 in between
    assert orth((1.0, 130.0, -130.0), 2) == TOO_BIG


def test_the_same_for_the_optimiser_step():
    def muon(coef, prec, kind):
        return _lib.load().linalg_muon_update(
            ctypes.byref(_m(1 << 20, ld=300, kind=kind)), ctypes.byref(_m(1 << 22, ld=300)),
            ctypes.byref(_m(1 << 24, ld=300, kind=2)), 1, 200, 300, 0.9, 1, 1.0, 0.1, len(coef) // 3,
            _floats(*coef), 0.0, prec, ctypes.c_void_p(4096), 100, None)

    wide = (6.0, 0.0, 0.0, 1.0, 0.0, 0.0)  # half's range, not full's
    assert muon(wide, 1, 2) == SPACE and muon(wide, 2, 2) == TOO_BIG
    assert muon(wide, 0, 0) == SPACE and muon(wide, 0, 2) == TOO_BIG  # by the weights' type
    assert muon((65600.0, 0.0, 0.0), 1, 0) == TOO_BIG
