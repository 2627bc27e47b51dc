"""CPU: include/linalg_b200.h is exported and bound, and every refusal of its entry points and of
their Python wrappers that needs no GPU (host-side checks run before any device call)."""

import ctypes
import re
from pathlib import Path

import pytest
import torch

from linalg_kernels_b200 import _lib
from linalg_kernels_b200 import grouped, orthogonal

ROOT = Path(__file__).resolve().parents[1]


def _functions():
    text = (ROOT / "include" / "linalg_b200.h").read_text()
    return re.findall(r"^CHOL_API\s+[\w\s\*]+?\b(linalg_\w+)\s*\(", text, flags=re.M)


def test_library_exports_and_binding():
    lib = ctypes.CDLL(str(_lib.LIB_PATH))
    assert _functions()
    for name in _functions():
        assert hasattr(lib, name), name
    assert set(_functions()) == set(_lib.LINALG_SIGNATURES)


def test_workspace():
    f = _lib.load().linalg_orthogonalize_workspace
    assert f(0, 5, 5, 1) == 0 and f(2, 0, 5, 1) == 0 and f(2, 5, 0, 1) == 0
    assert f(5, 128, 4096, 1) == 0 and f(5, 4096, 100, 1) == 0 and f(5, 129, 256, 1) == 0
    assert f(5, 129, 257, 1) > 0 and f(5, 129, 256, 2) > 0
    assert f(5, 128, 1536, 2) == 0 and f(5, 128, 1537, 2) > 0
    # two X and two squares of fp16, twice that for full precision
    assert f(3, 512, 1024, 1) >= 3 * 2 * 2 * (512 * 1024 + 512 * 512)
    assert f(3, 512, 1024, 2) >= 2 * 3 * 2 * 2 * (512 * 1024 + 512 * 512)
    assert f(3, 512, 1024, 0) == f(3, 512, 1024, 2)


def _m(data=4096, ld=64, stride=4096, kind=0):
    return _lib.Matrix(data, ld, stride, kind)


def _floats(*v):
    return (ctypes.c_float * len(v))(*v)


def _orth(x=None, out=None, batch=1, m=64, n=64, steps=1, coef=(3.0, -3.0, 1.0), eps=0.0, prec=1,
          ws=4096, size=1 << 40):
    return _lib.load().linalg_orthogonalize(
        ctypes.byref(x or _m()), ctypes.byref(out or _m(1 << 20)), batch, m, n, steps,
        _floats(*coef) if coef else None, eps, prec, ctypes.c_void_p(ws), size, None)


BAD, SPACE, TOO_BIG = _lib.CHOL_ERR_INVALID_ARG, _lib.CHOL_ERR_WORKSPACE, _lib.CHOL_ERR_UNSUPPORTED


def test_orthogonalize_refusals_of_the_c_entry():
    assert _orth(batch=0) == _lib.CHOL_OK and _orth(m=0) == _lib.CHOL_OK
    assert _orth(batch=-1) == BAD and _orth(n=-1) == BAD
    assert _orth(steps=0) == BAD and _orth(steps=33) == BAD and _orth(coef=None) == BAD
    assert _orth(coef=(float("nan"), 0.0, 0.0)) == BAD and _orth(coef=(0.0, float("inf"), 0.0)) == BAD
    assert _orth(eps=-1.0) == BAD and _orth(eps=float("nan")) == BAD
    assert _orth(prec=3) == BAD and _orth(prec=-1) == BAD
    assert _orth(x=_m(0)) == BAD and _orth(x=_m(4097)) == BAD and _orth(x=_m(kind=3)) == BAD
    assert _orth(x=_m(ld=63)) == BAD
    assert _orth(x=_m(stride=100), batch=2) == BAD
    assert _orth(out=_m(1 << 20, stride=0), batch=2) == BAD
    assert _orth(out=_m(4096 + 128)) == BAD  # overlaps x by all but a row
    big = dict(x=_m(ld=300), out=_m(1 << 20, ld=300), m=200, n=300)  # needs a workspace
    assert _orth(**big, ws=0) == SPACE and _orth(**big, ws=4096 + 16) == SPACE
    assert _orth(**big, size=100) == SPACE
    assert _orth(x=_m(ld=1 << 25), out=_m(1 << 40, ld=1 << 25), n=1 << 25) == TOO_BIG


def _muon(param=None, grad=None, momentum=None, beta=0.9, decay=1.0, rate=0.1, batch=1, steps=1, m=64):
    return _lib.load().linalg_muon_update(
        ctypes.byref(param or _m(1 << 20)), ctypes.byref(grad or _m(1 << 22)),
        ctypes.byref(momentum or _m(1 << 24, kind=2)), batch, m, m, beta, 1, decay, rate, steps,
        _floats(3.0, -3.0, 1.0), 0.0, 1, ctypes.c_void_p(4096), 100, None)


def test_muon_refusals_of_the_c_entry():
    assert _muon(batch=0) == _lib.CHOL_OK
    assert _muon(beta=float("nan")) == BAD and _muon(decay=float("inf")) == BAD
    assert _muon(rate=float("nan")) == BAD and _muon(steps=0) == BAD
    assert _muon(momentum=_m(0)) == BAD
    assert _muon(grad=_m(1 << 20)) == BAD  # the parameter's own memory
    assert _muon(momentum=_m((1 << 22) + 64)) == BAD
    assert _muon(param=_m(1 << 20, stride=0), batch=2) == BAD
    wide = [_m(1 << k, ld=300) for k in (20, 22)]
    assert _muon(wide[0], wide[1], _m(1 << 24, ld=300, kind=2), m=300) == SPACE


def _mul(x=None, w=None, y=None, off=4096, off64=0, groups=2, rows=10, k=64, n=64, fill=1):
    return _lib.load().linalg_grouped_matmul(
        ctypes.byref(x or _m()), ctypes.byref(w or _m(1 << 20)), 1,
        ctypes.byref(y or _m(1 << 22)), ctypes.c_void_p(off), off64, groups, rows, k, n, fill, None)


def _outer(a=None, b=None, dw=None, off=4096, groups=2, rows=10, k=64, n=64):
    return _lib.load().linalg_grouped_outer(
        ctypes.byref(a or _m()), ctypes.byref(b or _m(1 << 20)), ctypes.byref(dw or _m(1 << 22)),
        ctypes.c_void_p(off), 0, groups, rows, k, n, None)


def test_grouped_refusals_of_the_c_entries():
    assert _mul(rows=0) == _lib.CHOL_OK and _mul(n=0) == _lib.CHOL_OK
    assert _mul(groups=0, fill=0) == _lib.CHOL_OK
    assert _mul(groups=-1) == BAD and _mul(rows=-1) == BAD
    assert _mul(x=_m(0)) == BAD and _mul(off=0) == BAD and _mul(off=4098) == BAD
    assert _mul(off=4100, off64=1) == BAD
    assert _mul(x=_m(kind=2)) == BAD and _mul(w=_m(1 << 20, kind=1)) == BAD
    assert _mul(x=_m(ld=56)) == BAD and _mul(y=_m(1 << 22, ld=63)) == BAD
    assert _mul(groups=1025) == TOO_BIG and _mul(rows=1 << 31) == TOO_BIG
    assert _mul(x=_m(4096 + 8)) == TOO_BIG and _mul(x=_m(ld=68)) == TOO_BIG
    assert _mul(w=_m(1 << 20, stride=4100)) == TOO_BIG
    assert _mul(w=_m(1 << 20, stride=0)) == BAD
    assert _outer(groups=0) == _lib.CHOL_OK and _outer(rows=-1) == BAD
    assert _outer(dw=_m(1 << 22, stride=64)) == BAD  # the groups' results would overlap
    assert _outer(b=_m(1 << 20, kind=1)) == BAD and _outer(a=_m(ld=68)) == TOO_BIG
    assert _outer(groups=1025) == TOO_BIG


def test_binding_checks_its_arguments():
    lib = _lib.linalg()
    with pytest.raises(TypeError):
        lib.grouped_matmul(1, 2, 3)
    with pytest.raises(TypeError):
        lib.orthogonalize(*range(16), 0.0, 5)  # not a buffer
    # a coefficient buffer shorter than the steps is refused, not read past its end
    short = bytes(4 * 3)
    x, out = (4096, 300, 4096, 0), (1 << 20, 300, 4096, 0)
    assert lib.orthogonalize(*x, *out, 1, 300, 300, 2, 1, 4096, 0, 0, 0.0, short) == BAD
    assert lib.orthogonalize(*x, *out, 1, 300, 300, 1, 1, 4096, 0, 0, 0.0, short) == SPACE


def test_wrappers_refuse_what_has_no_gpu_path():
    x = torch.zeros(4, 8, 8)
    with pytest.raises(TypeError, match="CUDA"):
        orthogonal.orthogonalize(x)
    with pytest.raises(TypeError):
        orthogonal.orthogonalize([[1.0]])
    with pytest.raises(TypeError, match="CUDA"):
        orthogonal.muon_update_(x, x, x, lr=0.1)
    h = torch.zeros(4, 8, dtype=torch.bfloat16)
    off = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(TypeError, match="CUDA"):
        grouped.grouped_matmul(h, h.expand(2, 4, 8), off)
    with pytest.raises(TypeError, match="CUDA"):
        grouped.grouped_outer(h, h, off)
    with pytest.raises(TypeError):
        grouped.grouped_outer(None, h, off)


def test_iteration_arguments():
    check = orthogonal._check_iteration
    good = orthogonal.DEFAULT_COEFFICIENTS
    assert len(check(5, good, 1e-7, None)) == 15
    assert list(check(2, [[1, 2, 3], [4, 5, 6]], 0.0, "full")) == [1, 2, 3, 4, 5, 6]
    for steps in (0, 33, 2.5, "5"):
        with pytest.raises(ValueError):
            check(steps, good, 1e-7, None)
    for coef in ((), (1.0, 2.0), ((1.0, 2.0, 3.0),) * 3, (float("nan"), 1.0, 1.0), 5, None):
        with pytest.raises(ValueError):
            check(5, coef, 1e-7, None)
    for eps in (-1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            check(5, good, eps, None)
    with pytest.raises(ValueError):
        check(5, good, 1e-7, "double")


def test_layout_rules():
    """Which strides go to the library as they are (read from CPU tensors: only strides count)."""
    rows, cols = orthogonal._is_rows, orthogonal._is_transposed
    t = torch.zeros(2, 3, 6, 10)
    assert rows(t, True) and not cols(t)
    assert rows(t[..., 1:5, 2:7], True)
    assert cols(t.mT) and rows(t.mT.mT, True) and not rows(t.mT, True)
    assert not rows(t.transpose(0, 1), True) and not rows(t[..., ::2], True)
    assert rows(t[0, 0].expand(4, 6, 10), False) and not rows(t[0, 0].expand(4, 6, 10), True)
    assert not rows(torch.zeros(6, 1).expand(6, 10), True)  # every column the same element
    assert not rows(torch.zeros(1, 10).expand(6, 10), True)
    a = grouped._aligned
    x = torch.zeros(40, 72, dtype=torch.bfloat16)
    assert a(x) is x
    odd = torch.zeros(40, 77, dtype=torch.bfloat16)
    assert a(odd).stride() == (80, 1) and a(odd).shape == odd.shape
    assert a(x[:, ::2]).stride() == (40, 1)
    assert a(x.T).stride(-1) == 1
    w = torch.zeros(3, 8, 16, dtype=torch.bfloat16)
    assert a(w) is w and a(w[:1].expand(3, 8, 16)).stride() == (128, 16, 1)
