"""Refusals of the products and the orthogonalisation: no GPU is needed to be
told that a call is wrong."""

import ctypes

import numpy as np
import pytest
import torch

import mlx_addons_b200.linalg as la
from mlx_addons_b200 import _lib

f = lambda *s: np.zeros(s, np.float32)  # noqa: E731
t = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype)  # noqa: E731


@pytest.mark.parametrize("args,kw", [
    ((f(3), f(3, 2)), {}),
    ((f(2, 3), f(3)), {}),
    ((f(2, 3), f(4, 2)), {}),
    ((f(2, 2, 3), f(3, 3, 2)), {}),
    ((f(2, 3), f(5, 3, 2)), {}),
    ((f(2, 3), f(3, 2)), {"activation": "tanh"}),
    ((f(2, 3), f(3, 2), f(3)), {}),
    ((f(2, 3), f(3, 2), f(2, 2)), {}),
    ((f(2, 3), f(3, 2)), {"residual": f(2, 3)}),
    ((f(4, 2, 3), f(3, 2)), {"residual": f(2, 2)}),
    ((t(2, 3, dtype=torch.bfloat16), t(3, 2)), {}),
    ((t(2, 3), t(3, 2), t(2, dtype=torch.float16)), {}),
    ((t(2, 3), t(3, 2)), {"residual": t(2, 2, dtype=torch.bfloat16)}),
    ((t(2, 3, dtype=torch.complex64), t(3, 2)), {}),
])
def test_gemm_refuses(args, kw):
    with pytest.raises(ValueError, match="gemm"):
        la.gemm(*args, **kw)


@pytest.mark.parametrize("args,kw", [
    ((f(2, 3), f(2, 3), f(3, 2)), {}),
    ((f(2, 2), f(2, 3), f(4, 2)), {}),
    ((f(2, 2), f(2, 3), f(3, 2)), {"activation": "gelu"}),
    ((f(2, 2), f(2, 3), f(3, 2)), {"activation": "gelu", "pre": f(2, 3)}),
    ((f(2, 2), f(2, 3), f(3, 2)), {"activation": "nothing"}),
    ((t(2, 2, dtype=torch.float16), t(2, 3), t(3, 2)), {}),
])
def test_gemm_grad_refuses(args, kw):
    with pytest.raises(ValueError, match="gemm_grad"):
        la.gemm_grad(*args, **kw)


@pytest.mark.parametrize("args,kw", [
    ((f(3),), {}),
    ((f(3, 3),), {"steps": 0}),
    ((f(3, 3),), {"steps": 65}),
    ((f(3, 3),), {"steps": 2.5}),
    ((f(3, 3),), {"steps": True}),
    ((f(3, 3),), {"coefficients": (1.0, 2.0)}),
    ((f(3, 3),), {"coefficients": 3.0}),
    ((f(3, 3),), {"steps": 3, "coefficients": [(1.5, -0.5, 0.0)] * 2}),
])
def test_orthogonalize_refuses(args, kw):
    with pytest.raises(ValueError, match="orthogonalize"):
        la.orthogonalize(*args, **kw)


def test_inputs_that_want_a_gradient_are_refused():
    w = torch.zeros(3, 2, requires_grad=True)
    for call in (lambda: la.gemm(f(2, 3), w), lambda: la.gemm_grad(f(2, 2), f(2, 3), w), lambda: la.orthogonalize(w)):
        with pytest.raises(ValueError, match="gradient"):
            call()


def test_lists_are_refused():
    with pytest.raises(TypeError):
        la.gemm([[1.0]], [[1.0]])
    with pytest.raises(TypeError):
        la.orthogonalize([[1.0]])


@pytest.fixture(scope="module")
def lib():
    from mlx_addons_b200 import _build
    _build.build()
    return _lib.load()


def _m(ptr=None, *s):
    return ctypes.byref(_lib.Matrix(ptr, *(s or (0, 1, 1))))


def test_c_gemm_refuses_before_any_cuda_call(lib):
    bad, uns = _lib.B2C_ERR_INVALID_ARGUMENT, _lib.B2C_ERR_UNSUPPORTED

    def call(dtype=0, A=_m(), B=_m(), R=None, Y=None, batch=1, M=2, K=2, N=2, act=0):
        return lib.b2c_gemm(dtype, A, B, None, R, Y, None, batch, M, K, N, 1.0, 1.0, act, None, 0, None)

    assert call(dtype=3) == bad and call(dtype=-1) == bad
    assert call(act=5) == bad and call(act=-1) == bad
    assert call(batch=-1) == bad and call(M=-1) == bad and call(K=-1) == bad and call(N=-1) == bad
    assert call(M=1 << 31) == uns and call(N=1 << 31) == uns and call(K=1 << 31) == uns
    assert call(A=None) == bad and call(B=None) == bad
    assert call(A=_m(16, 0, -1, 1), B=_m(16), Y=16) == bad
    assert call(R=_m(None)) == bad
    assert call() == bad and b"b2c_gemm" in lib.b2c_last_error()
    assert call(M=0) == _lib.B2C_OK and call(batch=0) == _lib.B2C_OK and lib.b2c_last_error() == b""


def test_c_dact_refuses(lib):
    bad = _lib.B2C_ERR_INVALID_ARGUMENT

    def call(dtype=0, dY=_m(16), pre=None, act=0, dP=16, db=None, batch=1, M=2, N=2, ws=None, n=0):
        return lib.b2c_gemm_dact(dtype, dY, pre, act, 1.0, dP, db, None, batch, M, N, ws, n, None)

    assert call(dtype=9) == bad and call(act=7) == bad and call(M=-1) == bad
    assert call(act=2) == bad and call(dY=None) == bad and call(dY=_m(None)) == bad
    assert call(dY=_m(16, 0, 1, -1)) == bad
    assert call(db=16) == _lib.B2C_ERR_WORKSPACE
    assert lib.b2c_gemm_dact_workspace_size(1, 2, 2) > 0
    assert call(N=0) == _lib.B2C_OK and call(dP=None) == _lib.B2C_OK and call(M=0) == _lib.B2C_OK


def test_c_orthogonalize_refuses(lib):
    bad = _lib.B2C_ERR_INVALID_ARGUMENT
    muon = (ctypes.c_double * 3)(3.4445, -4.775, 2.0315)

    def call(dtype=0, G=_m(16), out=16, batch=1, m=4, n=4, coef=muon, steps=1, eps=1e-7, ws=None, nb=0):
        return lib.b2c_orthogonalize(dtype, G, out, batch, m, n, coef, steps, eps, ws, nb, None)

    assert call(dtype=3) == bad and call(m=-1) == bad and call(batch=-1) == bad
    assert call(m=1 << 21) == _lib.B2C_ERR_UNSUPPORTED
    assert call(steps=0) == bad and call(steps=65) == bad and call(coef=None) == bad
    assert call(eps=-1.0) == bad and call(eps=float("nan")) == bad and call(eps=float("inf")) == bad
    assert call(G=None) == bad and call(G=_m(None)) == bad and call(out=None) == bad
    assert call(G=_m(16, 0, -4, 1)) == bad
    three = ctypes.c_double * 3
    assert call(coef=three(float("nan"), 0, 0)) == bad and call(coef=three(float("inf"), 0, 0)) == bad
    assert call(coef=three(4.0, 0.0, 0.0)) == bad  # singular values up to 4
    assert b"3.5" in lib.b2c_last_error()
    assert call(coef=three(9.0, -6.0, 0.0)) == bad  # 4.24 inside [0, 1], 3 at its end
    assert call(coef=three(1.5, -0.5, 0.0), m=256, n=256) == _lib.B2C_ERR_WORKSPACE  # fine; and no scratch was given
    assert call(m=0) == _lib.B2C_OK and call(batch=0) == _lib.B2C_OK


def test_dual_numbers_are_refused():
    """A tangent of forward-mode differentiation would be lost like a gradient."""
    fwad = torch.autograd.forward_ad
    with fwad.dual_level():
        w = fwad.make_dual(torch.zeros(3, 2), torch.ones(3, 2))
        for call in (lambda: la.gemm(f(2, 3), w), lambda: la.gemm(t(2, 3), t(3, 2), residual=w[:2]),
                     lambda: la.gemm_grad(f(2, 2), f(2, 3), w), lambda: la.orthogonalize(w)):
            with pytest.raises(ValueError, match="gradient"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="gradient"):
                call()


def test_c_entries_refuse_misaligned_addresses(lib):
    """An address that is not a multiple of its element's size, or scratch that is not on 16 bytes, would fault the GPU."""
    bad, ws = _lib.B2C_ERR_INVALID_ARGUMENT, _lib.B2C_ERR_WORKSPACE
    muon = (ctypes.c_double * 3)(3.4445, -4.775, 2.0315)

    def gemm(dtype, A=16, B=16, bias=None, R=None, Y=16, pre=None):
        return lib.b2c_gemm(dtype, _m(A, 0, 2, 1), _m(B, 0, 2, 1), bias, None if R is None else _m(R, 0, 2, 1), Y, pre, 1, 2, 2, 2,
                            1.0, 1.0, 0, None, 0, None)

    def dact(dtype, dY=16, pre=16, dP=16, db=None, dR=None, w=16, n=1 << 20):
        return lib.b2c_gemm_dact(dtype, _m(dY, 0, 2, 1), _m(pre, 0, 2, 1), 2, 1.0, dP, db, dR, 1, 2, 2, w, n, None)

    def orth(dtype, G=16, out=16, w=16, m=4):
        return lib.b2c_orthogonalize(dtype, _m(G, 0, m, 1), out, 1, m, m, muon, 1, 1e-7, w, 1 << 30, None)

    for dtype, off in ((0, 17), (0, 18), (1, 17), (2, 17)):
        for call, names in ((gemm, ("A", "B", "bias", "R", "Y", "pre")), (dact, ("dY", "pre", "dP", "db", "dR")),
                            (orth, ("G", "out"))):
            for name in names:
                assert call(dtype, **{name: off}) == bad, (dtype, off, name)
                assert b"align" in lib.b2c_last_error()
    for w in (17, 20, 24):
        assert dact(0, db=16, w=w) == ws and orth(0, w=w, m=300) == ws


def test_c_workspace_size_without_addresses(lib):
    """Asked for before the operands have addresses, the size covers any that they may get."""
    for dtype in (0, 1, 2):
        for s in ((0, 1024, 1), (0, 1, 1024), (0, 1032, 1), (0, 1025, 1)):
            def size(a, b):
                return lib.b2c_gemm_workspace_size(dtype, _m(a, *s), _m(b, *s), 1, 1024, 1024, 1024)
            any_ = size(None, None)
            assert any_ == size(2 if dtype else 4, 2 if dtype else 4) > 0
            assert all(size(a, b) <= any_ for a in (None, 8, 16) for b in (None, 8, 16))


@pytest.mark.parametrize("coef", [(1e200, -2e200, 1e200), (1e39, -1e39, 0.0), (0.0, 0.0, 1e60), (1e39, 0.0, -1e39)])
def test_c_coefficients_beyond_float32(lib, coef):
    """They pass the bound at 1, where they cancel, and leave float32 in the kernels."""
    c = (ctypes.c_double * 3)(*coef)
    assert lib.b2c_orthogonalize(0, _m(16, 0, 256, 1), 16, 1, 256, 256, c, 1, 1e-7, None, 0, None) == _lib.B2C_ERR_INVALID_ARGUMENT


def test_c_coefficients_after_a_polynomial_of_zeros(lib):
    """Nothing can grow from zero, but a factor beyond float32 makes NaN of it."""
    c = (ctypes.c_double * 6)(0, 0, 0, 1e39, 0, 0)
    assert lib.b2c_orthogonalize(0, _m(16, 0, 256, 1), 16, 1, 256, 256, c, 2, 1e-7, None, 0, None) == _lib.B2C_ERR_INVALID_ARGUMENT
