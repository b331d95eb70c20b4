"""Torch tensors whose values are not what their memory holds: lazily negated
views (the imaginary part of a conjugate)."""

import pytest
import torch

import mlx_addons_b200.linalg as la

DEV = "cuda:0"


def _negated(*shape, seed=0, device="cpu"):
    """A float32 tensor with is_neg() set and the plain tensor of the same values."""
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(*shape, dtype=torch.complex64, generator=g).to(device)
    v = z.conj().imag
    assert v.is_neg()
    return v, -z.imag.clone()


@pytest.fixture
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def test_inputs_are_resolved():
    for make in (lambda: _negated(3, 4)[0], lambda: torch._neg_view(torch.ones(3, 4))):
        assert not la._as_tensor(make(), "x")[0].is_neg()
        assert not la._gemm._native(make(), "A", "x")[0].is_neg()
    t = torch.ones(2, 2)
    assert la._as_tensor(t, "x")[0] is t  # nothing is copied otherwise


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [(3, 40, 24), (70, 128, 96), (300, 256, 200)])
def test_products_of_negated_views(gpu, M, K, N):
    (A, a), (B, b), (R, r), (c, d) = (_negated(*s, seed=i, device=DEV) for i, s in enumerate([(M, K), (K, N), (M, N), (N,)]))
    assert torch.equal(la.gemm(A, B, c, "gelu", R), la.gemm(a, b, d, "gelu", r))
    assert torch.equal(la.gemm(A, b), la.gemm(a, b)) and torch.equal(la.gemm(a, B), la.gemm(a, b))
    got = la.gemm_grad(R, A, B, R, "silu", need_bias=True, need_residual=True)
    want = la.gemm_grad(r, a, b, r, "silu", need_bias=True, need_residual=True)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(24, 16), (3, 64, 64), (140, 200)])
def test_orthogonalisation_of_a_negated_view(gpu, shape):
    G, g = _negated(*shape, device=DEV)
    assert torch.equal(la.orthogonalize(G), la.orthogonalize(g))


@pytest.mark.gpu
def test_factorisations_of_negated_views(gpu):
    g = torch.Generator(device=DEV).manual_seed(0)
    L = torch.randn(4, 8, 8, generator=g, device=DEV)
    A = L @ L.mT + 8 * torch.eye(8, device=DEV)
    b = torch.randn(4, 8, 1, generator=g, device=DEV)
    An, bn = torch._neg_view(-A), torch._neg_view(-b)  # contiguous, so no copy resolves them
    assert An.is_neg() and bn.is_contiguous()
    assert torch.equal(la.solve(An, bn), la.solve(A, b)) and torch.equal(la.solve_lu(An, bn), la.solve_lu(A, b))
    assert torch.equal(la.cholesky(An), la.cholesky(A)) and torch.equal(la.logdet_spd(An), la.logdet_spd(A))
    assert torch.equal(la.qr(An)[1], la.qr(A)[1]) and torch.equal(la.slogdet(An)[0], la.slogdet(A)[0])
