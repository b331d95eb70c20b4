"""float32 products of very small values: as exact as those of any others, on
every kernel that a size may choose."""

import math

import pytest
import torch

import mlx_addons_b200.linalg as la
from tests._exact import check, gemm64

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
SIZES = [(3, 300, 200), (60, 40, 70), (200, 300, 160), (1000, 260, 640), (2304, 128, 2048)]


@pytest.fixture(autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _rand(seed, *shape, scale):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV, dtype=torch.float64) * scale).float()


@pytest.mark.parametrize("M,K,N", SIZES)
@pytest.mark.parametrize("e", [-100, -110, -114, -118, -122, -125])
def test_small_times_large(M, K, N, e):
    """|x| about 2^e against 2^-e; the bounds of check() are those of a float32 sum and know nothing of the size of x."""
    A, B = _rand(M + e, M, K, scale=2.0**e), _rand(N + e, K, N, scale=2.0 ** (-e) / math.sqrt(K))
    for a, b in ((A, B), (B.mT.contiguous(), A.mT.contiguous())):
        y, _, ey, _ = gemm64(a, b)
        check(la.gemm(a, b), y, ey, "Y", K)


@pytest.mark.parametrize("M,K,N", SIZES)
def test_every_magnitude_at_once(M, K, N):
    """Columns of A from 2^-125 to 2^60, each against a row of B that brings it to the size of the others."""
    p = torch.linspace(-125, 60, K, device=DEV, dtype=torch.float64).exp2()
    A = (_rand(1, M, K, scale=1.0).double() * p).float()
    B = (_rand(2, K, N, scale=1 / math.sqrt(K)).double() / p[:, None]).float()
    y, _, ey, _ = gemm64(A, B)
    check(la.gemm(A, B), y, ey, "Y", K)


@pytest.mark.parametrize("M,K,N", SIZES)
def test_gradients_of_small_values(M, K, N):
    dY, A, B = _rand(1, M, N, scale=2.0**-118), _rand(2, M, K, scale=2.0**100), _rand(3, K, N, scale=2.0**100)
    dA, dB, _, _ = la.gemm_grad(dY, A, B)
    for got, (a, b) in ((dA, (dY, B.mT)), (dB, (A.mT, dY))):
        y, _, ey, _ = gemm64(a, b)
        check(got, y, ey, "grad", a.shape[-1])


@pytest.mark.parametrize("M,K,N", SIZES)
def test_subnormal_values(M, K, N):
    """Whole multiples of 2^-149, the smallest float32, below 2^-126."""
    g = torch.Generator(device=DEV).manual_seed(5)
    A = (torch.randint(-(1 << 22), 1 << 22, (M, K), generator=g, device=DEV).double() * 2.0**-149).float()
    B = _rand(6, K, N, scale=2.0**120)
    y, _, ey, _ = gemm64(A, B)
    check(la.gemm(A, B), y, ey, "Y", K)


@pytest.mark.parametrize("M,K,N", SIZES)
def test_the_largest_values(M, K, N):
    """float32's largest, and others whose nearest bf16 would be infinite, among ordinary ones of that size and zeros."""
    top = torch.finfo(torch.float32).max
    A, B = _rand(7, M, K, scale=2.0**125).clamp(-top, top), _rand(8, K, N, scale=2.0**-127 / math.sqrt(K))
    A[:, ::5], A[1, ::7], A[:, 3] = top, -top * (1 - 2.0**-9), 0.0
    A[2] = torch.where(torch.arange(K, device=DEV) % 2 == 0, top, -top)
    y, _, ey, _ = gemm64(A, B)
    check(la.gemm(A, B), y, ey, "Y", K)
    check(la.gemm(B.mT, A.mT), y.mT, ey.mT, "transposed", K)
