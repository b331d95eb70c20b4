"""NaN and infinities among the operands give what IEEE arithmetic gives, on
every kernel that a size may choose: the product in 64 bits, where these
values do not overflow, says where NaN, inf and -inf stand."""

import pytest
import torch

import mlx_addons_b200.linalg as la

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DEV = "cuda:0"
INF, NAN = float("inf"), float("nan")


@pytest.fixture(autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _same_kind(out, ref):
    out = out.double()
    for mask in (torch.isnan, torch.isposinf, torch.isneginf):
        assert torch.equal(mask(out), mask(ref)), mask.__name__


SIZES = [(3, 300, 200), (60, 40, 70), (200, 300, 160), (1000, 260, 640), (2304, 128, 2048), (24, 2000, 3000), (700, 4096, 300)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_products(M, K, N, dtype):
    g = torch.Generator(device=DEV).manual_seed(M)
    A, B = (torch.randn(*s, generator=g, device=DEV).to(dtype) for s in ((M, K), (K, N)))
    B = B / 8
    clean = la.gemm(A, B)
    A2, B2 = A.clone(), B.clone()
    A2[0, 3], A2[1, 5], A2[1, 7], A2[M - 1, K - 1] = INF, -INF, 0.0, NAN
    A2[2, 2] = INF
    A2[2, 9] = INF  # two of one sign, or of both where B's signs differ
    rows = [0, 1, 2, M - 1]
    _same_kind(la.gemm(A2, B), torch.matmul(A2.double(), B.double()))
    keep = [r for r in range(M) if r not in rows]
    assert torch.equal(la.gemm(A2, B)[keep], clean[keep])
    # against zeros (NaN), infinities of either sign and the smallest values
    B2[3, 0], B2[3, 1], B2[3, 2], B2[3, 4], B2[3, 5] = 0.0, INF, -INF, 1.0, -1.0
    B2[7, N - 1] = INF
    B2[K - 1, N - 2] = -INF
    tiny = torch.finfo(dtype).smallest_normal
    B2[3, 6], B2[3, 7] = tiny, -tiny
    B2[3, 8], B2[3, 9] = (2.0**-149, -(2.0**-149)) if dtype == F32 else (tiny, -tiny)
    _same_kind(la.gemm(A2, B2), torch.matmul(A2.double(), B2.double()))
    _same_kind(la.gemm(B2.mT, A2.mT), torch.matmul(B2.double().mT, A2.double().mT))


@pytest.mark.parametrize("M,K,N", SIZES)
def test_gradients(M, K, N):
    g = torch.Generator(device=DEV).manual_seed(M)
    dY, A, B = (torch.randn(*s, generator=g, device=DEV) for s in ((M, N), (M, K), (K, N)))
    dY[1, 4], dY[2, 5], A[2, 3], B[1, 4] = INF, -INF, NAN, -INF
    dA, dB, _, _ = la.gemm_grad(dY, A, B)
    _same_kind(dA, torch.matmul(dY.double(), B.double().mT))
    _same_kind(dB, torch.matmul(A.double().mT, dY.double()))
