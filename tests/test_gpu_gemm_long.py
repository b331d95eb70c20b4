"""16-bit products over very long sums of one sign.

The tensor cores cut what they add to an accumulator off towards zero, so a
long sum of positive terms comes out too small by as much as its accumulator
has seen additions. An accumulator that is joined in float32 after 128
additions of 16 products, each cut to the accumulator's last place (17 values of
2^-24 of it at the most), loses up to 128 * 17 * 2^-24 of the sum; the joins,
one for each 2048 terms, round to nearest: up to 2^-24 each. Positive terms
make those relative bounds of every output. The outputs of such sums lie closer together
than a 16-bit step, so their roundings hide a bias instead of averaging out: a residual
takes the rounded value away before the output is rounded, which leaves the
error itself, to half a step of its own."""

import ctypes
import math

import pytest
import torch

import mlx_addons_b200.linalg as la
from mlx_addons_b200 import _lib
from tests._exact import ACTS, HALF, MUON, check, gemm64, orth64, orth_bound

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")


def _positive(gen, *shape, dtype):
    """Uniform in [0.5, 1.5)."""
    return torch.rand(*shape, generator=gen, device=DEV).add_(0.5).to(dtype)


def _bound(K):
    return (128 * 17 + K / 2048 + 16) * 2.0**-24


def _check(out, ref, K):
    half = HALF[out.dtype]
    rel = (out.double() / ref - 1).abs()
    assert float(rel.max()) <= half + _bound(K) + half * _bound(K), (float(rel.max()), _bound(K))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("M,K,N", [(16, 1 << 20, 256), (160, 1 << 20, 96), (2048, 1 << 17, 2304), (9, 300001, 1000)])
def test_products(M, K, N, dtype):
    g = torch.Generator(device=DEV).manual_seed(M)
    A, B = _positive(g, M, K, dtype=dtype), _positive(g, K, N, dtype=dtype)
    alpha = 2.0 ** -round(math.log2(K))
    pick = torch.arange(0, M, max(1, M // 8), device=DEV)
    ref = alpha * torch.matmul(A[pick].double(), B.double())
    R = torch.zeros(M, N, device=DEV, dtype=dtype)
    R[pick] = -ref.to(dtype)
    left = ref + R[pick].double()
    half = HALF[dtype]
    for out in (la.gemm(A, B, alpha=alpha, residual=R), la.gemm(B.mT, A.mT, alpha=alpha, residual=R.mT).mT):
        err = (out[pick].double() - left).abs()
        # the error of the sum, the output's own rounding (a float16 one may be subnormal), the epilogue's two
        over = err - _bound(K) * ref - half * (left.abs() + _bound(K) * ref) - 2.0**-25 - 2.0**-23 * ref
        assert float(over.max()) <= 0, (float((err / ref).max()), float(((out[pick].double() - left) / ref).mean()), _bound(K))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_gradient_of_shared_weights(dtype):
    """dB sums over all leading dimensions and dA over the columns; without an activation dP is dY itself."""
    g = torch.Generator(device=DEV).manual_seed(3)
    A, dY, B = (_positive(g, *s, dtype=dtype) for s in [(64, 16384, 64), (64, 16384, 96), (64, 96)])
    K = 64 * 16384
    _, dB, _, _ = la.gemm_grad(dY, A, B, alpha=1 / K)
    ref = torch.zeros(64, 96, dtype=torch.float64, device=DEV)
    for a, d in zip(A, dY):
        ref += a.double().mT @ d.double()
    _check(dB, ref / K, K)
    A, dY, B = (_positive(g, *s, dtype=dtype) for s in [(128, 64), (128, 1 << 18), (64, 1 << 18)])
    dA, _, _, _ = la.gemm_grad(dY, A, B, alpha=2.0**-18)
    _check(dA, 2.0**-18 * torch.matmul(dY.double(), B.double().mT), 1 << 18)


def test_orthogonalisation_of_a_very_long_side():
    """bfloat16 rows of 2^20 values: the squares on S's diagonal are sums of one sign.

    One step with P = S makes X' = S X. The diagonal of S is held in 32 bits, its other elements (1 / sqrt(n) = 2^-10
    of the diagonal) to 2^-12 of themselves, which moves the projection on the true result by less than 2^-18 of it; the
    roundings of the result, whose values spread over several of its steps, average out. What stays is S's own bias."""
    g = torch.Generator(device=DEV).manual_seed(4)
    m, n = 192, 1 << 20
    G = torch.randint(0, 2, (m, n), generator=g, device=DEV).mul_(2).sub_(1).to(BF16)
    got = la.orthogonalize(G, steps=1, coefficients=(0.0, 1.0, 0.0), eps=0.0)
    X = G.double() / math.sqrt(m * n)
    ref = (X @ X.mT) @ X
    mean = float((got.double() * ref).sum() / (ref * ref).sum() - 1)
    assert abs(mean) <= (128 * 17 + n / 2048 + 16) * 2.0**-24 + 2.0**-16, mean


@pytest.mark.parametrize("shape", [(300, 40000), (1000, 20000), (20000, 1000), (2, 260, 70001), (140, 300000)])
def test_orthogonalisations_of_long_sides(shape):
    """bfloat16, all steps, within the bound of their factors and sums, and the same bits again."""
    g = torch.Generator(device=DEV).manual_seed(shape[-1])
    G = torch.randn(*shape, generator=g, device=DEV).add_(0.3).to(BF16)  # with a mean, so that sums of one sign are among S
    out = la.orthogonalize(G)
    ref, its = orth64(G)
    flat = lambda t: t.reshape((-1,) + tuple(t.shape[-2:]))  # noqa: E731
    err = torch.linalg.matrix_norm(flat(out.double() - ref))
    bound = orth_bound([flat(x) for x in its], 5, MUON, 2.0**-12, BF16)
    assert bool((err <= bound).all()), (err.tolist(), bound.tolist())
    assert torch.equal(la.orthogonalize(G), out)


@pytest.mark.parametrize("M,K,N", [(300, 40000, 200), (40, 70000, 1000), (2048, 10000, 2304)])
def test_a_wait_that_runs_out(monkeypatch, M, K, N):
    """B2C_GEMM_INJECT_TIMEOUT=1 in the joined form: NaN for what is lost, the device flag, and a normal next call."""
    def fault():
        f = ctypes.c_uint(7)
        assert _lib.load().b2c_take_device_fault(ctypes.byref(f)) == 0
        return f.value

    g = torch.Generator(device=DEV).manual_seed(M)
    A, B = _positive(g, M, K, dtype=BF16), _positive(g, K, N, dtype=BF16)
    fault()
    want = la.gemm(A, B)
    torch.cuda.synchronize()
    assert fault() == 0
    monkeypatch.setenv("B2C_GEMM_INJECT_TIMEOUT", "1")
    bad = la.gemm(A, B)
    torch.cuda.synchronize()
    monkeypatch.delenv("B2C_GEMM_INJECT_TIMEOUT")
    assert fault() != 0 and fault() == 0
    lost = torch.isnan(bad)
    assert bool(lost.any()) and torch.equal(bad[~lost], want[~lost])
    assert torch.equal(la.gemm(A, B), want) and fault() == 0


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("M,K,N", [(300, 33001, 200), (20, 66000, 264), (1700, 8328, 1608), (1601, 8300, 1793), (2304, 16384, 2048)])
def test_epilogues_of_long_sums(M, K, N, dtype):
    """The joined forms with every part of the epilogue, in all orders of the operands, ragged and not."""
    g = torch.Generator(device=DEV).manual_seed(K)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    bias, R = rand(N).to(dtype), rand(M, N).to(dtype)
    for i, (ta, tb) in enumerate([(False, True), (True, False), (False, False), (True, True)]):
        A = rand(K, M).to(dtype).mT if ta else rand(M, K).to(dtype)
        B = (rand(N, K) / math.sqrt(K)).to(dtype).mT if tb else (rand(K, N) / math.sqrt(K)).to(dtype)
        act = ACTS[1 + i]
        Y, pre = la.gemm(A, B, bias, act, R, alpha=0.75, beta=-1.5, return_pre=True)
        y, p, ey, ep = gemm64(A, B, bias, act, R, 0.75, -1.5)
        check(pre, p, ep, "pre", K)
        check(Y, y, ey, "Y", K)
        assert torch.equal(la.gemm(A, B, bias, act, R, alpha=0.75, beta=-1.5), Y)
    A, B = rand(3, 140, 33000).to(dtype), (rand(3, 33000, 150) / 180).to(dtype)
    y, _, ey, _ = gemm64(A, B)
    check(la.gemm(A, B), y, ey, "batch", 33000)
