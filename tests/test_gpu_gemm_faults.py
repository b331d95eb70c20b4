"""Waits of the tensor-core products and of the orthogonalisation that run out.

B2C_GEMM_INJECT_TIMEOUT=1 (read per call) makes CTA 0's epilogue wait for an
mbarrier that nothing arrives on and limits every wait to 1 ms: the kernel must
end by itself, report through b2c_take_device_fault, and leave NaN for what it
did not compute; the next call runs normally."""

import ctypes

import pytest
import torch

import mlx_addons_b200.linalg as la
from mlx_addons_b200 import _lib

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _fault():
    f = ctypes.c_uint(7)
    assert _lib.load().b2c_take_device_fault(ctypes.byref(f)) == 0
    return f.value


def _run(monkeypatch, call):
    """(clean result, result with the timeout); the flag is set by the second alone."""
    _fault()
    want = call()
    torch.cuda.synchronize()
    assert _fault() == 0
    monkeypatch.setenv("B2C_GEMM_INJECT_TIMEOUT", "1")
    bad = call()
    torch.cuda.synchronize()
    monkeypatch.delenv("B2C_GEMM_INJECT_TIMEOUT")
    assert _fault() != 0 and _fault() == 0
    again = call()
    torch.cuda.synchronize()
    assert torch.equal(want, again) and _fault() == 0
    return want, bad


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,K,N", [(300, 2048, 200), (40, 2048, 1000), (2048, 512, 2048)])
def test_products(monkeypatch, M, K, N, dtype):
    g = torch.Generator(device=DEV).manual_seed(M)
    A = torch.randn(M, K, generator=g, device=DEV).to(dtype)
    B = torch.randn(K, N, generator=g, device=DEV).to(dtype)
    want, bad = _run(monkeypatch, lambda: la.gemm(A, B))
    lost = torch.isnan(bad)
    assert bool(lost.any()) and torch.equal(bad[~lost], want[~lost])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(50, 40, 64), (20, 100, 600), (2, 140, 500), (2, 300, 5000)])
def test_orthogonalisation(monkeypatch, shape, dtype):
    g = torch.Generator(device=DEV).manual_seed(3)
    G = torch.randn(*shape, generator=g, device=DEV).to(dtype)
    want, bad = _run(monkeypatch, lambda: la.orthogonalize(G))
    lost = torch.isnan(bad)
    assert bool(lost.any()) and torch.equal(bad[~lost], want[~lost])
