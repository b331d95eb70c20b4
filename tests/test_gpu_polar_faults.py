"""Waits of the grid-wide orthogonalisation that run out late.

B2C_GEMM_INJECT_TIMEOUT=2 lets a wait of CTA 0 run out (1 ms) before its tiles of
the last product, 3 its poll of the last barrier once it has been counted there:
the other CTAs finish normally, and of the result only what that CTA should
have written is NaN. The result's memory holds 7 before, so that what nobody
wrote shows."""

import ctypes

import pytest
import torch

from mlx_addons_b200 import _lib

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DEV = "cuda:0"
MUON = (3.4445, -4.7750, 2.0315)


@pytest.fixture(autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _fault():
    f = ctypes.c_uint(7)
    assert _lib.load().b2c_take_device_fault(ctypes.byref(f)) == 0
    return f.value


def _orthogonalize(G, steps):
    lib = _lib.load()
    b, m, n = G.shape
    code = {F32: _lib.F32, BF16: _lib.BF16, F16: _lib.F16}[G.dtype]
    g = _lib.Matrix(G.data_ptr(), *G.stride())
    ws = torch.empty(lib.b2c_orthogonalize_workspace_size(code, g, b, m, n), dtype=torch.uint8, device=DEV)
    out = torch.full(G.shape, 7.0, dtype=G.dtype, device=DEV)
    coef = (ctypes.c_double * (3 * steps))(*(MUON * steps))
    rc = lib.b2c_orthogonalize(code, g, out.data_ptr(), b, m, n, coef, steps, 1e-7, ws.data_ptr(), ws.numel(),
                               torch.cuda.current_stream().cuda_stream)
    _lib.check(rc, "orthogonalize")
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("mode", ["2", "3"])
@pytest.mark.parametrize("shape,dtype", [((1, 256, 256), F32), ((2, 140, 500), F32), ((2, 500, 140), F16), ((2, 300, 1000), BF16),
                                         ((64, 512, 512), BF16), ((1, 1000, 517), BF16)])
@pytest.mark.parametrize("steps", [1, 5])
def test_late(monkeypatch, shape, dtype, steps, mode):
    g = torch.Generator(device=DEV).manual_seed(3)
    G = torch.randn(*shape, generator=g, device=DEV).to(dtype)
    _fault()
    want = _orthogonalize(G, steps)
    assert _fault() == 0 and bool(torch.isfinite(want).all())
    monkeypatch.setenv("B2C_GEMM_INJECT_TIMEOUT", mode)
    bad = _orthogonalize(G, steps)
    monkeypatch.delenv("B2C_GEMM_INJECT_TIMEOUT")
    lost = torch.isnan(bad)
    assert torch.equal(bad[~lost], want[~lost])
    if mode == "2" or bool(lost.any()):  # (3: a CTA that is the last to reach the barrier does not poll)
        assert _fault() != 0 and bool(lost.any())
        # one CTA's tiles: a share of the whole that one CTA in two (the fewest here) can have
        assert float(lost.double().mean()) <= 0.5
    assert torch.equal(_orthogonalize(G, steps), want) and _fault() == 0
