"""Tails of the activations and of their slopes, relative to their values."""

import pytest
import torch

import mlx_addons_b200.linalg as la
from tests._exact import HALF, act64

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DEV = "cuda:0"
# half a subnormal step of the type
TINY = {F32: 2.0**-150, BF16: 2.0**-134, F16: 2.0**-25}


@pytest.fixture(autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _act64(x, name):
    if name == "gelu":  # log_ndtr keeps its relative accuracy in the lower tail
        return x * torch.special.log_ndtr(x).exp()
    return act64(x, name) if name != "gelu_tanh" else x * torch.sigmoid(2 * 0.7978845608028654 * (x + 0.044715 * x**3))


def _slope64(z, name):
    """(act'(z), the sum of its terms' sizes) by closed forms that keep their relative accuracy in both tails."""
    if name == "relu":
        return (z > 0).double(), (z > 0).double()
    if name == "gelu":
        cdf, bell = torch.special.log_ndtr(z).exp(), torch.exp(-z * z / 2) * 0.3989422804014327
        rest = torch.where(bell > 0, z * bell, torch.zeros_like(z))
    else:
        c = 2 * 0.7978845608028654
        u = z if name == "silu" else c * (z + 0.044715 * z**3)
        du = torch.ones_like(z) if name == "silu" else c * (1 + 3 * 0.044715 * z * z)
        cdf = torch.sigmoid(u)
        bell = torch.sigmoid(u) * torch.sigmoid(-u)
        rest = torch.where(bell > 0, z * bell * du, torch.zeros_like(z))
    return cdf + rest, cdf + rest.abs()


def _outputs(x, act):
    """act(x) for a column x through the FP32 units and, as rows of 64 against the identity, through the tensor cores."""
    one = torch.ones(1, 1, device=DEV, dtype=x.dtype)
    eye = torch.eye(64, device=DEV, dtype=x.dtype)
    return la.gemm(x, one, activation=act), la.gemm(x.reshape(-1, 64), eye, activation=act).reshape(-1, 1)


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_16_bit_values(dtype, act):
    """Every output within half a step of its own and 2^-14 of its value, down to the type's smallest. 2^-14 is an eighth
    of a half step of float16: exp(-x^2 / 2) takes its exponent, up to 88, from a product rounded to 2^-24 of it (about
    2^-17 of the result), which leaves the approximations of Phi and of the sigmoid the rest."""
    x = torch.linspace(-12.5, 12.5, 64 * 2048, device=DEV).to(dtype).reshape(-1, 1)
    ref = _act64(x.double(), act)
    for y in _outputs(x, act):
        over = (y.double() - ref).abs() - (HALF[dtype] * (1 + 2.0**-14) + 2.0**-14) * ref.abs() - TINY[dtype]
        at = int(over.argmax())
        assert float(over.max()) <= 0, (float(x[at]), float(y[at]), float(ref[at]))


def _check_slopes(got, x, act, scale):
    """dP is rounded once; evaluating the terms costs 2^-14 of them in 16 bits, as above, and 2^-17 in 32 (exp of up to 88
    from an argument rounded to 2^-24 of it); in 32 bits Phi comes from 1 + erf, rounded to 2^-24 in itself."""
    ref, terms = _slope64(x.double(), act)
    own = 2.0**-17 if x.dtype == F32 else 2.0**-14
    over = (got.double() - scale * ref).abs() - scale * (HALF[x.dtype] * ref.abs() + 2 * own * terms) - TINY[x.dtype]
    over = over - (scale * 2.0**-23 if x.dtype == F32 else 0)
    at = int(over.argmax())
    assert float(over.max()) <= 0, (float(x.flatten()[at]), float(got.flatten()[at]), float(scale * ref.flatten()[at]))
    return scale * ref


@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_slopes_far_out(dtype, act):
    """Finite pre-activations of any size have finite slopes, 0 or 1 far from zero."""
    top = float(torch.finfo(dtype).max)
    far = [v for v in (30.0, 1e2, 1e4, 6e4, 1e6, 1e13, 1e19, 2e19, 1e20, 1e30, 1e38, top) if v <= top]
    pre = torch.tensor([s * v for v in far for s in (1, -1)], device=DEV, dtype=dtype).reshape(-1, 1)
    dY = torch.full_like(pre, 3.0)
    one = torch.ones(1, 1, device=DEV, dtype=dtype)
    A = torch.ones_like(pre)
    dA, dB, db, _ = la.gemm_grad(dY, A, one, pre, act, need_bias=True)
    want = _check_slopes(dA, pre, act, 3.0)
    n = float(want.sum())  # 3 for each positive one
    assert abs(n - 3 * len(far)) < 1e-9 and float(db) == round(n) and float(dB) == round(n)


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_slopes_in_the_tail(dtype, act):
    """Slopes over the range where they vary, within roundings of their two terms."""
    x = torch.linspace(-12.5, 12.5, 64 * 512, device=DEV).to(dtype).reshape(-1, 1)
    one = torch.ones(1, 1, device=DEV, dtype=dtype)
    _check_slopes(la.gemm_grad(torch.ones_like(x), x, one, x, act)[0], x, act, 1.0)
