"""Matrix products with an epilogue, and their gradients.

    gemm(A, B, bias, activation, residual)   Y = act(alpha A B + bias) + beta R
    gemm_grad(dY, A, B, pre, activation)     dA, dB, dbias, dR

float32, bfloat16 and float16 are computed in their own type (operands and
outputs; sums and the epilogue are held in 32 bits, each output is rounded
once); anything else is cast to float32 like in the rest of the package. Any
strides are taken as they are: a layer's (N, K) weights go in as ``W.mT``
without a copy. The reference has no counterpart; its products are MLX's own.
"""

from __future__ import annotations

import contextlib
import sys
from typing import Optional

import torch
from torch.autograd import forward_ad as _fwad

from .. import _lib

_pkg = sys.modules[__package__]  # the helpers of linalg/__init__.py, which imports this module at its end
_NO_GUARD = contextlib.nullcontext()
_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def _native(x, what, name):
    """Any accepted array as a torch tensor of one of the three types."""
    t, kind = _pkg._as_tensor(x, name)
    # no_grad() leaves forward-mode tangents on, so these are refused there too
    if (t.requires_grad and torch.is_grad_enabled()) or (_fwad._current_level >= 0 and _fwad.unpack_dual(t).tangent is not None):
        raise ValueError(f"{name}: {what} requires a gradient, which {name} does not record; detach it, or for reverse "
                         "mode call under torch.no_grad() (gemm_grad computes the gradients of gemm)")
    if t.dtype not in _DTYPES:
        if t.is_complex():
            raise ValueError(f"{name}: {what} is complex")
        t = t.to(torch.float32)
    return t, kind


def _same_type(name, first, *others):
    for what, t in others:
        if t is not None and t.dtype != first.dtype:
            raise ValueError(f"{name}: {what} is {t.dtype}, expected {first.dtype}")


def _on_device(tensors):
    """Host tensors go to the current CUDA device, others to the first one's."""
    dev = tensors[0].device
    if dev.type != "cuda":
        _pkg._require_cuda()
        dev = torch.device("cuda", torch.cuda.current_device())
    return dev, [t if t is None or t.device == dev else t.to(dev) for t in tensors]


def _guard(dev):
    """The device as the current one, at no cost where it is."""
    return _NO_GUARD if torch._C._cuda_getDevice() == dev.index else torch.cuda.device(dev)


def _matrix(t):
    """b2c_matrix of a tensor (batch, rows, cols) or (rows, cols); torch has no
    negative strides."""
    s = t.stride()
    return _lib.Matrix(t.data_ptr(), 0 if len(s) == 2 else s[-3], s[-2], s[-1])


def _addr(t):
    return None if t is None else t.data_ptr()


def _call(what, fn, args, ws_fn, ws_args, dev, scratch=False):
    """fn(*args, workspace, bytes, stream); a call that needs scratch says so
    before it launches anything, unless it is known to need some."""
    stream = torch._C._cuda_getCurrentRawStream(dev.index)
    rc = _lib.B2C_ERR_WORKSPACE if scratch else fn(*args, None, 0, stream)
    if rc == _lib.B2C_ERR_WORKSPACE:
        n = ws_fn(*ws_args)
        ws = torch.empty(n, dtype=torch.uint8, device=dev)
        rc = fn(*args, ws.data_ptr(), n, stream)
    if rc:
        _lib.check(rc, what)


def _gemm_dev(A, B, bias, act, R, alpha, beta, want_pre):
    """A (batch, M, K) or (M, K), B (batch, K, N) or (K, N), on one device."""
    lib = _lib.load()
    dev = A.device
    M, K = A.shape[-2:]
    N = B.shape[-1]
    batch = A.shape[0] if A.dim() == 3 else 1
    Y = torch.empty((batch, M, N) if A.dim() == 3 else (M, N), dtype=A.dtype, device=dev)
    pre = torch.empty_like(Y) if want_pre else None
    code, a, b = _DTYPES[A.dtype], _matrix(A), _matrix(B)
    r = None if R is None else _matrix(R)
    with _guard(dev):
        _call("b2c_gemm", lib.b2c_gemm,
              (code, a, b, _addr(bias), r, Y.data_ptr(), _addr(pre), batch, M, K, N, alpha, beta, act),
              lib.b2c_gemm_workspace_size, (code, a, b, batch, M, K, N), dev)
    return Y, pre


def _activation(activation, name):
    if activation not in _lib.ACTIVATIONS:
        raise ValueError(f"{name}: activation must be one of {list(_lib.ACTIVATIONS)}, got {activation!r}")
    return _lib.ACTIVATIONS[activation]


def _check_product(A, B, name):
    if A.dim() < 2 or B.dim() < 2:
        raise ValueError(f"{name}: A and B need two dimensions or more, got {tuple(A.shape)} and {tuple(B.shape)}")
    if A.shape[-1] != B.shape[-2]:
        raise ValueError(f"{name}: A is {tuple(A.shape)} but B is {tuple(B.shape)}")
    if B.dim() > 2 and A.shape[:-2] != B.shape[:-2]:
        raise ValueError(f"{name}: leading dimensions differ: A is {tuple(A.shape)}, B is {tuple(B.shape)}")


def _flat(t, lead, shared):
    """(..., M, K) as one matrix of all rows (a shared B) or a batch of them."""
    if not lead or (len(lead) == 1 and not shared):
        return t
    rows, cols = t.shape[-2:]
    n = 1
    for d in lead:
        n *= d
    return t.reshape((n * rows, cols) if shared else (n, rows, cols))


def _back(out, kind, host):
    if not host:
        return out
    out = tuple(None if o is None else o.cpu() for o in out)
    if kind == "numpy":
        out = tuple(None if o is None else o.numpy() for o in out)
    return out


def gemm(A, B, bias=None, activation: Optional[str] = None, residual=None, *, alpha: float = 1.0, beta: float = 1.0,
         return_pre: bool = False):
    """act(alpha * A @ B + bias) + beta * residual, the epilogue in the product's kernel.

    A (..., M, K); B (K, N), or (..., K, N) with A's leading dimensions; bias
    (N,); residual of the result's shape (an expanded view will do);
    activation None, "relu", "gelu", "gelu_tanh" or "silu". All of one type.
    With ``return_pre`` returns (Y, pre), pre = alpha A B + bias being what
    ``gemm_grad`` needs of the activation.

    float32 products are as exact as float32 arithmetic, for values of any size;
    16-bit operands are multiplied exactly and summed in 32 bits. A NaN or an
    infinity stays in the rows and columns that it meets, where it gives what IEEE
    arithmetic gives; a float32 sum whose terms add up, by size, beyond
    float32's range may give NaN in the place of inf. Larger float32 products read three bf16 planes an
    operand, 16-bit ones whose rows do not start on 16 bytes a copy: these take a
    pass of their own and scratch from torch's allocator, 6 and 2 bytes an element. Records no gradient, in neither mode: operands that carry one are refused."""
    name = "gemm"
    act = _activation(activation, name)
    At, kind = _native(A, "A", name)
    Bt, _ = _native(B, "B", name)
    bt = None if bias is None else _native(bias, "bias", name)[0]
    Rt = None if residual is None else _native(residual, "residual", name)[0]
    _check_product(At, Bt, name)
    _same_type(name, At, ("B", Bt), ("bias", bt), ("residual", Rt))
    M, N, lead, shared = At.shape[-2], Bt.shape[-1], tuple(At.shape[:-2]), Bt.dim() == 2
    if bt is not None and tuple(bt.shape) != (N,):
        raise ValueError(f"{name}: bias must have shape ({N},), got {tuple(bt.shape)}")
    if Rt is not None and tuple(Rt.shape) != lead + (M, N):
        raise ValueError(f"{name}: residual must have shape {lead + (M, N)}, got {tuple(Rt.shape)}")
    host = not At.is_cuda
    _, (At, Bt, bt, Rt) = _on_device([At, Bt, bt, Rt])
    Y, pre = _gemm_dev(_flat(At, lead, shared), Bt if shared else _flat(Bt, lead, False),
                       None if bt is None else bt.contiguous(), act, None if Rt is None else _flat(Rt, lead, shared),
                       float(alpha), float(beta), bool(return_pre))
    if len(lead) > 1 or (lead and shared):
        Y = Y.reshape(lead + (M, N))
        pre = None if pre is None else pre.reshape(Y.shape)
    out = _back((Y, pre), kind, host)
    return out if return_pre else out[0]


def gemm_grad(dY, A, B, pre=None, activation: Optional[str] = None, *, alpha: float = 1.0, beta: float = 1.0,
              need_bias: bool = False, need_residual: bool = False):
    """Gradients of ``gemm``: (dA, dB, dbias, dresidual) for the gradient dY
    of its result, with the operands, activation, alpha and beta of the call.

        dP = dY * act'(pre)   dA = alpha dP B^T   dB = alpha A^T dP
        dbias = sum of dP's rows        dresidual = beta dY

    ``pre`` is the second result of ``gemm(..., return_pre=True)``; it is
    needed where there is an activation. dbias and dresidual are None unless
    asked for; dresidual has the result's full shape. A shared B (two
    dimensions) gets the sum over A's leading dimensions. dP is rounded to the
    operands' type once, as an operand of the two products; dbias takes it
    before that. Every sum runs in a fixed order."""
    name = "gemm_grad"
    act = _activation(activation, name)
    dYt, _ = _native(dY, "dY", name)
    At, kind = _native(A, "A", name)
    Bt, _ = _native(B, "B", name)
    pt = None if pre is None else _native(pre, "pre", name)[0]
    _check_product(At, Bt, name)
    _same_type(name, At, ("B", Bt), ("dY", dYt), ("pre", pt))
    M, K, N, lead, shared = At.shape[-2], At.shape[-1], Bt.shape[-1], tuple(At.shape[:-2]), Bt.dim() == 2
    for what, t in (("dY", dYt), ("pre", pt)):
        if t is not None and tuple(t.shape) != lead + (M, N):
            raise ValueError(f"{name}: {what} must have shape {lead + (M, N)}, got {tuple(t.shape)}")
    if act and pt is None:
        raise ValueError(f"{name}: the gradient of {activation} needs pre")
    if not act:
        pt = None
    host = not At.is_cuda
    dev, (At, Bt, dYt, pt) = _on_device([At, Bt, dYt, pt])
    A3, dY3 = _flat(At, lead, shared), _flat(dYt, lead, shared)
    B3 = Bt if shared else _flat(Bt, lead, False)
    batch, rows = A3.shape[0] if A3.dim() == 3 else 1, A3.shape[-2]
    full = tuple(A3.shape[:-1]) + (N,)
    dP, dbias, dR = dY3, None, None
    if act:
        dP = torch.empty(full, dtype=At.dtype, device=dev)
    if need_bias:
        dbias = torch.empty((N,), dtype=At.dtype, device=dev)
    if need_residual:
        dR = torch.empty(full, dtype=At.dtype, device=dev)
    if act or need_bias or need_residual:
        lib = _lib.load()
        dy, p = _matrix(dY3), None if pt is None else _matrix(_flat(pt, lead, shared))
        with _guard(dev):
            _call("b2c_gemm_dact", lib.b2c_gemm_dact,
                  (_DTYPES[At.dtype], dy, p, act, float(beta), _addr(dP) if act else None, _addr(dbias), _addr(dR), batch,
                   rows, N), lib.b2c_gemm_dact_workspace_size, (batch, rows, N), dev, need_bias)
    dA, _ = _gemm_dev(dP, B3.mT, None, 0, None, float(alpha), 1.0, False)
    dB, _ = _gemm_dev(A3.mT, dP, None, 0, None, float(alpha), 1.0, False)
    if len(lead) > 1 or (lead and shared):
        dA = dA.reshape(lead + (M, K))
        dB = dB if shared else dB.reshape(lead + (K, N))
        dR = None if dR is None else dR.reshape(lead + (M, N))
    return _back((dA, dB, dbias, dR), kind, host)
