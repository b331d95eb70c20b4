"""Newton-Schulz orthogonalisation of matrices, the step that the Muon
optimiser takes on an update. The reference has no counterpart."""

from __future__ import annotations

import ctypes

import torch

from .. import _lib
from ._gemm import _DTYPES, _back, _call, _guard, _matrix, _native, _on_device

_COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def _triples(coefficients, steps, name):
    try:
        flat = [float(c) for row in coefficients for c in (row if hasattr(row, "__len__") else (row,))]
    except TypeError:
        raise ValueError(f"{name}: coefficients must be (a, b, c) or one such triple a step") from None
    if len(flat) == 3:
        flat = flat * steps
    if len(flat) != 3 * steps:
        raise ValueError(f"{name}: {steps} steps need 3 coefficients or {3 * steps}, got {len(flat)}")
    return flat


def orthogonalize(G, steps: int = 5, coefficients=_COEFFICIENTS, eps: float = 1e-7):
    """Newton-Schulz iteration towards the orthogonal polar factor of G.

        X = G / (|G|_F + eps);   steps times   X <- a X + (b S + c S S) X,  S = X X^T

    G (..., m, n), every matrix with its own norm; the iteration runs on the
    smaller side (S = X^T X from the right where m > n). ``coefficients`` is
    one (a, b, c) or a sequence of one for each step; the default takes every
    singular value above about 1/400 of |G|_F to 0.68 ... 1.21, as an optimiser's update
    needs it; (1.875, -1.25, 0.375) converges to 1 in more steps. The
    polynomials may not let a singular value grow past 3.5.

    float32 and float16 inputs are computed with 22-bit factors, which comes
    closer to the exact iteration than float32 products do, larger bfloat16 ones with 11-bit factors (8 times finer than bfloat16);
    sums and norms are held in 32 bits or more and the result is rounded once to
    G's type. A matrix of zeros gives zeros (NaN where eps is 0); one with a NaN or an infinity
    gives NaN. Records no gradient, in neither mode: operands that carry one are refused."""
    name = "orthogonalize"
    Gt, kind = _native(G, "G", name)
    if Gt.dim() < 2:
        raise ValueError(f"{name}: G needs two dimensions or more, got {tuple(Gt.shape)}")
    if isinstance(steps, bool) or int(steps) != steps or not 1 <= steps <= 64:
        raise ValueError(f"{name}: steps must be a whole number from 1 to 64, got {steps!r}")
    steps = int(steps)
    coef = _triples(coefficients, steps, name)
    host = not Gt.is_cuda
    dev, (Gt,) = _on_device([Gt])
    m, n = Gt.shape[-2:]
    batch = 1
    for d in Gt.shape[:-2]:
        batch *= d
    G3 = Gt if Gt.dim() <= 3 else Gt.reshape((batch, m, n))
    out = torch.empty(Gt.shape, dtype=Gt.dtype, device=dev)
    lib = _lib.load()
    g, code = _matrix(G3), _DTYPES[Gt.dtype]
    with _guard(dev):
        _call("b2c_orthogonalize", lib.b2c_orthogonalize,
              (code, g, out.data_ptr(), batch, m, n, (ctypes.c_double * len(coef))(*coef), steps, float(eps)),
              lib.b2c_orthogonalize_workspace_size, (code, g, batch, m, n), dev)
    return _back((out,), kind, host)[0]
