"""64-bit values and error bounds of the products and the orthogonalisation.

A rounding to a type is off by at most half a step, finfo(t).eps / 2 of the
value: HALF. A float32 sum of K terms, in any order, tensor-core sums that
truncate instead of round included, is off by at most K 2^-23 sum |terms|;
over independent terms the errors of the additions add like a random walk,
which the norm-wise bounds use: sqrt(K) steps of 2^-23 of the sum, and at most
32 one-sided ones (a truncating sum runs over 32 additions at the most before
it is joined in float32).
"""

from __future__ import annotations

import math

import torch

HALF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
ACTS = [None, "relu", "gelu", "gelu_tanh", "silu"]


def act64(x, name):
    if name is None:
        return x
    if name == "relu":
        return torch.where(x < 0, torch.zeros_like(x), x)
    if name == "gelu":
        return x * torch.special.ndtr(x)
    if name == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x**3)))
    return x * torch.sigmoid(x)


def slope64(x, name):
    """act'(x) through differentiation by torch in 64 bits."""
    if name is None:
        return torch.ones_like(x)
    z = x.detach().clone().requires_grad_(True)
    with torch.enable_grad():
        (g,) = torch.autograd.grad(act64(z, name).sum(), z)
    return g


def gemm64(A, B, bias=None, act=None, R=None, alpha=1.0, beta=1.0):
    """(Y, pre, bound of Y's error before its own rounding, the same of pre)."""
    A, B = A.double(), B.double()
    K = A.shape[-1]
    pre = alpha * torch.matmul(A, B)
    size = abs(alpha) * torch.matmul(A.abs(), B.abs())
    if bias is not None:
        pre = pre + bias.double()
        size = size + bias.double().abs()
    # sum, alpha, bias: K + 2 roundings
    e_pre = (K + 4) * 2.0**-23 * size
    y = act64(pre, act)
    # every activation here has a slope within 1.13; evaluating it costs a few roundings of its terms
    e_y = 1.13 * e_pre + (8 * 2.0**-23 * (pre.abs() + 1e-3) if act else 0)
    if R is not None:
        y = y + beta * R.double()
        e_y = e_y + 2.0**-22 * (y.abs() + abs(beta) * R.double().abs())
    return y, pre, e_y, e_pre


def check(out, ref, err, what="", K=1, roundings=1.0):
    """Every element within its bound plus the rounding of the output, and the whole within the norm-wise bound."""
    half = HALF[out.dtype]
    o, r = out.double(), ref
    tiny = 2.0**-24 if out.dtype == torch.float16 else 0.0  # half a subnormal step
    over = (o - r).abs() - (err + half * (r.abs() + err) + tiny)
    assert out.shape == ref.shape, (what, out.shape, ref.shape)
    assert bool(torch.isfinite(o).all()), what
    if r.numel():
        assert float(over.max()) <= 0, (what, float(over.max()), float((o - r).abs().max()))
        n = float(torch.linalg.vector_norm(r))
        rel = float(torch.linalg.vector_norm(o - r)) / n if n else 0.0
        assert rel <= roundings * half + 2.0**-23 * (math.sqrt(K) + 32), (what, rel)


# ---------------------------------------------------------------------------
# orthogonalisation
# ---------------------------------------------------------------------------

MUON = (3.4445, -4.7750, 2.0315)


def orth64(G, steps=5, coefficients=MUON, eps=1e-7):
    """The iteration in 64 bits and its iterates (on the smaller side)."""
    rows = coefficients if hasattr(coefficients[0], "__len__") else [coefficients] * steps
    X = G.double()
    X = X / (torch.linalg.matrix_norm(X, keepdim=True) + eps)
    tall = X.shape[-2] > X.shape[-1]
    X = X.mT if tall else X
    its = [X]
    for a, b, c in rows:
        S = torch.matmul(X, X.mT)
        X = a * X + torch.matmul(b * S + c * torch.matmul(S, S), X)
        its.append(X)
    return (X.mT if tall else X), its


def orth_bound(its, steps, coefficients, unit, dtype):
    """Bound of every matrix's error in the Frobenius norm, for factors held
    to `unit` (half a step) and sums in 32 bits. its: iterates (batch, m, n).

    A step maps X to p(X) on its singular values; its Lipschitz constant in
    the Frobenius norm is the largest |p'| over [0, s], s the largest of them.
    Its own error: S, P and X' are each held to `unit`, and their sums add
    2^-23 (sqrt(K) + 32) of the products of their norms."""
    rows = coefficients if hasattr(coefficients[0], "__len__") else [coefficients] * steps
    fro = torch.linalg.matrix_norm
    grid = torch.linspace(0, 1, 1001, dtype=torch.float64, device=its[0].device)
    e = (unit + 2.0**-23) * fro(its[0])
    for t, (a, b, c) in enumerate(rows):
        X, Xn = its[t], its[t + 1]
        S = torch.matmul(X, X.mT)
        Q = S @ S
        Q = Q @ Q  # |S|_2 <= |S^4|_F^(1/4)
        s = fro(Q) ** 0.125 + e
        x = (s[:, None] * grid) ** 2
        lip = (a + 3 * b * x + 5 * c * x**2).abs().amax(-1)
        fs = fro(S) + 2 * s * e
        u = 2 * unit + 2.0**-23 * (math.sqrt(max(X.shape[-2:])) + 32)
        e_p = (abs(b) + 2 * abs(c) * s * s) * u * fs + u * (abs(b) + abs(c) * s * s) * fs
        e = lip * e + e_p * s + u * (fro(Xn) + abs(a) * fro(X))
    return e + HALF[dtype] * (fro(its[-1]) + e)
