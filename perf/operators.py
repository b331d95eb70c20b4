"""Cases, plain forms and 64-bit values of the products that a model trains and answers with:

    gemm           Y = act(alpha A B + bias) + beta R, and the pre-activation where it is kept for the gradient
    gemm_grad      its gradients: dA, dB, dbias (and beta dY)
    orthogonalize  the Newton-Schulz iteration X <- a X + (b X X^T + c (X X^T)^2) X on X = G / (|G|_F + eps)

With ``own`` false, ``run`` computes them with elementary torch operations in 32 bits (norms and angles of
activations in the same), rounded once at the end; with ``own`` true it calls mlx_addons_b200.linalg.
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
EPS = 1e-7


def listed():
    return [
        # one token through a layer's weights, 134 MB of them: the step of an answer
        _gemm("token_bf16", "bf16", 1, 8192, 8192, weights=True, bias=True, activation="silu"),
        # one short vector through a small odd layer: latency alone
        _gemm("token_small_f32", "f32", 1, 1000, 777, weights=True, bias=True),
        # sixteen sequences answered together, weights stored (K, N), added to the residual stream
        _gemm("few_f16", "f16", 16, 4096, 16384, bias=True, activation="gelu_tanh", residual=True),
        # a training batch's first projection, its pre-activation kept for the gradient
        _gemm("forward_bf16", "bf16", 8192, 4096, 16384, weights=True, bias=True, activation="gelu", keep=True),
        # odd sizes in 32 bits: no row starts on a 16-byte boundary
        _gemm("ragged_f32", "f32", 1000, 777, 1301, bias=True, activation="silu", residual=True),
        # a thousand products of the blocked tier's size, each added to its own matrix
        _gemm("batched_f32", "f32", 256, 256, 256, batch=1000, residual=True),
        # the projection's gradients in a training step
        _grad("grad_bf16", "bf16", 4096, 4096, 8192, weights=True, activation="gelu", bias=True),
        # gradients of a ragged layer in 32 bits
        _grad("grad_ragged_f32", "f32", 333, 257, 514, activation="silu", bias=True),
        # the headline batch of this package, orthogonalised: 10,000 matrices of 64 x 64
        _orth("orth_batch_f32", "f32", 10000, 64, 64),
        # one small projection's update: latency
        _orth("orth_small_bf16", "bf16", 1, 128, 512),
        # odd sides, tall, in 32 bits
        _orth("orth_ragged_f32", "f32", 3, 1000, 517),
        # the updates of four square projections
        _orth("orth_large_bf16", "bf16", 4, 4096, 4096),
    ]


def _gemm(name, dtype, m, k, n, batch=0, weights=False, bias=False, activation="", residual=False, keep=False):
    """weights: B is the transposed view of an (N, K) array. batch 0: two-dimensional."""
    return {"name": name, "op": "gemm", "dtype": dtype, "m": m, "k": k, "n": n, "batch": batch, "weights": weights,
            "bias": bias, "activation": activation, "residual": residual, "keep": keep}


def _grad(name, dtype, m, k, n, batch=0, weights=False, activation="", bias=False):
    return {"name": name, "op": "grad", "dtype": dtype, "m": m, "k": k, "n": n, "batch": batch, "weights": weights,
            "bias": bias, "activation": activation}


def _orth(name, dtype, batch, m, n):
    return {"name": name, "op": "orth", "dtype": dtype, "batch": batch, "m": m, "n": n}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A product of 1 to 8192 rows, its gradients, or an orthogonalisation, in any of the types."""
    op = rng.choice(["gemm", "gemm", "grad", "orth", "orth"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    act = rng.choice(["", "relu", "gelu", "gelu_tanh", "silu"])
    yes = lambda: rng.random() < 0.5  # noqa: E731
    if op == "orth":
        batch, m, n = rng.choice([1, 1, _log(rng, 2, 500)]), _log(rng, 16, 4096), _log(rng, 16, 8192)
        while batch > 1 and batch * m * n > 4 << 24:
            batch //= 2
        if m * n > 1 << 25:
            m //= 2
        case = _orth("", dtype, batch, m, n)
    else:
        batch = rng.choice([0, 0, _log(rng, 2, 200)])
        m = rng.choice([_log(rng, 1, 32), _log(rng, 1, 8192)])
        k, n = _log(rng, 64, 8192), _log(rng, 64, 16384)
        if yes():  # whole multiples of 64, as layers mostly are
            k, n = -(-k // 64) * 64, -(-n // 64) * 64
        while batch and batch * (m * k + k * n + m * n) > 1 << 27:
            batch //= 2
        if op == "gemm":
            case = _gemm("", dtype, m, k, n, batch, yes(), yes(), act, yes(), bool(act) and yes())
        else:
            case = _grad("", dtype, m, k, n, batch, yes(), act, yes())
    del case["name"]
    return case


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    b, m, n = max(1, case["batch"]), case["m"], case["n"]
    if case["op"] == "orth":
        s, l = min(m, n), max(m, n)
        # X X^T and its square are symmetric: half of each; then one full product
        return {"bytes": 2 * size * b * m * n, "flops": STEPS * b * (3.0 * s * s * l + float(s) ** 3)}
    k = case["k"]
    if case["op"] == "gemm":
        outs = 1 + case["keep"] + case["residual"]
        return {"bytes": size * (b * (m * k + k * n + outs * m * n) + case["bias"] * n), "flops": 2.0 * b * m * k * n}
    ins = 2 if case["activation"] else 1
    return {"bytes": size * (b * (2 * m * k + 2 * k * n + ins * m * n) + case["bias"] * n), "flops": 4.0 * b * m * k * n}


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------

def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def rand(*shape, scale=1.0):
        t = torch.randn(*shape, generator=g, device="cuda")
        return (t * scale).to(dt)

    b, m, n = case["batch"], case["m"], case["n"]
    if case["op"] == "orth":
        # a gradient: a few strong directions over a broad floor
        r = min(8, m, n)
        u = torch.randn(b, m, r, generator=g, device="cuda")
        v = torch.randn(b, r, n, generator=g, device="cuda")
        floor = torch.randn(b, m, n, generator=g, device="cuda")
        G = torch.baddbmm(floor, u, v, beta=1e-3, alpha=2e-3 / math.sqrt(r)).to(dt)
        return {"G": G[0] if b == 1 else G}
    k = case["k"]
    lead = (b,) if b else ()
    A = rand(*lead, m, k)
    if case["weights"]:
        B = rand(*lead, n, k, scale=1 / math.sqrt(k)).mT
    else:
        B = rand(*lead, k, n, scale=1 / math.sqrt(k))
    out = {"A": A, "B": B, "bias": rand(n, scale=0.1) if case["bias"] and case["op"] == "gemm" else None}
    if case["op"] == "gemm":
        out["R"] = rand(*lead, m, n) if case["residual"] else None
    else:
        out["dY"] = rand(*lead, m, n, scale=1e-2)
        out["pre"] = rand(*lead, m, n) if case["activation"] else None
    return out


def prepare(case, seed):
    return {"case": case, **_inputs(case, seed)}


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    dt = DTYPES[case["dtype"]]
    if case["op"] == "orth":
        return _plain_orth(state["G"].float()).to(dt)
    A, B = state["A"].float(), state["B"].float()
    if case["op"] == "gemm":
        pre = A @ B
        if state["bias"] is not None:
            pre = pre + state["bias"].float()
        y = _act(pre, case["activation"])
        if state["R"] is not None:
            y = y + state["R"].float()
        return (y.to(dt), pre.to(dt)) if case["keep"] else (y.to(dt),)
    dP = state["dY"].float()
    if case["activation"]:
        dP = dP * _act_slope(state["pre"].float(), case["activation"])
    outs = [(dP @ B.mT).to(dt), (A.mT @ dP).to(dt)]
    if case["bias"]:
        outs.append(dP.reshape(-1, case["n"]).sum(0).to(dt))
    return tuple(outs)


def _run_own(case, state):
    from mlx_addons_b200 import linalg

    if case["op"] == "orth":
        return linalg.orthogonalize(state["G"])
    act = case["activation"] or None
    if case["op"] == "gemm":
        out = linalg.gemm(state["A"], state["B"], bias=state["bias"], activation=act, residual=state["R"],
                          return_pre=case["keep"])
        return out if case["keep"] else (out,)
    dA, dB, dbias, _ = linalg.gemm_grad(state["dY"], state["A"], state["B"], pre=state["pre"], activation=act,
                                        need_bias=case["bias"])
    return (dA, dB, dbias) if case["bias"] else (dA, dB)


def _act(x, name):
    if name == "relu":
        return x.clamp_min(0)
    if name == "gelu":
        return 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))
    if name == "silu":
        return x / (1 + torch.exp(-x))
    return x


def _act_slope(x, name):
    if name == "relu":
        return (x > 0).to(x.dtype)
    if name == "gelu":
        return 0.5 * (1 + torch.erf(x * math.sqrt(0.5))) + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        t = torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x))
        return 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * x * x)
    s = 1 / (1 + torch.exp(-x))
    return s * (1 + x * (1 - s))


def _plain_orth(G):
    norm = G.double().square().sum((-2, -1), keepdim=True).sqrt().float()
    tall = G.shape[-2] > G.shape[-1]
    X = (G.mT if tall else G) / (norm + EPS)
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        S = X @ X.mT
        X = a * X + (b * S + c * (S @ S)) @ X
    return X.mT if tall else X


# ---------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------

def exact(case, seed):
    x = _inputs(case, seed)
    if case["op"] == "orth":
        G = x["G"].double()
        G = G / (torch.linalg.matrix_norm(G, keepdim=True) + EPS)
        # every step multiplies by a polynomial in the smaller Gram matrix, and these commute: the product of
        # the polynomials is kept, and meets G once at the end
        wide = G.shape[-2] <= G.shape[-1]
        S = torch.matmul(G, G.mT) if wide else torch.matmul(G.mT, G)
        Q = eye = torch.eye(S.shape[-1], dtype=torch.float64, device=S.device)
        a, b, c = COEFFICIENTS
        for _ in range(STEPS):
            P = torch.matmul(S, b * eye + c * S) + a * eye
            Q = torch.matmul(P, Q)
            S = torch.matmul(P, torch.matmul(S, P))
        return torch.matmul(Q, G) if wide else torch.matmul(G, Q)
    A, B = x["A"].double(), x["B"].double()
    name = case["activation"]
    if case["op"] == "gemm":
        z = torch.matmul(A, B)
        if x["bias"] is not None:
            z += x["bias"].double()
        y = {"": lambda t: t, "relu": torch.relu, "silu": lambda t: t * torch.sigmoid(t),
             "gelu": lambda t: t * torch.special.ndtr(t),
             "gelu_tanh": lambda t: t * torch.sigmoid(2 * math.sqrt(2 / math.pi) * t * (1 + 0.044715 * t ** 2))}[name](z)
        if x["R"] is not None:
            y = y + x["R"].double()
        return (y, z) if case["keep"] else (y,)
    D = x["dY"].double()
    if name:
        z = x["pre"].double()
        if name == "relu":
            D = torch.where(z > 0, D, torch.zeros_like(D))
        elif name == "gelu":
            D = D * (torch.special.ndtr(z) + z * torch.exp(-z ** 2 / 2) / math.sqrt(2 * math.pi))
        else:
            # z sigmoid(u(z)): sigmoid + z u' sigmoid (1 - sigmoid)
            h = 2 * math.sqrt(2 / math.pi)
            u = z if name == "silu" else h * (z + 0.044715 * z ** 3)
            du = 1 if name == "silu" else h * (1 + 3 * 0.044715 * z ** 2)
            D = D * (torch.sigmoid(u) + z * du * torch.sigmoid(u) * torch.sigmoid(-u))
    outs = [torch.matmul(D, B.mT), torch.matmul(A.mT, D)]
    if case["bias"]:
        outs.append(D.flatten(0, -2).sum(0))
    return tuple(outs)
