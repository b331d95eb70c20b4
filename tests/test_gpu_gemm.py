"""Products with an epilogue and their gradients against 64-bit values."""

import math

import numpy as np
import pytest
import torch

import mlx_addons_b200.linalg as la
from tests._exact import ACTS, HALF, act64, check, gemm64, slope64

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _rand(gen, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device=DEV) * scale).to(dtype)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _problem(M, K, N, dtype, lead=(), shared=True, trans_a=False, trans_b=False, seed=0):
    g = _gen(seed + 7 * M + 3 * K + N)
    A = _rand(g, *lead, K, M, dtype=dtype).mT if trans_a else _rand(g, *lead, M, K, dtype=dtype)
    bl = () if shared else lead
    s = 1 / math.sqrt(max(K, 1))
    B = _rand(g, *bl, N, K, dtype=dtype, scale=s).mT if trans_b else _rand(g, *bl, K, N, dtype=dtype, scale=s)
    return A, B, _rand(g, N, dtype=dtype), _rand(g, *lead, M, N, dtype=dtype)


SIZES = [(1, 1, 1), (1, 64, 1), (1, 512, 640), (1, 1000, 777), (2, 130, 96), (3, 257, 129), (5, 2049, 65), (8, 1024, 256),
         (9, 96, 1000), (16, 4096, 320), (17, 72, 48), (31, 63, 33), (33, 200, 1), (64, 64, 64), (65, 65, 65),
         (100, 1, 100), (127, 128, 255), (128, 1024, 256), (129, 264, 257), (200, 500, 7), (256, 256, 256),
         (300, 136, 520), (640, 2048, 4), (1000, 777, 301), (1, 8, 20000), (20000, 8, 3)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", SIZES)
def test_sizes(M, K, N, dtype):
    for i, (ta, tb) in enumerate([(False, False), (False, True), (True, False), (True, True)]):
        A, B, bias, R = _problem(M, K, N, dtype, trans_a=ta, trans_b=tb)
        act = ACTS[(M + i) % 5]
        Y, pre = la.gemm(A, B, bias, act, R, alpha=0.75, beta=-1.5, return_pre=True)
        y, p, ey, ep = gemm64(A, B, bias, act, R, 0.75, -1.5)
        assert Y.dtype == dtype and pre.dtype == dtype and Y.device == A.device
        check(pre, p, ep, "pre", K)
        check(Y, y, ey, "Y", K, roundings=1.0)
        check(la.gemm(A, B), *_plain(A, B), what="plain", K=K)


def _plain(A, B):
    y, _, ey, _ = gemm64(A, B)
    return y, ey


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ta,tb", [(False, False), (False, True), (True, False), (True, True)])
@pytest.mark.parametrize("M,K,N,batch", [(1700, 328, 1608, 0), (2048, 64, 2048, 0), (1601, 200, 1793, 0), (300, 136, 520, 13),
                                         (256, 512, 256, 60)])
def test_many_tiles(M, K, N, batch, ta, tb, dtype):
    """Sizes that fill the GPU with the largest tiles, their edges ragged."""
    A, B, bias, R = _problem(M, K, N, dtype, (batch,) if batch else (), shared=not batch, trans_a=ta, trans_b=tb)
    Y, pre = la.gemm(A, B, bias, "gelu", R, return_pre=True)
    y, p, ey, ep = gemm64(A, B, bias, "gelu", R)
    check(pre, p, ep, "pre", K)
    check(Y, y, ey, "Y", K)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N,batch", [(145, 449, 148, 0), (65, 128, 64, 0), (129, 255, 97, 0), (256, 1024, 255, 0), (33, 700, 40, 9),
                                         (77, 150, 30, 31), (13, 2100, 192, 0), (4, 3001, 70, 0), (7, 640, 64, 5)])
def test_sums_split_over_a_cluster(M, K, N, batch, dtype):
    """Few tiles and a long k, in every order of the operands."""
    for ta, tb in [(False, False), (False, True), (True, False), (True, True)]:
        A, B, bias, R = _problem(M, K, N, dtype, (batch,) if batch else (), shared=not batch, trans_a=ta, trans_b=tb)
        Y, pre = la.gemm(A, B, bias, "gelu_tanh", R, alpha=-0.5, beta=2.0, return_pre=True)
        y, p, ey, ep = gemm64(A, B, bias, "gelu_tanh", R, -0.5, 2.0)
        check(pre, p, ep, "pre", K)
        check(Y, y, ey, "Y", K)
        assert torch.equal(la.gemm(A, B, bias, "gelu_tanh", R, alpha=-0.5, beta=2.0), Y)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N", [(1, 96), (70, 40), (160, 144)])
def test_activations(M, N, dtype, act):
    """The whole range of an activation, both tails among it: A = x, B = 1."""
    x = torch.linspace(-30, 30, M * N, device=DEV).to(dtype).reshape(M * N, 1)
    one = torch.ones(1, 1, device=DEV, dtype=dtype)
    Y = la.gemm(x, one, activation=act)
    y, _, ey, _ = gemm64(x, one, None, act)
    check(Y, y, ey, "Y")
    Z = la.gemm(x.reshape(1, -1), torch.eye(M * N, device=DEV, dtype=dtype), activation=act) if M * N <= 96 else Y
    check(Z.reshape(-1, 1), y, ey, "row")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lead,shared", [((5,), True), ((5,), False), ((2, 3), True), ((2, 3), False), ((1,), False)])
@pytest.mark.parametrize("M,K,N", [(1, 64, 48), (20, 33, 70), (130, 128, 64), (64, 256, 192)])
def test_batches(M, K, N, lead, shared, dtype):
    A, B, bias, R = _problem(M, K, N, dtype, lead, shared, trans_b=True)
    Y, pre = la.gemm(A, B, bias, "silu", R, return_pre=True)
    y, p, ey, ep = gemm64(A, B, bias, "silu", R)
    check(pre, p, ep, "pre", K)
    check(Y, y, ey, "Y", K)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides(dtype):
    """Slices, steps, odd offsets, expanded operands and addends."""
    g = _gen(3)
    big = _rand(g, 140, 300, dtype=dtype)
    A, W = big[1:131:2, 3:260], _rand(g, 90, 600, dtype=dtype)[:, 1:515:2].mT  # no unit stride in W
    R = _rand(g, 90, dtype=dtype).expand(65, 90)
    bias = _rand(g, 180, dtype=dtype)[::2]
    Y = la.gemm(A, W, bias, "gelu", R)
    y, _, ey, _ = gemm64(A, W, bias, "gelu", R)
    check(Y, y, ey, "steps", 257)
    row = _rand(g, 1, 128, dtype=dtype).expand(200, 128)
    B = _rand(g, 128, 136, dtype=dtype, scale=0.1)
    check(la.gemm(row, B), *_plain(row, B), what="expanded A", K=128)
    A3 = _rand(g, 1, 70, 128, dtype=dtype).expand(4, 70, 128)
    B3 = _rand(g, 128, 4, 72, dtype=dtype, scale=0.1).permute(1, 0, 2)
    check(la.gemm(A3, B3), *_plain(A3, B3), what="permuted batch", K=128)


@pytest.mark.parametrize("dtype", TYPES)
def test_expanded_operands(dtype):
    """Strides of 0 in every place, their batch stride that of whole rows among them."""
    g = _gen(5)
    for b, M, K, N in [(4, 1, 1024, 1024), (3, 40, 256, 512), (5, 200, 136, 264), (2, 24, 2048, 640)]:
        t, B = _rand(g, b, K, dtype=dtype), _rand(g, b, K, N, dtype=dtype, scale=1 / K)
        for A in (t[:, :1].unsqueeze(1).expand(b, M, K), t.unsqueeze(1).expand(b, M, K),
                  _rand(g, b, M, 1, dtype=dtype).expand(b, M, K), _rand(g, 1, M, K, dtype=dtype).expand(b, M, K),
                  _rand(g, b * M, K, dtype=dtype).as_strided((b, M, K), (K, K, 1))):
            Y = la.gemm(A, B)
            check(Y, *_plain(A, B), what=(A.stride(), M), K=K)
            Z = la.gemm(B.mT, A.mT)
            check(Z, *_plain(B.mT, A.mT), what=(A.stride(), M, "right"), K=K)


@pytest.mark.parametrize("dtype", TYPES)
def test_empty(dtype):
    z = lambda *s: torch.zeros(*s, device=DEV, dtype=dtype)  # noqa: E731
    assert la.gemm(z(0, 5), z(5, 3)).shape == (0, 3)
    assert la.gemm(z(4, 5), z(5, 0)).shape == (4, 0)
    assert la.gemm(z(0, 4, 5), z(5, 3)).shape == (0, 4, 3)
    assert la.gemm(z(0, 4, 5), z(0, 5, 3)).shape == (0, 4, 3)
    bias = torch.arange(3, device=DEV).to(dtype) - 1
    Y, pre = la.gemm(z(4, 0), z(0, 3), bias, "relu", z(4, 3) + 2, return_pre=True)
    assert torch.equal(pre, bias.expand(4, 3)) and torch.equal(Y, (bias.clamp_min(0) + 2).expand(4, 3))
    dA, dB, db, dR = la.gemm_grad(z(0, 3), z(0, 5), z(5, 3), need_bias=True, need_residual=True)
    assert dA.shape == (0, 5) and dR.shape == (0, 3)
    assert torch.equal(dB, z(5, 3)) and torch.equal(db, z(3))
    dA, dB, db, _ = la.gemm_grad(z(4, 0), z(4, 5), z(5, 0), need_bias=True)
    assert torch.equal(dA, z(4, 5)) and dB.shape == (5, 0) and db.shape == (0,)


def _grad64(dY, A, B, pre, act, alpha, beta):
    dP = dY.double()
    if act:
        dP = dP * slope64(pre.double(), act)
    shared = B.dim() == 2
    A2 = A.double().reshape(-1, A.shape[-1]) if shared else A.double()
    dP2 = dP.reshape(-1, dP.shape[-1]) if shared else dP
    B = B.double()
    half = HALF[A.dtype] if act else 0.0
    rows = dP.numel() // max(1, dP.shape[-1])

    def prod(x, y, k, e):
        return alpha * torch.matmul(x, y), ((k + 8) * 2.0**-23 + e) * abs(alpha) * torch.matmul(x.abs(), y.abs())

    # the slope is evaluated to a few float32 roundings of its terms, and dP is rounded once
    e = half + 16 * 2.0**-23
    dA, eA = prod(dP2, B.mT, B.shape[-1], e)
    dB, eB = prod(A2.mT, dP2, A2.shape[-2], e)
    if act:  # a slope near zero is off by roundings of its terms, not of itself
        eA = eA + 16 * 2.0**-23 * abs(alpha) * torch.matmul(dY.double().reshape(dP2.shape).abs(), B.mT.abs())
        eB = eB + 16 * 2.0**-23 * abs(alpha) * torch.matmul(A2.mT.abs(), dY.double().reshape(dP2.shape).abs())
    db = dP.reshape(-1, dP.shape[-1]).sum(0)
    eb = (rows + 24) * 2.0**-23 * dY.double().abs().reshape(-1, dP.shape[-1]).sum(0) * 1.2
    return dA.reshape(A.shape), eA.reshape(A.shape), dB, eB, db, eb


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", [(1, 64, 96), (7, 33, 21), (64, 128, 192), (100, 257, 65), (200, 96, 300), (513, 40, 8)])
@pytest.mark.parametrize("lead,shared", [((), True), ((3,), True), ((3,), False)])
def test_gradients(M, K, N, lead, shared, dtype):
    act = ACTS[(M + K + len(lead)) % 5]
    A, B, _, dY = _problem(M, K, N, dtype, lead, shared, trans_b=K % 2 == 0)
    pre = _rand(_gen(5), *lead, M, N, dtype=dtype, scale=2.0)
    dA, dB, db, dR = la.gemm_grad(dY, A, B, pre, act, alpha=0.5, beta=3.0, need_bias=True, need_residual=True)
    xA, eA, xB, eB, xb, eb = _grad64(dY, A, B, pre, act, 0.5, 3.0)
    check(dA, xA, eA, "dA", N, roundings=2.0)
    check(dB, xB, eB, "dB", M * max(1, math.prod(lead)), roundings=2.0)
    check(db, xb, eb, "dbias", M * max(1, math.prod(lead)), roundings=1.0)
    check(dR, 3.0 * dY.double(), 0.0 * dY.double(), "dR")


@pytest.mark.parametrize("act", ACTS)
def test_gradient_against_differences(act):
    """(Y(x + h) - Y(x - h)) / 2h along random directions, in float32: the difference
    quotient is off by h^2 times the third derivatives and by 2^-22 |Y| / h."""
    g = _gen(11)
    A, B, bias, R = (_rand(g, *s) for s in [(40, 24), (24, 30), (30,), (40, 30)])
    B = B * 0.3
    dY = _rand(g, 40, 30)
    if act == "relu":  # no kink within reach of h
        keep = (A @ B + bias).abs() > 0.2
        dY = dY * keep
    _, pre = la.gemm(A, B, bias, act, R, return_pre=True)
    dA, dB, db, dR = la.gemm_grad(dY, A, B, pre, act, need_bias=True, need_residual=True)
    h = 2.0**-7
    for grad, at in ((dA, 0), (dB, 1), (db, 2), (dR, 3)):
        x = [A, B, bias, R]
        d = _rand(g, *x[at].shape)
        d = d / torch.linalg.vector_norm(d)
        up, down = list(x), list(x)
        up[at], down[at] = x[at] + h * d, x[at] - h * d
        f = lambda v: (la.gemm(v[0], v[1], v[2], act, v[3]).double() * dY.double()).sum()  # noqa: E731
        want = float((f(up) - f(down)) / (2 * h))
        got = float((grad.double() * d.double()).sum())
        # |d| = 1 moves an entry of pre by at most |A|_row or |B|_col < 8, third derivatives are below 2
        scale = float(dY.abs().sum())
        assert abs(want - got) <= 2 * (8 * h) ** 2 * 0.02 * scale + 2.0**-20 * scale / h, (act, at, want, got)


def test_grad_without_activation_reads_dY_as_it_lies():
    g = _gen(2)
    dY = _rand(g, 1, 72, dtype=BF16).expand(130, 72)
    A, B = _rand(g, 130, 64, dtype=BF16), _rand(g, 64, 72, dtype=BF16)
    dA, dB, db, dR = la.gemm_grad(dY, A, B, need_bias=True, need_residual=True)
    xA, eA, xB, eB, xb, eb = _grad64(dY, A, B, None, None, 1.0, 1.0)
    check(dA, xA, eA, "dA", 72)
    check(dB, xB, eB, "dB", 130)
    check(db, xb, eb, "db", 130)
    assert torch.equal(dR, dY)


@pytest.mark.parametrize("dtype", TYPES)
def test_non_finite_values_stay_in_their_rows(dtype):
    g = _gen(8)
    for M, K, N in [(3, 64, 40), (140, 136, 72)]:
        A, B = _rand(g, M, K, dtype=dtype), _rand(g, K, N, dtype=dtype)
        clean = la.gemm(A, B)
        A2 = A.clone()
        A2[1, 5], A2[2, 7] = float("nan"), float("inf")
        Y = la.gemm(A2, B)
        assert bool(torch.isnan(Y[1]).all()) and not bool(torch.isfinite(Y[2]).any())
        rest = [r for r in range(M) if r not in (1, 2)]
        assert torch.equal(Y[rest], clean[rest])


@pytest.mark.parametrize("dtype", TYPES)
def test_repeats_bit_for_bit(dtype):
    for M, K, N in [(1, 4096, 512), (16, 2048, 512), (300, 1000, 200)]:
        A, B, bias, R = _problem(M, K, N, dtype)
        a = la.gemm(A, B, bias, "gelu", R)
        for _ in range(3):
            assert torch.equal(a, la.gemm(A, B, bias, "gelu", R))
    dY, pre = _rand(_gen(1), 700, 96, dtype=dtype), _rand(_gen(2), 700, 96, dtype=dtype)
    A, B, _, _ = _problem(700, 64, 96, dtype)
    first = la.gemm_grad(dY, A, B, pre, "silu", need_bias=True)
    again = la.gemm_grad(dY, A, B, pre, "silu", need_bias=True)
    assert all(torch.equal(x, y) for x, y in zip(first[:3], again[:3]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", [(1, 512, 300), (33, 129, 65), (256, 512, 128)])
def test_on_another_stream_and_in_a_graph(M, K, N, dtype):
    A, B, bias, R = _problem(M, K, N, dtype, trans_b=True)
    want = la.gemm(A, B, bias, "silu", R)
    gw = la.gemm_grad(R, A, B, want, "silu", need_bias=True)[:3]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = la.gemm(A, B, bias, "silu", R)
    s.synchronize()
    assert torch.equal(got, want)
    graphs, outs = [], []
    for _ in range(2):  # two graphs with their own workspaces
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = la.gemm(A, B, bias, "silu", R)
            outs.append((y,) + la.gemm_grad(R, A, B, want, "silu", need_bias=True)[:3])
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(x, y) for x, y in zip(o, (want,) + gw))
    keep = A.clone()
    A.mul_(2)  # a replay reads what the operands hold then
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0][0], la.gemm(A, B, bias, "silu", R))
    A.copy_(keep)


def test_host_inputs():
    r = np.random.default_rng(0)
    A, B, b = (r.standard_normal(s).astype(np.float32) for s in [(2, 30, 40), (40, 50), (50,)])
    Y = la.gemm(A, B, b, "relu")
    assert isinstance(Y, np.ndarray) and Y.dtype == np.float32
    y, _, ey, _ = gemm64(torch.from_numpy(A), torch.from_numpy(B), torch.from_numpy(b), "relu")
    check(torch.from_numpy(Y), y, ey, "numpy", 40)
    T = la.gemm(torch.from_numpy(A), torch.from_numpy(B), torch.from_numpy(b), "relu")
    assert not T.is_cuda and np.array_equal(T.numpy(), Y)
    I = la.gemm(np.arange(6).reshape(2, 3), np.arange(6).reshape(3, 2))  # cast to float32 like everywhere here
    assert np.array_equal(I, (np.arange(6).reshape(2, 3) @ np.arange(6).reshape(3, 2)).astype(np.float32))
    outs = la.gemm_grad(Y, A, B, Y, "relu", need_bias=True)
    assert isinstance(outs[0], np.ndarray) and outs[0].shape == A.shape and outs[2].shape == (50,)


def test_residual_in_place_of_its_own_result_is_untouched():
    """Inputs are never written."""
    g = _gen(4)
    A, B, R = (_rand(g, *s, dtype=BF16) for s in [(130, 64), (64, 72), (130, 72)])
    keep = [t.clone() for t in (A, B, R)]
    la.gemm(A, B, None, None, R)
    la.gemm_grad(R, A, B, R, "gelu", need_bias=True, need_residual=True)
    assert all(torch.equal(x, y) for x, y in zip((A, B, R), keep))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_training_step(dtype):
    """Forward, gradients and the orthogonalised update of two layers together, against the same chain in 64 bits."""
    from tests._exact import orth64

    g = _gen(21)
    x, t = _rand(g, 96, 40, dtype=dtype), _rand(g, 96, 24, dtype=dtype)
    W1, W2 = _rand(g, 64, 40, dtype=dtype, scale=0.15), _rand(g, 24, 64, dtype=dtype, scale=0.15)
    b1 = _rand(g, 64, dtype=dtype, scale=0.1)
    h, pre = la.gemm(x, W1.mT, b1, "gelu", return_pre=True)
    d = la.gemm(h, W2.mT, None, None, t, beta=-1.0)  # prediction - target
    dh, dW2, _, _ = la.gemm_grad(d, h, W2.mT)
    dx, dW1, db1, _ = la.gemm_grad(dh, x, W1.mT, pre, "gelu", need_bias=True)
    u1, u2 = la.orthogonalize(dW1.mT), la.orthogonalize(dW2.mT)

    P = [v.double().requires_grad_(True) for v in (W1, b1, W2, x)]
    hh = act64(P[3] @ P[0].mT + P[1], "gelu")
    loss = 0.5 * (hh @ P[2].mT - t.double()).square().sum()
    grads = torch.autograd.grad(loss, P)
    # h, d, dh and dP are each rounded once before the gradients, whose own rounding comes last: five roundings
    tol = 5 * HALF[dtype] + 2.0**-23 * 64
    for got, want in zip((dW1.mT, db1, dW2.mT, dx), grads):
        assert float(torch.linalg.vector_norm(got.double() - want) / torch.linalg.vector_norm(want)) <= tol
    # the update is the orthogonalisation of the gradient that came out
    from tests._exact import MUON, orth_bound
    for u, dW in ((u1, dW1.mT), (u2, dW2.mT)):
        ref, its = orth64(dW)
        unit = 2.0**-12 if dtype == BF16 else 2.0**-23
        bound = orth_bound([x[None] for x in its], 5, MUON, unit, dtype)
        assert float(torch.linalg.matrix_norm(u.double() - ref)) <= float(bound)


@pytest.mark.parametrize("K", [8, 64])
def test_offsets_beyond_32_bits(K):
    """More outputs than 31 bits count, by the FP32 units and by the tensor cores, and the epilogue's gradient on them."""
    M, N = 70001, 31000
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    g = _gen(K)
    A, B = _rand(g, M, K, dtype=BF16), _rand(g, K, N, dtype=BF16, scale=1 / math.sqrt(K))
    Y, pre = la.gemm(A, B, None, "gelu", return_pre=True)
    rows = torch.tensor([0, 1, 34000, 69270, 69273, 69999, 70000], device=DEV)
    y, p, ey, ep = gemm64(A[rows], B, None, "gelu")
    check(pre[rows], p, ep, "pre", K)
    check(Y[rows], y, ey, "Y", K)
    dA = la.gemm_grad(Y, A, B, pre, "gelu")[0]
    # the same rows alone: every sum runs over N in an order that the sizes choose, so up to its own rounding
    ref = la.gemm_grad(Y[rows], A[rows], B, pre[rows], "gelu")[0].double()
    rel = float((dA[rows].double() - ref).norm() / ref.norm())
    assert rel <= 2 * (2.0**-8 + 2.0**-23 * (math.sqrt(N) + 32))


@pytest.mark.parametrize("M", [2, 4, 11])
def test_thin_products_of_long_streams(M):
    """Weights that no cache holds, read as they lie and transposed."""
    g = _gen(M)
    A, W = _rand(g, M, 5300), _rand(g, 5200, 5300, scale=1 / math.sqrt(5300))
    for B in (W.mT, _rand(g, 5300, 5200, scale=1 / math.sqrt(5300))):
        check(la.gemm(A, B), *_plain(A, B), what="Y", K=5300)
