"""Newton-Schulz orthogonalisation against the iteration in 64 bits."""

import numpy as np
import pytest
import torch

import mlx_addons_b200.linalg as la
from tests._exact import MUON, orth64, orth_bound

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]
DEV = "cuda:0"
# half a step of the factors inside: pairs of 11-bit halves, or one
UNIT = {F32: 2.0**-23, F16: 2.0**-23, BF16: 2.0**-12}


@pytest.fixture(autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _grad_like(shape, dtype, seed=0, scale=1e-3):
    """A few strong directions over a broad floor."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    *lead, m, n = shape
    r = min(4, m, n)
    u, v = torch.randn(*lead, m, r, generator=g, device=DEV), torch.randn(*lead, r, n, generator=g, device=DEV)
    return (scale * (torch.randn(*lead, m, n, generator=g, device=DEV) + torch.matmul(u, v))).to(dtype)


def _check(out, G, steps=5, coefficients=MUON, eps=1e-7):
    assert out.shape == G.shape and out.dtype == G.dtype and out.device == G.device
    ref, its = orth64(G, steps, coefficients, eps)
    flat = lambda t: t.reshape((-1,) + tuple(t.shape[-2:]))  # noqa: E731
    o, r, its = flat(out.double()), flat(ref), [flat(x) for x in its]
    bound = orth_bound(its, steps, coefficients, UNIT[G.dtype], G.dtype)
    err = torch.linalg.matrix_norm(o - r)
    assert bool((err <= bound).all()), (float((err / bound).max()), float(err.max()), float(bound.max()))


SHAPES = [(1, 1), (1, 7), (7, 1), (2, 2), (3, 5), (16, 16), (17, 33), (31, 64), (33, 31), (64, 64), (64, 65), (65, 64),
          (100, 20), (128, 128), (128, 129), (129, 128), (128, 512), (512, 128), (200, 136), (257, 300), (300, 1000),
          (1, 3000), (3001, 2), (520, 64), (40, 1024), (700, 100), (128, 640), (128, 320), (321, 120), (257, 64), (50, 256)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n", SHAPES)
def test_shapes(m, n, dtype):
    G = _grad_like((m, n), dtype, seed=m + n)
    _check(la.orthogonalize(G), G)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(3, 64, 64), (2, 3, 20, 48), (5, 130, 70), (4, 64, 256), (1, 16, 16), (300, 8, 8),
                                   (7, 128, 128), (3, 136, 264)])
def test_batches_have_their_own_norms(shape, dtype):
    G = _grad_like(shape, dtype, seed=1)
    k = torch.logspace(-3, 2, shape[0], device=DEV).reshape((-1,) + (1,) * (len(shape) - 1)).to(dtype)
    G = G * k
    _check(la.orthogonalize(G), G)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n", [(48, 64), (64, 48), (150, 260), (260, 150)])
def test_strides(m, n, dtype):
    G = _grad_like((n, m), dtype, seed=2).mT
    _check(la.orthogonalize(G), G)
    G = _grad_like((2 * m, 2 * n + 3), dtype, seed=3)[1::2, 3::2]
    _check(la.orthogonalize(G), G)
    G = _grad_like((m, 3, n), dtype, seed=4).permute(1, 0, 2)
    _check(la.orthogonalize(G), G)
    G = _grad_like((1, m, n), dtype, seed=5).expand(3, m, n)
    out = la.orthogonalize(G)
    _check(out, G)
    assert torch.equal(out[0], out[2])


@pytest.mark.parametrize("m,n", [(20, 30), (64, 64), (140, 200)])
@pytest.mark.parametrize("steps,coefficients", [(1, MUON), (2, MUON), (10, (1.875, -1.25, 0.375)), (12, (1.5, -0.5, 0.0)),
                                                (3, [(3.0, -3.2, 1.2), (2.5, -2.0, 0.5), (1.875, -1.25, 0.375)])])
def test_coefficients(m, n, steps, coefficients):
    G = _grad_like((m, n), F32, seed=6)
    _check(la.orthogonalize(G, steps=steps, coefficients=coefficients), G, steps, coefficients)


def test_converges_to_the_polar_factor():
    """Twenty steps of the convergent quintic leave X X^T = I to the accuracy of the factors."""
    for m, n in [(24, 40), (64, 64), (150, 170)]:
        g = torch.Generator(device=DEV).manual_seed(m)
        G = torch.randn(m, n, generator=g, device=DEV) + (2 * torch.eye(m, n, device=DEV) * n**0.5)
        X = la.orthogonalize(G, steps=20, coefficients=(1.875, -1.25, 0.375)).double()
        U, _, Vt = torch.linalg.svd(G.double(), full_matrices=False)
        # a step's own roundings, 6.5 u sqrt(m) of the Frobenius norm (the terms of _exact.orth_bound at singular
        # values of 1); earlier ones are carried along with a factor of at most the ratio of G's singular values (< 5)
        u = 2.0**-22 + 2.0**-23 * (n**0.5 + 32)
        assert float(torch.linalg.matrix_norm(X - U @ Vt)) <= 20 * 6.5 * u * m**0.5 * 5


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n", [(16, 24), (64, 64), (140, 200)])
def test_zeros_and_non_finite(m, n, dtype):
    G = _grad_like((5, m, n), dtype, seed=8)
    clean = la.orthogonalize(G)
    G2 = G.clone()
    G2[1] = 0
    G2[2, 3, 4] = float("nan")
    G2[3, 0, 1] = float("inf")
    out = la.orthogonalize(G2)
    assert torch.equal(out[0], clean[0]) and torch.equal(out[4], clean[4])
    assert float(out[1].abs().max()) == 0.0
    assert bool(torch.isnan(out[2]).all()) and bool(torch.isnan(out[3]).all())


@pytest.mark.parametrize("m,n", [(24, 16), (150, 140)])
def test_norms_beyond_the_range_of_a_float32_square(m, n):
    """|G|_F^2 over- or underflows float32; the norm does not."""
    for scale in (1e-30, 1e30):
        G = _grad_like((m, n), F32, seed=9, scale=scale)
        _check(la.orthogonalize(G, eps=0.0), G, eps=0.0)
    G = _grad_like((m, n), BF16, seed=9, scale=1e30)
    _check(la.orthogonalize(G), G)
    tiny = _grad_like((m, n), F32, seed=9, scale=1e-12)  # eps counts
    _check(la.orthogonalize(tiny, eps=1e-7), tiny, eps=1e-7)


@pytest.mark.parametrize("dtype", TYPES)
def test_rank_one_keeps_its_direction(dtype):
    u, v = torch.randn(150, device=DEV, dtype=torch.float64), torch.randn(190, device=DEV, dtype=torch.float64)
    u, v = u / u.norm(), v / v.norm()
    G = torch.outer(u, v).to(dtype)
    _check(la.orthogonalize(G), G)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(40, 64, 64), (96, 160), (3, 200, 300)])
def test_graphs_streams_and_repeats(shape, dtype):
    G = _grad_like(shape, dtype, seed=10)
    want = la.orthogonalize(G)
    keep = G.clone()
    for _ in range(3):
        assert torch.equal(want, la.orthogonalize(G))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = la.orthogonalize(G)
    s.synchronize()
    assert torch.equal(want, got)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = la.orthogonalize(G)
        graphs.append((g, o))
    for _ in range(2):
        for g, _ in graphs:
            g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for _, o in graphs)
    assert torch.equal(G, keep)
    G.copy_(G.flip(0))
    graphs[1][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[1][1], la.orthogonalize(G))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,m,n", [(1000, 32, 40), (700, 20, 96), (2000, 64, 64), (900, 40, 33), (640, 100, 128),
                                       (5000, 5, 5), (4096, 1, 9), (1300, 16, 16), (600, 128, 100), (700, 72, 200)])
def test_batches_that_share_a_tile(batch, m, n, dtype):
    """Several matrices stacked in one CTA keep apart, a broken one among them."""
    G = _grad_like((batch, m, n), dtype, seed=m)
    G = G * torch.logspace(-2, 2, batch, device=DEV).reshape(-1, 1, 1).to(dtype)
    out = la.orthogonalize(G)
    _check(out, G)
    G2 = G.clone()
    G2[1, 0, 0], G2[batch - 2, m - 1, n - 1] = float("nan"), float("-inf")
    out2 = la.orthogonalize(G2)
    keep = torch.ones(batch, dtype=torch.bool, device=DEV)
    keep[1] = keep[batch - 2] = False
    assert torch.equal(out2[keep], out[keep]) and bool(torch.isnan(out2[~keep]).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 129, 129), (1, 256, 256), (1, 1000, 517), (3, 517, 1000), (2, 130, 1500), (1, 700, 2000),
                                   (5, 384, 384), (1, 2048, 640), (40, 200, 260), (300, 140, 136), (2, 2100, 2300)])
def test_middle_sizes(shape, dtype):
    """The sizes between one CTA's shared memory and the largest, on both sides of each border."""
    G = _grad_like(shape, dtype, seed=sum(shape))
    out = la.orthogonalize(G)
    if dtype == F32:  # 64-bit values of the large ones once
        _check(out, G)
    else:
        ref, its = orth64(G)
        err, bound = torch.linalg.matrix_norm(out.double() - ref), orth_bound(its, 5, MUON, UNIT[dtype], dtype)
        assert bool((err <= bound).all()), float((err / bound).max())
    again = la.orthogonalize(G)
    assert torch.equal(out, again)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,m,n", [(1, 128, 513), (1, 64, 300), (2, 20, 1500), (5, 1469, 38), (1, 1, 2000), (3, 100, 1536),
                                       (1, 128, 1537), (400, 20, 700), (300, 33, 600), (160, 600, 64), (20, 16, 2560)])
def test_a_long_side(batch, m, n, dtype):
    """Matrices shared by a cluster of CTAs, alone and stacked, transposed and with a broken one among them."""
    G = _grad_like((batch, m, n), dtype, seed=m + 1)
    G = G * torch.logspace(-2, 2, batch, device=DEV).reshape(-1, 1, 1).to(dtype)
    out = la.orthogonalize(G)
    _check(out, G)
    _check(la.orthogonalize(G.mT.contiguous().mT), G)
    assert all(torch.equal(la.orthogonalize(G), out) for _ in range(3))
    if batch > 2:
        G2 = G.clone()
        G2[1, m - 1, n - 1], G2[batch - 1, 0, 0] = float("nan"), float("inf")
        out2 = la.orthogonalize(G2)
        keep = torch.ones(batch, dtype=torch.bool, device=DEV)
        keep[1] = keep[batch - 1] = False
        assert torch.equal(out2[keep], out[keep]) and bool(torch.isnan(out2[~keep]).all())


def test_two_streams_at_once():
    """Calls that need every SM together, side by side on two streams."""
    G = [_grad_like((3, 300 + 50 * i, 500), F32, seed=i) for i in range(2)]
    want = [la.orthogonalize(g) for g in G]
    streams = [torch.cuda.Stream() for _ in G]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(la.orthogonalize(G[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])


def test_host_inputs_and_empty():
    G = _grad_like((3, 20, 30), F32, seed=12)
    want = la.orthogonalize(G).cpu()
    out = la.orthogonalize(G.cpu().numpy())
    assert isinstance(out, np.ndarray) and np.array_equal(out, want.numpy())
    out = la.orthogonalize(G.cpu())
    assert not out.is_cuda and torch.equal(out, want)
    assert la.orthogonalize(torch.empty(0, 4, 5, device=DEV)).shape == (0, 4, 5)
    assert la.orthogonalize(torch.empty(3, 0, 5, device=DEV, dtype=BF16)).shape == (3, 0, 5)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_many_matrices(dtype):
    """More matrices than one axis of a launch grid holds."""
    G = _grad_like((70000, 4, 6), dtype, seed=13)
    out = la.orthogonalize(G)
    pick = torch.tensor([0, 1, 65534, 65535, 65536, 69999], device=DEV)
    _check(out[pick], G[pick])


def test_offsets_beyond_32_bits():
    """More elements than 31 bits count, in small matrices and in one of a product's tiles."""
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    G = torch.randn(540000, 64, 64, device=DEV, dtype=BF16)
    out = la.orthogonalize(G)
    pick = torch.tensor([0, 524287, 524288, 524289, 539999], device=DEV)
    _check(out[pick], G[pick])
    del out
    G = G.reshape(9000, 240, 1024)
    out = la.orthogonalize(G)
    pick = torch.tensor([0, 8737, 8738, 8999], device=DEV)
    _check(out[pick], G[pick])
