"""Newton-Schulz orthogonalisation (csrc/orth.hip, muon.orthogonalize) against the iteration in 64 bits.

Tolerance, by arithmetic, in the Frobenius norm F.  With X = U diag(s) V^T the step is the odd polynomial
p(s) = a s + b s^3 + c s^5 of the singular values; its derivative maps the (i, j) entry of an error in
the singular bases by divided differences of p and by (p(si) + p(sj)) / (si + sj), so it grows an error
by at most L = max |p'| over the interval the values lie in (the second kind is bounded by max p(s)/s <= a).
A step's own roundings: an entry of a K-term product passes at most K fp32 additions, each off by at most
2^-24 times a partial sum <= |x_i| |y_j|; the roundings are independent, so their root mean square is below
sqrt(K) 2^-24 |x_i| |y_j| and the product's F error below sqrt(K) 2^-24 F(X) F(Y).  The dropped lo lo^T and
the two halves' roundings are 2^-24 of an operand each: added as 3 more.  Through B = b A + c A A and
X' = a X + B X (S = the largest singular value):
  e_A = r(n) F(X)^2,  e_B = |b| e_A + |c| (2 S^2 e_A + r(m) F(A)^2) + 3 u F(B),
  e_X = e_B S + r(m) F(B) F(X) + 4 u F(X'),     r(K) = (sqrt(K) + 3) u,  u = 2^-24.
The error at the end is the sum of the steps' errors, each grown by the later steps' L; the result's store adds
half a step of its type, relative."""
import math

import pytest
import torch

from regcn_amd import muon

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF_STEP = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
U = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def reference(G, steps=5, coeffs=muon.COEFFS, eps=1e-7):
    """(result in 64 bits, tolerance in the Frobenius norm before the store's rounding)."""
    a, b, c = coeffs
    X = G.detach().double()
    flip = X.shape[0] > X.shape[1]
    if flip:
        X = X.t().contiguous()
    X = X / (X.norm() + eps)
    m, n = X.shape
    r = lambda k: (math.sqrt(k) + 3) * U  # noqa: E731
    err = 2 * U * float(X.norm())
    for _ in range(steps):
        A = X @ X.t().contiguous()
        S = float(torch.linalg.eigvalsh(A)[-1].clamp(min=0).sqrt())
        B = b * A + c * (A @ A)
        Y = a * X + B @ X
        fx, fa, fb = float(X.norm()), float(A.norm()), float(B.norm())
        e_a = r(n) * fx * fx
        e_b = abs(b) * e_a + abs(c) * (2 * S * S * e_a + r(m) * fa * fa) + 3 * U * fb
        e_x = e_b * S + r(m) * fb * fx + 4 * U * float(Y.norm())
        s = torch.linspace(0, S * 1.001 + 1e-6, 4097, dtype=torch.float64)
        L = max(float((a + 3 * b * s ** 2 + 5 * c * s ** 4).abs().max()), float((a + b * s ** 2 + c * s ** 4).abs().max()))
        err = L * err + e_x
        X = Y
    return (X.t() if flip else X), err


def check(out, G, **kw):
    ref, tol = reference(G, **kw)
    assert out.shape == G.shape and out.dtype == G.dtype
    tol += HALF_STEP[G.dtype] * 1.01 * float(ref.norm()) + (2.0 ** -25 * math.sqrt(G.numel()) if G.dtype == F16 else 0.0)
    off = float((out.double() - ref).norm())
    assert off <= tol, "off by %.3g of %.3g, allowed %.3g" % (off, float(ref.norm()), tol)


def matrix(m, n, seed, dt=F32, kind="flat"):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(m, n, generator=gen)
    if kind == "decay":
        r = max(1, min(m, n) // 16)
        x = 0.05 * x + torch.randn(m, r, generator=gen) @ torch.randn(r, n, generator=gen) / math.sqrt(r)
    return (x * 1e-2).to(DEV).to(dt)


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("m,n,kind", [
    (1, 1, "flat"), (1, 7, "flat"), (7, 1, "flat"), (2, 2, "flat"), (31, 33, "decay"), (64, 64, "flat"), (65, 63, "decay"),
    (128, 200, "flat"), (200, 200, "decay"), (100, 200, "flat"), (600, 400, "decay"), (33, 1000, "flat"),
    (3000, 3, "flat"), (129, 8193, "decay"), (200, 10000, "flat")])
def test_sizes(m, n, kind, dt):
    G = matrix(m, n, m + n, dt, kind)
    out = muon.orthogonalize(G)
    check(out, G)
    assert torch.equal(out, muon.orthogonalize(G))  # the same bits on every call


@pytest.mark.parametrize("m,n", [(1700, 1701), (1921, 1600), (129, 30011), (3585, 3500), (500, 28001), (2305, 2700)])
def test_wide_tiles(m, n):
    """From 192 tiles of 128, and of 256, on: ragged sides, both orientations, k in pieces, a cut last round."""
    for kind in ("flat", "decay"):
        G = matrix(m, n, 3, F32, kind)
        check(muon.orthogonalize(G), G)


@pytest.mark.parametrize("m,n", [(1, 300000), (3, 30), (64, 1024), (32, 100003), (50001, 64), (65, 40000), (40000, 128)])
def test_few_rows(m, n):
    """Up to 64 rows (held in fp32) and just above, however long they are; a set that holds both."""
    G = [matrix(m, n, s) for s in (1, 2)] + [matrix(100, 90, 3)]
    together = muon.orthogonalize(G)
    for g, o in zip(G, together):
        check(o, g)
        assert torch.equal(o, muon.orthogonalize(g))


@pytest.mark.parametrize("steps,coeffs", [(1, muon.COEFFS), (2, muon.COEFFS), (8, muon.COEFFS), (5, (1.5, -0.5, 0.0)),
                                          (12, (1.875, -1.25, 0.375))])
def test_steps_and_coefficients(steps, coeffs):
    for m, n in ((40, 90), (70, 70)):
        G = matrix(m, n, 7)
        check(muon.orthogonalize(G, steps=steps, coeffs=coeffs), G, steps=steps, coeffs=coeffs)


def test_singular_values_end_near_one():
    G = matrix(150, 320, 1, kind="decay")
    s = torch.linalg.svdvals(muon.orthogonalize(G, steps=8).double().cpu())
    assert 0.6 < float(s.min()) and float(s.max()) < 1.3


def test_lists_stacks_and_views():
    """Any number of shapes, types and layouts in one call give what each gives alone, bit for bit."""
    mats = [matrix(5 + 13 * (k % 7), 200 - 27 * (k % 6), k, (F32, BF16, F16)[k % 3]) for k in range(70)]
    mats += [matrix(1700, 1700, 1), matrix(48, 96, 2).t(), matrix(300, 40, 3)[::2, 1:33], torch.zeros(0, 4, device=DEV)]
    outs = muon.orthogonalize(mats)
    assert isinstance(outs, list) and len(outs) == len(mats)
    for g, o in zip(mats, outs):
        assert o.shape == g.shape and o.dtype == g.dtype
        assert torch.equal(o, muon.orthogonalize(g.contiguous()))
    check(outs[71], mats[71])
    assert isinstance(muon.orthogonalize(tuple(mats[:2])), tuple)
    assert muon.orthogonalize([]) == []
    stack = torch.stack([matrix(24, 50, k) for k in range(6)]).view(2, 3, 24, 50)
    got = muon.orthogonalize(stack)
    for i in range(2):
        for j in range(3):
            assert torch.equal(got[i, j], muon.orthogonalize(stack[i, j]))
    assert muon.orthogonalize(stack[:0]).shape == (0, 3, 24, 50)


@pytest.mark.parametrize("scale", [1e-5, 1e30, 1e-38])
def test_range_of_the_input(scale):
    """The norm is taken in 64 bits: the squares of large and small entries are kept."""
    G = matrix(60, 80, 4) * (100.0 * scale)
    assert bool(torch.isfinite(G).all())
    check(muon.orthogonalize(G, eps=0.0), G, eps=0.0)


def test_norm_past_the_range_of_fp32():
    """Finite entries whose norm is not an fp32 number."""
    for m, n in ((60, 80), (300, 200)):
        G = matrix(m, n, 5) * 1e38 * 40.0
        assert bool(torch.isfinite(G).all())
        assert float(G.double().norm()) > 3.5e38
        check(muon.orthogonalize(G), G)


def test_zero_and_not_finite():
    zero = torch.zeros(70, 30, device=DEV)
    bad = matrix(40, 40, 1).clone()
    bad[3, 4] = float("nan")
    inf = matrix(40, 50, 2).clone()
    inf[0, 0] = float("inf")
    good = matrix(40, 60, 3)
    z, b, i, g = muon.orthogonalize([zero, bad, inf, good])
    assert not bool(z.any())
    assert bool(b.isnan().all()) and bool(i.isnan().any())
    assert torch.equal(g, muon.orthogonalize(good))


def test_second_stream_and_replays():
    mats = [[matrix(200, 200, k), matrix(600, 400, 10 + k), matrix(200, 5000, 20 + k)] for k in range(2)]
    want = [muon.orthogonalize(m) for m in mats]
    torch.cuda.synchronize()
    side, graphs = torch.cuda.Stream(), []
    for m in mats:
        with torch.cuda.stream(side):
            outs = muon.orthogonalize(m)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = muon.orthogonalize(m)
        graphs.append((graph, outs))
    for _ in range(3):
        for (graph, outs), w in zip(graphs, want):
            for o in outs:
                o.zero_()
            torch.cuda.synchronize()
            graph.replay()
            muon.orthogonalize(mats[0][0])
            torch.cuda.synchronize()
            assert all(torch.equal(o, x) for o, x in zip(outs, w))
