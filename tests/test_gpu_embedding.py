"""Embedding lookup and its gradient (csrc/lookup.hip) against plain 64-bit sums.

Tolerances, by arithmetic.  The lookup multiplies a row by the scale in fp32 and rounds once to the
table's type: torch's own fp32 product and cast give the same bits.  A gradient row is an fp32 sum of
at most 63 + 63 + 63 + k + 63 + 63 terms for a run of up to 4096 k tokens (its ends, block sums, group
sums), each term of which is itself a sum of 64 (64 * 64): along any path an element passes fewer than
D = 63 * 5 + k + 64 + 64 additions, so |error| <= D 2^-24 sum|g| |s|, one more rounding (2^-24) for the
product with the scale, and half a step of the type for the store (2^-8 bf16, 2^-11 fp16 relative;
2^-25 absolute for fp16's subnormals)."""
import numpy as np
import pytest
import torch

from regcn_amd import autograd as A

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF_STEP = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def tokens(V, n, seed, skew):
    rng = np.random.default_rng(seed)
    if skew == "one":
        return torch.full((n,), V - 1, dtype=torch.int64)
    if skew == "hubs":  # three rows take most tokens
        hub = rng.integers(0, V, 3)
        pick = rng.random(n) < 0.8
        return torch.from_numpy(np.where(pick, hub[rng.integers(0, 3, n)], rng.integers(0, V, n)))
    return torch.from_numpy(rng.integers(0, V, n))


def ref_grad(g, idx, V, scale, pad=None):
    """64-bit sums, and the sums of |g| that the tolerance scales with."""
    d = g.shape[-1]
    g, idx = g.reshape(-1, d).double().cpu(), idx.reshape(-1).long().cpu()
    ok = (idx >= 0) & (idx < V)
    if pad is not None:
        ok &= idx != pad
    out, mag = torch.zeros(V, d, dtype=torch.float64), torch.zeros(V, d, dtype=torch.float64)
    out.index_add_(0, idx[ok], g[ok])
    mag.index_add_(0, idx[ok], g[ok].abs())
    return out * scale, mag * abs(scale)


def check_grad(got, g, idx, scale, pad=None):
    V, dt = got.shape[0], got.dtype
    ref, mag = ref_grad(g, idx, V, scale, pad)
    depth = 63 * 5 + 128 + idx.numel() // 4096 + 2
    tol = depth * 2.0 ** -24 * mag + HALF_STEP[dt] * ref.abs() * 1.001 + (2.0 ** -25 if dt == F16 else 0.0)
    err = (got.double().cpu() - ref).abs()
    assert bool((err <= tol).all()), "max excess %.3g" % float((err - tol).max())


def both(table, idx, scale, pad=None, seed=0):
    t = table.detach().clone().requires_grad_(True)
    out = A.embedding(t, idx, scale, padding_idx=pad)
    gen = torch.Generator().manual_seed(seed)
    g = torch.randn(out.shape, generator=gen).to(DEV).to(table.dtype)
    grad = torch.autograd.grad(out, t, g)[0]
    return out.detach(), g, grad


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("V,d,n,skew", [
    (1, 1, 1, "flat"), (1, 200, 5, "one"), (3, 7, 64, "flat"), (7128, 200, 1, "flat"), (512, 200, 3080, "flat"),
    (10007, 333, 4999, "hubs"), (50, 4, 65, "one"), (50, 8, 4095, "one"), (50, 36, 4097, "one"), (2, 1025, 130, "flat"),
    (999, 1, 8193, "hubs"), (1024, 24, 16384, "hubs"), (1023, 24, 16385, "hubs"), (1 << 20, 12, 20001, "flat"),
    (70000, 40, 70001, "hubs"), (5, 3, 300007, "flat"), (6, 16, 262145, "one")])
def test_forward_and_gradient(V, d, n, skew, dt):
    gen = torch.Generator().manual_seed(V + d + n)
    table = torch.randn(V, d, generator=gen).to(DEV).to(dt)
    idx = tokens(V, n, n, skew).to(DEV)
    out, g, grad = both(table, idx, 1.75)
    assert torch.equal(out, (table[idx].float() * 1.75).to(dt))
    check_grad(grad, g, idx, 1.75)
    again = both(table, idx, 1.75)[2]
    assert torch.equal(again, grad)  # a fixed order: the same bits


@pytest.mark.parametrize("V", [600, 3000, 200000])
def test_int32_shapes_strides_padding(V):
    n = 20000 if V > 100000 else 900
    gen = torch.Generator().manual_seed(1)
    wide = torch.randn(V, 48, generator=gen).to(DEV)
    idx = tokens(V, n, 3, "hubs").to(torch.int32).to(DEV)
    want = None
    for table in (wide[:, :20].contiguous(), wide[:, :20], wide[:, 1:21]):  # packed, strided, off 16 bytes
        ref = table[idx.long()] * 0.5
        out = A.embedding(table, idx.view(-1, 4), 0.5)
        assert out.shape == (n // 4, 4, 20)
        assert torch.equal(out.view(n, 20), ref)
    cols = wide.t()[:20].t()  # the same columns, made of a transposed view
    assert torch.equal(A.embedding(cols.t().contiguous().t(), idx, 0.5), wide[:, :20][idx.long()] * 0.5)
    every = torch.stack([idx, idx], 1)[:, 0]  # strided indices
    assert torch.equal(A.embedding(wide, every), wide[idx.long()])
    pad = int(idx[0])
    for p in (pad, pad - V):
        out, g, grad = both(wide[:, :20].contiguous(), idx, -2.0, pad=p)
        check_grad(grad, g, idx, -2.0, pad=pad)
        assert float(grad[pad].abs().max()) == 0.0
        want = grad if want is None else want
        assert torch.equal(grad, want)


@pytest.mark.parametrize("V,d,dt", [(40000, 333, F16), (70001, 100, F32), (9001, 1024, F32), (131, 70000, F32), (5, 1000001, F32),
                                    (3, 2000001, BF16), (600000, 7, F32), (4500000, 1, F32), (33, 64, BF16), (1000, 4, F32)])
def test_every_row_is_written_once(V, d, dt):
    """Outputs below and above the caches, rows that are whole 128-byte lines and rows that are not; small whole numbers,
    so that each sum is exact in the type: at most 4 in absolute value, 255 / 4 of a row's tokens at the most."""
    rng = np.random.default_rng(V + d)
    n = 60 if d > 10000 else 3000
    idx = torch.from_numpy(np.minimum(rng.zipf(1.3, n) - 1, V - 1))
    idx[torch.bincount(idx, minlength=V)[idx] > 60] = -1  # rows that would pass 240 take nothing
    g = torch.from_numpy(rng.integers(-4, 5, (n, d))).to(dt)
    table = torch.empty(V, d, device=DEV, dtype=dt).requires_grad_(True)
    out = A.embedding(table, idx.to(DEV))
    got, = torch.autograd.grad(out, table, g.to(DEV))
    want = torch.zeros(V, d)
    want.index_add_(0, idx[idx >= 0], g[idx >= 0].float())
    assert torch.equal(got.cpu().float(), want)


@pytest.mark.parametrize("n", [100, 17000])
def test_index_outside(n):
    """Rows that do not exist: a NaN output row, no gradient; the others are as without them."""
    V, d = 37, 12
    table = torch.randn(V, d, device=DEV)
    idx = tokens(V, n, 0, "flat").to(DEV)
    bad = torch.zeros(n, dtype=torch.bool, device=DEV)
    for j, v in ((3, -1), (40, V), (77, 1 << 40), (n - 1, -(1 << 40))):
        idx[j], bad[j] = v, True
    out, g, grad = both(table, idx, 3.0)
    assert bool(out[bad].isnan().all()) and torch.equal(out[~bad], table[idx[~bad]] * 3.0)
    check_grad(grad, g, idx, 3.0)


def test_nothing_to_do():
    table = torch.randn(5, 8, device=DEV, requires_grad=True)
    none = torch.zeros(0, 3, dtype=torch.int64, device=DEV)
    out = A.embedding(table, none)
    assert out.shape == (0, 3, 8)
    out.sum().backward()
    assert torch.equal(table.grad, torch.zeros_like(table))
    empty = torch.zeros(0, 8, device=DEV, requires_grad=True)
    assert A.embedding(empty, none).shape == (0, 3, 8)
    assert bool(A.embedding(empty.detach(), torch.zeros(2, dtype=torch.int64, device=DEV)).isnan().all())
    assert A.embedding(torch.zeros(4, 0, device=DEV), torch.zeros(2, dtype=torch.int64, device=DEV)).shape == (2, 0)


def test_values_that_are_not_numbers_stay_in_their_rows():
    table = torch.randn(6, 5, device=DEV)
    table[2, 1], table[3, 0] = float("inf"), float("nan")
    idx = torch.tensor([2, 3, 1, 2], device=DEV)
    assert torch.equal(A.embedding(table, idx).nan_to_num(7.0), table[idx].nan_to_num(7.0))
    t = table.requires_grad_(True)
    g = torch.ones(4, 5, device=DEV)
    g[1] = float("nan")
    grad = torch.autograd.grad(A.embedding(t, idx), t, g)[0]
    assert bool(grad[3].isnan().all())
    rest = grad[[0, 1, 2, 4, 5]]
    assert torch.equal(rest, torch.tensor([0., 1., 2., 0., 0.], device=DEV)[:, None].expand(5, 5))


def test_gradient_against_differences():
    """Central differences of a smooth function of the looked-up rows, in 64 bits on the host: the
    gradient of sum f(s T[idx]) with f = sin.  cos has curvature <= 1: the difference quotient is off by
    h^2 s^3 / 6 per token, the fp32 gradient by the rounding of cos and of a sum of <= 9 terms."""
    V, d, n, s, h = 7, 3, 9, 0.5, 1e-4
    gen = torch.Generator().manual_seed(5)
    table = torch.randn(V, d, generator=gen)
    idx = torch.tensor([0, 1, 1, 6, 6, 6, 2, 0, 6])
    t = table.to(DEV).requires_grad_(True)
    torch.sin(A.embedding(t, idx.to(DEV), s)).sum().backward()
    f = lambda x: torch.sin(s * x[idx]).sum()  # noqa: E731
    for v in range(V):
        for j in range(d):
            e = torch.zeros(V, d, dtype=torch.float64)
            e[v, j] = h
            diff = (f(table.double() + e) - f(table.double() - e)) / (2 * h)
            assert abs(float(diff) - float(t.grad[v, j])) <= 9 * (h * h / 6 + 4 * 2.0 ** -23) + 1e-11 / h


def test_gradient_of_the_gradient():
    """grad(table) is linear in the output's gradient g: with f = sum(grad^2) / 2, df/dg_i = s grad[idx_i],
    0 for a token left out.  Each side is one fp32 product of the same fp32 row."""
    V, d = 11, 6
    table = torch.randn(V, d, device=DEV, requires_grad=True)
    idx = torch.tensor([1, 4, 4, 0, 10, 10, 10, V, 3], device=DEV)
    g = torch.randn(9, d, device=DEV, requires_grad=True)
    out = A.embedding(table, idx, 0.5, padding_idx=3)
    grad, = torch.autograd.grad(out, table, g, create_graph=True)
    dg, = torch.autograd.grad((grad * grad).sum() * 0.5, g)
    keep = ((idx < V) & (idx != 3)).unsqueeze(1)
    want = torch.where(keep, 0.5 * grad.detach()[idx.clamp(max=V - 1)], torch.zeros((), device=DEV))
    assert torch.equal(dg, want)


def test_second_stream_and_broadcast_gradient():
    table = torch.randn(300, 64, device=DEV, requires_grad=True)
    idx = tokens(300, 5000, 2, "hubs").to(DEV)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        out = A.embedding(table, idx, 2.0)
        out.sum().backward()  # the gradient of every output element is one expanded 1
    side.synchronize()
    assert torch.equal(out.detach(), table.detach()[idx] * 2.0)
    count = torch.bincount(idx, minlength=300).float() * 2.0
    assert torch.equal(table.grad, count[:, None].expand(300, 64))  # small whole numbers: exact sums


@pytest.mark.parametrize("n", [3000, 20000])
def test_captured_and_replayed(n):
    """Two captured graphs of forward and gradient with their own workspaces, replayed in turn with eager
    work between, give the eager bits on every replay."""
    V, d = 4000, 52
    data = []
    side = torch.cuda.Stream()
    for k in range(2):
        table = torch.randn(V, d, device=DEV).requires_grad_(True)
        idx = tokens(V, n, k, "hubs").to(DEV)
        g = torch.randn(n, d, device=DEV)
        with torch.cuda.stream(side):
            out = A.embedding(table, idx, 1.5)
            grad = torch.autograd.grad(out, table, g)[0]
            eager = out.detach().clone(), grad
            del out
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = A.embedding(table, idx, 1.5)
            grad = torch.autograd.grad(out, table, g)[0]
        data.append((graph, out.detach(), grad, eager, (table, idx, g)))
    for _ in range(3):
        for graph, out, grad, eager, _keep in data:
            out.zero_(), grad.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.randn(1000, device=DEV).sum()
            torch.cuda.synchronize()
            assert torch.equal(out, eager[0]) and torch.equal(grad, eager[1])


def test_large_offsets():
    """Elements past 2^31 of a table: 9 M rows of 256 bf16 (4.6 GB)."""
    V, d = 9_000_001, 256
    table = torch.zeros(V, d, device=DEV, dtype=BF16)
    rows = torch.tensor([0, 8_388_607, 8_388_608, V - 1, V - 1], device=DEV)
    table[rows] = torch.randn(5, d, device=DEV).to(BF16)
    out, g, grad = both(table, rows, 1.0)
    assert torch.equal(out, table[rows])
    used = torch.unique(rows)
    ref, _ = ref_grad(g, torch.searchsorted(used, rows), len(used), 1.0)
    assert float((grad[used].double().cpu() - ref).abs().max()) <= 2.0 ** -8 * float(ref.abs().max())
    grad[used] = 0
    assert not bool(grad.any())


@pytest.mark.parametrize("d,dt", [(4_400_001, F32), (8_500_000, BF16)])
def test_rows_wider_than_a_launch_holds(d, dt):
    """More column slices than a launch's second dimension holds; whole numbers, so exact sums."""
    idx = torch.tensor([2] * 70 + [0] * 300 + [1], device=DEV)
    g = torch.randint(-1, 2, (len(idx), 1), device=DEV).to(dt)
    table = torch.zeros(3, d, device=DEV, dtype=dt, requires_grad=True)
    wide = torch.arange(d, device=DEV).remainder(3).sub(1).to(dt)
    wide[:300] = 0
    wide[-5:] = 1
    grad, = torch.autograd.grad(A.embedding(table, idx), table, g * wide)
    count = torch.zeros(3, device=DEV).index_add_(0, idx, g[:, 0].float())
    assert torch.equal(grad.float(), count[:, None] * wide.float())


def test_forward_mode():
    """The lookup is linear in the table and its gradient in g: their tangents are the same maps of the tangents."""
    from torch.autograd import forward_ad
    V, d = 30, 12
    table, tangent = torch.randn(V, d, device=DEV), torch.randn(V, d, device=DEV)
    idx = tokens(V, 50, 1, "flat").to(DEV)
    for t, v in ((table, tangent), (table.clone().requires_grad_(True), tangent), (table.t().contiguous().t(), tangent.t().contiguous().t())):
        with forward_ad.dual_level():
            out = A.embedding(forward_ad.make_dual(t, v), idx, 0.5)
            primal, got = forward_ad.unpack_dual(out)
            assert torch.equal(primal.detach(), table[idx] * 0.5)
            assert got is not None and torch.equal(got.detach(), tangent[idx] * 0.5)
            assert forward_ad.unpack_dual(A.embedding(table, idx)).tangent is None
    f = lambda t: A.embedding(t, idx, 0.5, padding_idx=3)  # noqa: E731
    out, got = torch.func.jvp(f, (table,), (tangent,))
    assert torch.equal(out, table[idx] * 0.5) and torch.equal(got, tangent[idx] * 0.5)
    g = torch.randn(50, d, device=DEV)
    leaf = table.clone().requires_grad_(True)
    want, = torch.autograd.grad(f(leaf), leaf, g)
    assert torch.equal(torch.func.vjp(f, table)[1](g)[0], want)
    assert torch.equal(torch.func.grad(lambda t: (f(t) * g).sum())(table), want)
    # forward over reverse: the gradient of sum(f(t)^3) / 3 along the tangent
    with forward_ad.dual_level():
        leaf = table.clone().requires_grad_(True)
        dual = forward_ad.make_dual(leaf, tangent)
        grad, = torch.autograd.grad((f(dual) ** 3).sum() / 3, leaf, create_graph=True)
        got = forward_ad.unpack_dual(grad).tangent
    y, dy = (table[idx] * 0.5).double(), (tangent[idx] * 0.5).double()
    check_grad(got.detach(), 2 * y * dy, idx, 0.5, pad=3)


def test_traced_launches():
    """Under a launch trace the entries are called from Python and show up; the results are the same bits."""
    from regcn_amd import _lib
    table, idx = torch.randn(40, 12, device=DEV), tokens(40, 70, 1, "flat").to(DEV)
    want = both(table, idx, 2.0)
    plain = A.embedding(table, idx, 2.0)
    _lib.EVENT_TRACE = []
    try:
        got = both(table, idx, 2.0)
        assert torch.equal(A.embedding(table, idx, 2.0), plain)
        names = [n for n, _ in _lib.EVENT_TRACE]
    finally:
        _lib.EVENT_TRACE = None
    assert names == ["regcn_embedding", "regcn_embedding_grad", "regcn_embedding"]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_leaves_views_and_modes():
    """The node's place in a graph: a result without one under no_grad, gradients into views and through two uses."""
    table, idx = torch.randn(40, 12, device=DEV, requires_grad=True), tokens(40, 70, 1, "flat").to(DEV)
    with torch.no_grad():
        assert A.embedding(table, idx).grad_fn is None
    with torch.inference_mode():
        assert torch.equal(A.embedding(table, idx), table[idx])
    assert not A.embedding(table.detach(), idx).requires_grad
    part = (table * 1.0)[3:30, 2:9]  # rows off 16 bytes, wider apart than long
    inside = idx.clamp(max=26)
    out = A.embedding(part, inside) + A.embedding(part, inside.flip(0), 2.0)
    g = torch.randint(-3, 4, out.shape, device=DEV).float()
    got, = torch.autograd.grad(out, table, g)
    ref = table.detach().clone().requires_grad_(True)
    want, = torch.autograd.grad(ref[3:30, 2:9][inside] + 2.0 * ref[3:30, 2:9][inside.flip(0)], ref, g)
    assert torch.equal(got, want)  # whole numbers: exact in any order
    seen = []
    hooked = A.embedding(table, idx)
    hooked.register_hook(lambda g: seen.append(g.shape))
    hooked.sum().backward()
    assert seen == [(70, 12)] and torch.equal(table.grad[:, 0], torch.bincount(idx, minlength=40).float())
