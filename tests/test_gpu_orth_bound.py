"""Orthogonalisation held to a small multiple of the error that fp32 products leave on the same input (tests/orth_model.py;
test_orth_bound.py shows what the bound sees), rows of very different sizes, and inputs that are not finite."""
import pytest
import torch

from orth_model import bound, error, graded, iterate
from regcn_amd import muon

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF_STEP = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def matrix(m, n, kind):
    gen = torch.Generator().manual_seed(m + n)
    x = torch.randn(m, n, generator=gen)
    if kind == "decay":
        r = max(1, min(m, n) // 16)
        x = 0.05 * x + torch.randn(m, r, generator=gen) @ torch.randn(r, n, generator=gen) / r ** 0.5
    return (x * 1e-2).to(DEV)


def check(G, steps=5, **kw):
    """The bound on the iteration, and half a step of the type for the store (the root mean square of a rounding is less;
    fp16's subnormals are 2^-25 apart, absolute)."""
    out = muon.orthogonalize(G, steps=steps, **kw)
    ref = iterate(G, steps)
    limit = bound(G, ref, steps) + 1.01 * HALF_STEP[G.dtype]
    if G.dtype == F16:
        limit += 2.0 ** -25 * G.numel() ** 0.5 / float(ref.norm())
    off = error(out, ref)
    assert off <= limit, "off by %.3g, allowed %.3g" % (off, limit)
    return out


# tiles of 64, of 128 with symmetric tiles of 64 and 128, of 256; k whole and in pieces; fp32 operands (up to 64 rows)
SIZES = [(3, 30), (64, 1024), (65, 63), (65, 66), (128, 200), (200, 200), (600, 400), (100, 5000), (200, 10000), (1333, 777),
         (1024, 4096), (1700, 1701), (129, 30011), (2305, 2700), (2900, 2900)]


@pytest.mark.parametrize("kind", ["flat", "decay"])
@pytest.mark.parametrize("m,n", SIZES)
def test_as_exact_as_fp32_products(m, n, kind):
    check(matrix(m, n, kind))


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("m,n", [(200, 200), (1333, 777), (300, 2000), (40, 3000)])
def test_16_bits_are_rounded_once(m, n, dt):
    check(matrix(m, n, "flat").to(dt))


@pytest.mark.parametrize("steps", [1, 2, 3, 8, 9, 12, 20])
@pytest.mark.parametrize("m,n", [(70, 70), (200, 300), (1700, 1701)])
def test_any_number_of_steps(m, n, steps):
    check(matrix(m, n, "flat"), steps)


@pytest.mark.parametrize("scale", [1e-2, 1e-4, 1e-6, 1e-8])
@pytest.mark.parametrize("steps", [5, 8, 9, 12, 16])
def test_rows_of_very_different_sizes(scale, steps):
    """Of the whole matrix; above 8 steps the small rows have grown, and fp32 operands keep them."""
    for m, n in ((100, 200), (300, 260)):
        check(graded(m, n, scale).to(DEV), steps)
    check(graded(200, 100, scale).to(DEV).t(), steps)


@pytest.mark.parametrize("scale", [1e-4, 1e-6, 1e-8])
@pytest.mark.parametrize("m,n", [(100, 200), (300, 260), (1700, 1900), (64, 300)])
def test_small_rows_on_fp32_operands(m, n, scale):
    """full_fp32: the small rows are as exact as the others.  Without it they keep what 2^-37 of the matrix's norm leaves: an
    entry is about scale / sqrt(m n / 2) of the norm, so 2^-37 sqrt(m n / 2) / scale relative to itself, twice that allowed for
    the operands A and B, which are held alike."""
    G = graded(m, n, scale).to(DEV)
    ref = iterate(G, 5)
    small, small_ref = slice(m // 2, None), ref[m // 2:]
    limit = max(4.0 * error(iterate(G, 5, dtype=F32)[small], small_ref), 2.0 ** -21)
    out = check(G, full_fp32=True)
    assert error(out[small], small_ref) <= limit
    out = check(G)
    kept = 0.0 if m <= 64 else 2 * 2.0 ** -37 * (m * n / 2) ** 0.5 / scale
    assert error(out[small], small_ref) <= limit + kept


@pytest.mark.parametrize("m,n", [(40, 50), (100, 90), (600, 400), (1600, 2000), (1700, 1701), (2900, 2900)])
def test_not_finite_and_zero(m, n):
    """On every tile size: an infinity or a NaN anywhere makes the whole result NaN, zeros stay zero (with an eps of 0: NaN),
    and the matrices beside them are as alone."""
    good = matrix(m, n, "flat")
    nan, inf = good.clone(), good.clone()
    nan[m - 1, n // 2] = float("nan")
    inf[m // 3, 0] = -float("inf")
    a, z, b, c = muon.orthogonalize([good, torch.zeros_like(good), nan, inf])
    assert torch.equal(a, muon.orthogonalize(good))
    assert not bool(z.any()) and bool(b.isnan().all()) and bool(c.isnan().all())
    assert bool(muon.orthogonalize(torch.zeros_like(good), eps=0.0).isnan().all())
    small = muon.orthogonalize(good * 1e-30, eps=0.0)  # the norm alone scales it
    ref = iterate(good * 1e-30, 5, eps=0.0)
    assert error(small, ref) <= bound(good * 1e-30, ref, 5, eps=0.0)


def test_muon_with_fp32_operands():
    p = torch.randn(100, 80, device=DEV).requires_grad_(True)
    start, grad = p.detach().clone(), graded(100, 80, 1e-6).to(DEV)
    steps = {}
    for full in (False, True):
        with torch.no_grad():
            p.copy_(start)
        opt = muon.Muon([p], lr=0.5, momentum=0.0, nesterov=False, full_fp32=full)
        p.grad = grad.clone()
        opt.step()
        steps[full] = start - p.detach()
    want = muon.orthogonalize(grad, full_fp32=True) * (100 / 80) ** 0.5 * 0.5
    assert float((steps[True] - want).abs().max()) <= 4 * 2.0 ** -24 * float(start.abs().max())
    del opt.param_groups[0]["full_fp32"]  # a state saved before there was such a setting
    opt.step()
