"""Sampling (csrc/sample.hip, ranking.sample) against a plain 64-bit restatement on the host.

Ids are whole numbers and have to be equal.  The kernel's weights are exact multiples of 2^-S,
S = min(51, 63 - ceil(log2 N)), the restatement's are doubles: a border is off by at most N 2^-(S+1)
of the largest weight (2^-33 at N = 2^15), so a draw lands between the two borders of one id with
probability below N times that: under 1e-5 for the largest case here; the numbers are fixed by their seeds.
The log-probability is (s - max) / T - log(sum), rounded once to fp32; sum is off by at most N 2^-(S+1)
<= 2^-23 in its last terms (>= 1 in all): |error| <= 2^-24 |logp| + 2^-23 + 2^-46."""
import math

import numpy as np
import pytest
import torch

from regcn_amd import ranking

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def plain_row(s, u, T, k, p, m):
    """(ids, logp) of one row of float64 scores at the float64 numbers u."""
    s = np.where(np.isnan(s), -np.inf, s)
    N = len(s)
    order = np.lexsort((np.arange(N), -s))
    order = order[s[order] > -np.inf]
    if not len(order):
        return np.full(len(u), -1), np.full(len(u), -np.inf)
    if not T > 0:
        T, k = 1.0, 1
    top = s[order[0]]
    with np.errstate(invalid="ignore"):
        x = np.where(s[order] == top, 0.0, (s[order] - top) / T)
    w = np.exp(x)
    if 0 < k < len(order):
        order, w, x = order[:k], w[:k], x[:k]
    before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
    keep = np.ones(len(w), bool)
    if p < 1:
        keep &= before < max(p * math.fsum(w), 5e-324)
    if m > 0:
        keep &= (w >= m) | (np.arange(len(w)) == 0) | (x == 0)
    order, w, x = order[keep], w[keep], x[keep]
    by_id = np.argsort(order)
    ids, ws, xs = order[by_id], w[by_id], x[by_id]
    run = np.cumsum(ws)
    at = np.searchsorted(run, np.clip(np.nan_to_num(u), 0, None) * run[-1], side="right")
    at = np.minimum(at, np.nonzero(ws > 0)[0][-1])
    return ids[at], xs[at] - math.log(math.fsum(ws))


def check(score, u, T=1.0, k=0, p=1.0, m=0.0, **kw):
    got, logp = ranking.sample(score, u, temperature=T, top_k=k, top_p=p, min_p=m, return_logp=True)
    assert got.shape == u.shape and got.dtype == torch.int64 and logp.dtype == F32
    B = score.shape[0]
    val = lambda v, r: float(v[r]) if torch.is_tensor(v) else float(v)  # noqa: E731
    s, un = score.double().cpu().numpy(), u.double().cpu().numpy().reshape(B, -1)
    g, lg = got.cpu().numpy().reshape(B, -1), logp.double().cpu().numpy().reshape(B, -1)
    for r in range(B):
        ids, lp = plain_row(s[r], un[r], val(T, r), int(val(k, r)), val(p, r), val(m, r))
        np.testing.assert_array_equal(g[r], ids, err_msg="row %d" % r)
        fin = np.isfinite(lp)
        np.testing.assert_array_equal(fin, np.isfinite(lg[r]))
        assert (np.abs(lg[r][fin] - lp[fin]) <= 2.0 ** -24 * np.abs(lp[fin]) * 1.01 + 2.0 ** -22).all()
    again = ranking.sample(score, u, temperature=T, top_k=k, top_p=p, min_p=m)
    assert torch.equal(again, got)


def make(B, N, S, seed, dt=F32, spread=2.0, masked=0.0, filtered=0.0):
    g = torch.Generator().manual_seed(seed)
    s = torch.randn(B, N, generator=g) * spread
    if filtered:
        s[torch.rand(B, N, generator=g) < filtered] = ranking.FILTERED_SCORE
    s = s.to(dt)
    if masked:
        s[torch.rand(B, N, generator=g) < masked] = -float("inf")
    return s.to(DEV), torch.rand(B, S, generator=g, dtype=torch.float64).to(DEV)


LIMITS = [dict(), dict(k=1), dict(k=10), dict(p=0.9), dict(m=0.05), dict(T=0.7, k=50, p=0.8, m=0.01), dict(T=2.5, p=0.3),
          dict(T=0.0), dict(k=7, p=0.5), dict(p=0.0), dict(m=1.0)]


@pytest.mark.parametrize("lim", range(len(LIMITS)))
@pytest.mark.parametrize("N,dt", [(1, F32), (2, F16), (63, F32), (64, BF16), (65, F32), (460, F32), (2048, BF16), (2049, F32),
                                  (7128, F32), (7691, F16), (16385, BF16), (23033, F32), (32768, F16), (32769, F32),
                                  (70001, BF16)])
def test_sizes_and_limits(N, dt, lim):
    s, u = make(5, N, 3, N + lim, dt)
    check(s, u, **LIMITS[lim])


@pytest.mark.parametrize("N", [10, 4000, 23033, 40000])
def test_masks(N):
    s, u = make(8, N, 4, 1, masked=0.5, filtered=0.2)
    s[0] = -float("inf")                  # nothing to take
    s[1] = float("nan")
    s[2] = torch.finfo(F32).min           # masks of the type's lowest value are scores
    s[3, ::2] = torch.finfo(F32).min
    s[4, 3], s[4, 7] = float("inf"), float("inf")  # share all weight
    s[5, 1:] = -float("inf")              # one score left
    s[6, ::3] = float("nan")
    for lim in LIMITS:
        check(s, u, **lim)


@pytest.mark.parametrize("N", [64, 5000, 33000])
def test_ties(N):
    """Equal scores: the lowest ids are kept, whatever the limit cuts through."""
    s, u = make(4, N, 6, 2)
    s[0] = 1.5
    s[1] = torch.randint(0, 3, (N,)).float()
    s[2, : N // 2] = 4.0
    s[3] = torch.where(torch.arange(N) % 2 == 0, torch.zeros(N), -torch.zeros(N))  # 0 and -0 are equal
    for lim in (dict(k=17), dict(p=0.5), dict(p=0.37), dict(k=N // 3, p=0.61), dict(k=N // 2 + 1), dict(m=0.2, k=9),
                dict(k=1, p=0.9), dict(k=2, p=0.99), dict(k=N - 1, p=0.999)):
        check(s, u, **lim)
    # keeping only the first 17 ids of a constant row, evenly spaced numbers take each of them
    even = ((torch.arange(17, dtype=torch.float64) + 0.5) / 17).to(DEV)
    assert ranking.sample(s[0], even, top_k=17).tolist() == list(range(17))


def test_numbers_at_the_ends():
    s, _ = make(3, 300, 1, 5)
    u = torch.tensor([[0.0, 1.0 - 2.0 ** -53, 0.5, 1.0, 2.0, -1.0, float("nan")]] * 3, dtype=torch.float64, device=DEV)
    got = ranking.sample(s, u)
    assert (got[:, 0] == 0).all() and (got[:, 1] == 299).all() and (got[:, 3] == 299).all() and (got[:, 4] == 299).all()
    assert (got[:, 5] == 0).all() and (got[:, 6] == 0).all()
    f = torch.rand(3, 2, device=DEV)
    assert torch.equal(ranking.sample(s, f), ranking.sample(s, f.double()))


@pytest.mark.parametrize("N", [1, 700, 50000])
def test_a_certain_draw_has_log_probability_zero(N):
    s, u = make(3, N, 2, 6)
    for lim in (dict(top_k=1), dict(temperature=0.0), dict(top_p=0.0), dict(min_p=1.0)):
        ids, logp = ranking.sample(s, u, return_logp=True, **lim)
        assert torch.equal(ids, s.argmax(1, keepdim=True).expand(3, 2)) and not bool(logp.any())


@pytest.mark.parametrize("N", [500, 40000])
def test_limits_per_row(N):
    B = 9
    s, u = make(B, N, 2, 9)
    T = torch.tensor([1.0, 0.5, 2.0, 0.0, 1.0, 3.0, 0.1, 1.0, 1.0], device=DEV)
    k = torch.tensor([0, 5, 1, 9, N, N + 7, -3, 20, 3], device=DEV)
    p = torch.tensor([1.0, 0.5, 0.9, 0.2, 0.75, 1.5, 0.99, 0.0, 1.0], device=DEV)
    m = torch.tensor([0.0, 0.0, 0.1, 0.0, 0.5, -1.0, 0.01, 0.0, 1.0], device=DEV)
    check(s, u, T=T, k=k, p=p, m=m)


@pytest.mark.parametrize("scale", [1e-30, 1e-3, 1e3, 3e37])
def test_scales_of_scores(scale):
    s, u = make(4, 3000, 3, 11)
    s = s * scale
    for T in (1.0, float(scale)):
        for lim in (dict(), dict(p=0.9), dict(k=100, p=0.7)):
            check(s, u, T=T, **lim)


def test_strides_and_shapes():
    s, u = make(6, 500, 3, 12)
    wide = torch.zeros(6, 700, device=DEV)
    wide[:, 101:601] = s
    want = ranking.sample(s, u, top_p=0.9)
    assert torch.equal(ranking.sample(wide[:, 101:601], u, top_p=0.9), want)
    assert torch.equal(ranking.sample(s.t().contiguous().t(), u, top_p=0.9), want)
    assert torch.equal(ranking.sample(s, u.t().contiguous().t(), top_p=0.9), want)
    assert torch.equal(ranking.sample(s, u[:, 0], top_p=0.9), want[:, 0])
    assert torch.equal(ranking.sample(s[2], u[2], top_p=0.9), want[2])
    assert ranking.sample(s[2], u[2, 0], top_p=0.9).shape == ()
    assert int(ranking.sample(s[2], u[2, 0], top_p=0.9)) == int(want[2, 0])
    one = s[:1].expand(6, 500)
    assert torch.equal(ranking.sample(one, u), ranking.sample(one.contiguous(), u))
    assert ranking.sample(s[:0], u[:0]).shape == (0, 3) and ranking.sample(s, u[:, :0]).shape == (6, 0)
    none, lp = ranking.sample(s[:, :0], u, return_logp=True)
    assert (none == -1).all() and (lp == -float("inf")).all()


def test_many_rows_and_draws():
    s, u = make(700, 1000, 33, 13)
    check(s, u, T=0.9, k=200, p=0.95)


@pytest.mark.parametrize("N", [3000, 60000])
@pytest.mark.parametrize("k", [1, 2, 3, 40])
def test_equal_scores_at_the_top(N, k):
    """Several scores share the top: top_k leaves some of them out, and top_p must not let them in again."""
    s, u = make(6, N, 5, k, BF16)
    top = float(s.float().max()) + 1.0
    for r, n in enumerate((2, 2, 3, 5, 100, 700)):
        s[r, torch.randperm(N, generator=torch.Generator().manual_seed(r))[:n].to(DEV)] = top
    for lim in (dict(), dict(p=0.93), dict(p=0.999999), dict(p=0.4), dict(m=0.5)):
        check(s, u, k=k, **lim)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_a_million(dt):
    s, u = make(2, 1000000, 8, 14, dt, masked=0.3)
    for lim in (dict(T=1.3, k=5000, p=0.95, m=0.001), dict(p=0.5), dict(k=1), dict()):
        check(s, u, **lim)


def test_frequencies_follow_the_weights():
    """At evenly spaced numbers the draws of an id are its share of the kept weight, to one draw."""
    s = torch.randn(40, generator=torch.Generator().manual_seed(3)).to(DEV)
    n = 100000
    u = ((torch.arange(n, dtype=torch.float64) + 0.5) / n).to(DEV)
    got = torch.bincount(ranking.sample(s, u, temperature=0.5), minlength=40).double()
    want = torch.softmax(s.double() / 0.5, 0) * n
    assert float((got - want).abs().max()) <= 1.0 + 1e-6


def test_second_stream_and_replays():
    """Two captured graphs replayed in turn with eager work between give the eager ids every time."""
    data, side = [], torch.cuda.Stream()
    for k, (B, N) in enumerate(((50, 7128), (3, 200000))):
        s, u = make(B, N, 4, 20 + k)
        kw = dict(temperature=0.8, top_k=300, top_p=0.9, return_logp=True)
        with torch.cuda.stream(side):
            want = ranking.sample(s, u, **kw)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = ranking.sample(s, u, **kw)
        data.append((graph, outs, want, s, u))
    for _ in range(3):
        for graph, outs, want, s, u in data:
            for o in outs:
                o.zero_()
            torch.cuda.synchronize()
            graph.replay()
            ranking.sample(s, u, top_p=0.5)
            torch.cuda.synchronize()
            assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_large_offsets():
    """Rows whose scores lie past 2^31 elements."""
    s = torch.zeros(2200, 1000003, device=DEV, dtype=BF16)
    s[2199, 77777] = 50.0
    s[2100, 1000002] = 50.0
    u = torch.full((2200,), 0.5, dtype=torch.float64, device=DEV)
    got = ranking.sample(s, u, top_k=1)
    assert int(got[2199]) == 77777 and int(got[2100]) == 1000002 and int(got[0]) == 0


@pytest.mark.parametrize("N", [40, 5000, 40000])
def test_limits_per_row_in_64_bits(N):
    """A limit given per row keeps what the same number keeps for all rows, its bits beyond fp32 and int32 among them.
    The weights are 1, 1/2, 1/4, ...: top_p = 3/4 of a sum of 2 - 2^-39 keeps two, a little less one more or fewer."""
    s, u = make(6, N, 5, 21)
    s[0] = -float("inf")
    s[0, :40] = -math.log(2.0) * torch.arange(40, dtype=torch.float64).float().to(DEV)
    s[1:3] = s[0]
    full = lambda v, dt=torch.float64: torch.full((6,), v, dtype=dt, device=DEV)  # noqa: E731
    for T in (1.0, 0.7, 1.0 / 3.0):
        for p in (0.9, 0.75, 0.75 - 1e-12, 0.75 + 1e-9, 1.0 / 3.0):
            for m in (0.0, 0.1, 0.25):
                want = ranking.sample(s, u, temperature=T, top_p=p, min_p=m, return_logp=True)
                got = ranking.sample(s, u, temperature=full(T), top_p=full(p), min_p=full(m), return_logp=True)
                assert all(torch.equal(a, b) for a, b in zip(got, want)), (T, p, m)
    for k in (2 ** 32 + 5, 2 ** 40, -(2 ** 35) + 3):  # off
        assert torch.equal(ranking.sample(s, u, top_k=full(k, torch.int64)), ranking.sample(s, u))
    assert torch.equal(ranking.sample(s, u, top_k=full(5, torch.int64)), ranking.sample(s, u, top_k=5))


def test_more_rows_and_draws_than_a_launch_holds():
    """18 million rows of 3 scores; 9 million draws from a row of 40,000: each takes more than one launch."""
    gen = torch.Generator(device=DEV).manual_seed(5)
    s = torch.rand(18_000_001, 3, device=DEV, generator=gen)
    u = torch.rand(18_000_001, device=DEV, generator=gen)
    assert torch.equal(ranking.sample(s, u, top_k=1), s.argmax(1))
    T = torch.where(torch.arange(18_000_001, device=DEV) % 2 == 0, 0.0, 1e-6)  # both: one of the best, others are 1 below
    far = (s * 1e4).round()
    first = ranking.sample(far, u, temperature=T)
    assert bool((far.gather(1, first[:, None])[:, 0] == far.amax(1)).all())
    del s, u, far, first
    row = torch.zeros(40000, device=DEV)
    n = 9_000_000
    u = (torch.arange(n, dtype=torch.float64, device=DEV) + 0.5) / n
    got = ranking.sample(row, u)  # equal weights: the place of u in the row, to the weight's rounding
    assert torch.equal(got, (u * 40000).long())


@pytest.mark.parametrize("N,dt", [(1 << 20, F32), ((1 << 20) + 1, F16), (3_000_001, F32), (1 << 24, F32)])
def test_the_widest_rows(N, dt):
    """Every draw is that of the stated weights, whole multiples of 2^-S: an id's running sum on the host, in whole numbers.
    The exponentials here are numpy's and may round to another multiple than the kernel's (both within 2^-52, so
    fewer than N 2^(S-52) of the weights, each by 1): a draw may lie that far over a border.  Against the weights
    before their rounding it lies within the stated N 2^-(S+1), and again that."""
    S = min(51, 63 - math.ceil(math.log2(N)))
    g = torch.Generator().manual_seed(N)
    s = (torch.rand(N, generator=g) * -33.0).to(dt)
    s[N // 3], s[5::1000] = 0.0, -30.0
    u = torch.rand(200, generator=g, dtype=torch.float64)
    got, logp = ranking.sample(s.to(DEV), u.to(DEV), return_logp=True)
    w = np.exp(s.double().numpy())
    whole = np.rint(w * 2.0 ** S).astype(np.uint64)
    run = np.cumsum(whole)
    total = int(run[-1])
    assert total <= 1 << 63
    slack = max(2, math.ceil(N * 2.0 ** (S - 52)) + 2)
    exact = np.cumsum(w.astype(np.longdouble))
    for i, x, lp in zip(got.tolist(), u.tolist(), logp.tolist()):
        t = x * float(total)
        assert int(run[i]) - int(whole[i]) - slack <= t + t * 2.0 ** -52 and t - t * 2.0 ** -52 < int(run[i]) + slack
        assert int(whole[i]) > 0
        lost = 2.0 * N * 2.0 ** -(S + 1)
        assert float(exact[i]) - w[i] - lost <= x * float(exact[-1]) <= float(exact[i]) + lost
        assert abs(lp - (float(s[i]) - math.log(float(exact[-1])))) <= 2.0 ** -24 * abs(lp) * 1.01 + lost / float(exact[-1]) + 2.0 ** -40
    for lim in (dict(k=1000), dict(p=0.7), dict(k=100000, p=0.5, m=1e-6)):
        assert torch.equal(ranking.sample(s.to(DEV), u.to(DEV), top_k=lim.get("k", 0), top_p=lim.get("p", 1.0), min_p=lim.get("m", 0.0)),
                           ranking.sample(s.to(DEV)[None], u.to(DEV)[None], top_k=lim.get("k", 0), top_p=lim.get("p", 1.0),
                                          min_p=lim.get("m", 0.0))[0])
        check(s.to(DEV)[None], u.to(DEV)[None], **lim)
