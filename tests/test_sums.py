"""The staged sums of autograd.py: whole numbers, so every order of summation is exact."""
import ctypes

import pytest
import torch

from regcn_amd import _lib
from regcn_amd import autograd as A

S, W = A.SUM_STAGE, A.SUM_WHOLE


@pytest.mark.parametrize("n", [0, 1, 63, 64, 65, S, W - 1, W, W + 1, W + S, W + S + 17, W * S + 1])
def test_total_is_the_sum(n):
    x = torch.randint(-8, 9, (n,), generator=torch.Generator().manual_seed(n)).double().requires_grad_(True)
    out = A.total(x)
    assert out.shape == () and float(out.detach()) == float(x.detach().sum())
    out.backward()
    assert torch.equal(x.grad, torch.ones(n, dtype=torch.float64))


@pytest.mark.parametrize("shape", [(3, 1), (5, W + 3), (2, 3, W + S), (0, 7), (4, 0), (1, W + 3 * S + 1), (0, W + 1)])
def test_sum_of_the_last_dimension(shape):
    x = torch.randint(-8, 9, shape, generator=torch.Generator().manual_seed(1)).float()
    assert torch.equal(A.sum_last(x), x.sum(-1))
    wide = torch.randint(-8, 9, (shape[-1], 3), generator=torch.Generator().manual_seed(2)).float()
    assert torch.equal(A.total(wide[:, 1]), wide[:, 1].sum())  # a strided column


@pytest.mark.parametrize("small,shape", [((), (3, 5)), ((1,), (200, 7)), ((1, 1), (1, 1)), ((7,), (200, 7)), ((200, 1), (200, 7)),
                                         ((1, 7), (130, 7)), ((3, 1, 2), (4, 3, 65, 2)), ((), (0, 4)), ((4,), (0, 4)),
                                         ((1,), (W + 5, 3)), ((3, 1), (3, W + 5))])
def test_sum_to_is_the_gradient_of_broadcasting(small, shape):
    g = torch.randint(-8, 9, shape, generator=torch.Generator().manual_seed(0)).double()
    t = torch.zeros(small, dtype=torch.float64, requires_grad=True)
    want, = torch.autograd.grad(t.expand(shape), t, g)
    assert torch.equal(A.sum_to(g, t.shape), want)
    assert torch.equal(A.sum_to(g.t().contiguous().t(), t.shape) if g.dim() == 2 else want, want)
    got, = torch.autograd.grad(A.spread(t, shape), t, g)
    assert got.shape == t.shape and torch.equal(got, want)


def test_spread_is_differentiable_in_every_mode():
    t = torch.randn(1, 5, dtype=torch.float64, requires_grad=True)
    f = lambda t: (torch.sin(A.spread(t, (70, 5))) * torch.arange(70.0, dtype=torch.float64)[:, None]).sum(0)  # noqa: E731
    plain = lambda t: (torch.sin(t.expand(70, 5)) * torch.arange(70.0, dtype=torch.float64)[:, None]).sum(0)  # noqa: E731
    assert torch.autograd.gradcheck(f, t, check_forward_ad=True)
    assert torch.autograd.gradgradcheck(f, t)
    v = torch.randn(1, 5, dtype=torch.float64)
    assert torch.allclose(torch.func.jvp(f, (t.detach(),), (v,))[1], torch.func.jvp(plain, (t.detach(),), (v,))[1])
    assert torch.allclose(torch.func.jacrev(f)(t.detach()), torch.func.jacrev(plain)(t.detach()))
    assert A.spread(None, (3,)) is None and A.spread(0.5, (3,)) == 0.5


def dist_ce_inputs(scale_shape, margin_shape):
    g = torch.Generator().manual_seed(3)
    q, e = (torch.randn(n, 4, generator=g, dtype=torch.float64) * 0.3 for n in (6, 9))
    target = torch.randint(0, 9, (6,), generator=g)
    c, bias = torch.rand(6, generator=g, dtype=torch.float64) + 0.1, torch.randn(9, generator=g, dtype=torch.float64)
    scale, margin = (torch.rand(s, generator=g, dtype=torch.float64) + 0.5 for s in (scale_shape, margin_shape))
    return q, e, target, c, bias, scale, margin


def plain_dist_ce(q, e, target, c, bias, scale, margin):
    """The loss pair by pair from the distance's definition."""
    c = c.reshape(-1, 1, 1)
    x, y = -q.unsqueeze(1), e.unsqueeze(0)
    xy, x2, y2 = (x * y).sum(-1, keepdim=True), (x * x).sum(-1, keepdim=True), (y * y).sum(-1, keepdim=True)
    num = (1 + 2 * c * xy + c * y2) * x + (1 - c * x2) * y
    n = (num / (1 + 2 * c * xy + c * c * x2 * y2 + A.EPS)).norm(dim=-1)
    root = torch.sqrt(c + A.EPS).reshape(-1, 1)
    dist = 2 / (root + A.EPS) * torch.atanh(root * n)
    return torch.nn.functional.cross_entropy(scale * (margin - dist) + bias, target)


@pytest.mark.parametrize("scale_shape,margin_shape", [((), ()), ((1,), (1,)), ((6, 1), (6, 1)), ((9,), (1, 9)), ((6, 9), ())])
def test_scale_and_margin_of_any_broadcastable_shape(scale_shape, margin_shape):
    """Both sides are 64-bit sums of 9 terms and a few elementary functions, well conditioned here (1e-10); the loss is
    rounded to fp32 once: half a step of a value below 8, 2^-22."""
    args = dist_ce_inputs(scale_shape, margin_shape)
    q, e, target, c, bias, scale, margin = [a.requires_grad_(True) if a.is_floating_point() else a for a in args]
    leaves = (q, e, c, bias, scale, margin)
    loss = A.hyp_dist_ce_loss(q, e, target, c, bias=bias, scale=scale, margin=margin)
    ref = plain_dist_ce(q, e, target, c, bias, scale, margin)
    assert abs(float(loss.detach()) - float(ref.detach())) <= 2.0 ** -22 + 1e-10
    for a, b, x in zip(torch.autograd.grad(loss, leaves), torch.autograd.grad(ref, leaves), leaves):
        assert a.shape == x.shape
        assert float((a - b).abs().max()) <= 1e-10 * max(1.0, float(b.abs().max()))


def test_forward_mode_through_scale_and_margin():
    q, e, target, c, bias, scale, margin = dist_ce_inputs((), ())
    f = lambda s, m: A.hyp_dist_ce_loss(q, e, target, c, bias=bias, scale=s, margin=m)  # noqa: E731
    one = torch.ones((), dtype=torch.float64)
    _, tangent = torch.func.jvp(f, (scale, margin), (one, 2 * one))
    s, m = scale.clone().requires_grad_(True), margin.clone().requires_grad_(True)
    ds, dm = torch.autograd.grad(f(s, m), (s, m))
    assert abs(float(tangent) - float(ds + 2 * dm)) <= 2.0 ** -24 * abs(float(ds + 2 * dm)) + 1e-10


def test_graph_entry_refuses():
    n = ctypes.c_int64(7)
    assert _lib.lib().regcn_graph_memset_nodes(None, ctypes.byref(n)) < 0
    assert _lib.lib().regcn_graph_memset_nodes(ctypes.byref(n), None) < 0
    assert b"graph_memset_nodes" in _lib.lib().regcn_last_error_string()


@pytest.mark.parametrize("n", [1, 5, W, W + 1, 4 * W])
def test_mean(n):
    x = torch.randint(-8, 9, (n,), generator=torch.Generator().manual_seed(n)).double().requires_grad_(True)
    out = A.mean(x)
    assert abs(float(out.detach()) - float(x.detach().sum()) / n) <= 2.0 ** -52 * 8
    out.backward()
    assert torch.equal(x.grad, torch.full((n,), 1.0 / n, dtype=torch.float64))
