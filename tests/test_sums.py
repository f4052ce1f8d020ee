"""The staged sums of autograd.py: whole numbers, so every order of summation is exact."""
import pytest
import torch

from regcn_amd import autograd as A

S = A.SUM_STAGE


@pytest.mark.parametrize("n", [0, 1, 63, 64, 65, S - 1, S, S + 1, 2 * S, 2 * S + 17, S * S + 1])
def test_total_is_the_sum(n):
    x = torch.randint(-8, 9, (n,), generator=torch.Generator().manual_seed(n)).double().requires_grad_(True)
    out = A.total(x)
    assert out.shape == () and float(out.detach()) == float(x.detach().sum())
    out.backward()
    assert torch.equal(x.grad, torch.ones(n, dtype=torch.float64))


@pytest.mark.parametrize("shape", [(3, 1), (5, S + 3), (2, 3, 2 * S), (0, 7), (4, 0), (1, 3 * S + 1)])
def test_sum_of_the_last_dimension(shape):
    x = torch.randint(-8, 9, shape, generator=torch.Generator().manual_seed(1)).float()
    assert torch.equal(A.sum_last(x), x.sum(-1))
    wide = torch.randint(-8, 9, (shape[-1], 3), generator=torch.Generator().manual_seed(2)).float()
    assert torch.equal(A.total(wide[:, 1]), wide[:, 1].sum())  # a strided column
