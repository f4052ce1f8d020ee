"""The bound that the orthogonalisation is held to on the GPU tells its arithmetic from a poorer one (modelled on the CPU)."""
import pytest
import torch

from orth_model import bound, error, graded, iterate, split_iterate

ALL = ((0, 0), (0, 1), (1, 0))


@pytest.mark.parametrize("m,n,steps", [(128, 200, 5), (200, 200, 5), (100, 200, 8), (300, 260, 5), (200, 1000, 3)])
def test_the_bound_sees_a_dropped_product(m, n, steps):
    G = torch.randn(m, n, generator=torch.Generator().manual_seed(m + n))
    ref = iterate(G, steps)
    limit = bound(G, ref, steps)
    assert error(split_iterate(G, steps, ALL), ref) <= limit / 2
    for terms in (((0, 0),), ((0, 0), (0, 1)), ((0, 0), (1, 0)), ((0, 0), (0, 0), (0, 0))):
        assert error(split_iterate(G, steps, terms), ref) > 4 * limit, terms


@pytest.mark.parametrize("scale", [1e-2, 1e-4, 1e-6, 1e-8])
def test_halves_serve_up_to_eight_steps(scale):
    """Why more steps take fp32 operands: rows that start below what the halves hold have grown by then."""
    G = graded(100, 200, scale)
    for steps in (1, 3, 5, 8):
        ref = iterate(G, steps)
        assert error(split_iterate(G, steps, ALL), ref) <= bound(G, ref, steps)
    if scale <= 1e-6:
        ref = iterate(G, 12)
        assert error(split_iterate(G, 12, ALL), ref) > 4 * bound(G, ref, 12)
