"""The embedding gradient's sums at the borders of its sort and its tree (csrc/lookup.hip).

Tolerance, by arithmetic.  A run of sorted tokens is summed over a tree of fan 16 and five levels: a node is a sum of 16 nodes
of the level below, so an element passes at most 16 additions at each of 4 levels inside nodes; the row then adds at most 15
tokens or nodes at each end of each level, 30 at the level where it ends, and at the last level one node for every 65,536
tokens.  In all D = 4 * 16 + 4 * 30 + 30 + n / 65536 additions, each off by at most 2^-24 of a partial sum's magnitudes; one more
rounding for the product with the scale; half a step of the type for the store (fp16's subnormals: 2^-25)."""
import pytest
import torch

from regcn_amd import autograd as A
from test_gpu_embedding import HALF_STEP, ref_grad

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def check(V, d, idx, dt, scale=1.25, seed=0):
    gen = torch.Generator().manual_seed(seed)
    g = torch.randn(len(idx), d, generator=gen).to(DEV).to(dt)
    table = torch.randn(V, d, generator=gen).to(DEV).to(dt).requires_grad_(True)
    out = A.embedding(table, idx.to(DEV), scale)
    got, = torch.autograd.grad(out, table, g)
    ref, mag = ref_grad(g, idx, V, scale)
    depth = 4 * 16 + 4 * 30 + 30 + len(idx) // 65536 + 1
    tol = depth * 2.0 ** -24 * mag + HALF_STEP[dt] * ref.abs() * 1.001 + (2.0 ** -25 if dt == F16 else 0.0)
    err = (got.double().cpu() - ref).abs()
    assert bool((err <= tol).all()), "max excess %.3g" % float((err - tol).max())
    assert torch.equal(out.detach(), (table.detach()[idx.to(DEV)].float() * scale).to(dt))


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("n", [63, 64, 8191, 8192, 8193, 65535, 65536, 65537])
def test_borders_of_the_sort(n, dt):
    """8,192 tokens are ranked by counting, more in radix passes of 2,048 tokens and more a workgroup."""
    gen = torch.Generator().manual_seed(n)
    check(300, 20, torch.randint(0, 300, (n,), generator=gen), dt)
    check(2000, 4, (torch.randint(0, 2000, (n,), generator=gen).float() ** 0.3).long(), dt)


@pytest.mark.parametrize("run", [15, 16, 17, 31, 255, 256, 257, 271, 4095, 4096, 4097, 4352, 65536, 69632, 131072])
@pytest.mark.parametrize("before", [0, 1, 15, 16, 250])
def test_runs_that_end_anywhere_in_the_tree(run, before):
    """One row's tokens begin `before` places into the sorted order and take `run`; a row after them takes 40."""
    idx = torch.tensor([0] * before + [1] * run + [2] * 40)
    check(3, 8, idx[torch.randperm(len(idx), generator=torch.Generator().manual_seed(run))], F32)


@pytest.mark.parametrize("n", [(1 << 20) + 5, 3_000_000])
def test_a_row_with_every_token(n):
    check(2, 4, torch.ones(n, dtype=torch.int64), F32)
