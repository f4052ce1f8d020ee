"""The lookup and the Muon optimiser in training steps, held to what a step's own sums allow and to the same bits on replay."""
import numpy as np
import pytest
import torch

from regcn_amd import cli, training
from test_gpu_cli import _graph_vs_eager
from test_gpu_train_forecast import _args, _model

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


@pytest.mark.parametrize("encoder,decoder", [("lgcn", "roth"), ("hyperbolic_uvrgcn", "murp"), ("hyperbolic_uvrgcn", "atth")])
def test_gradients_with_and_without_the_sorted_lookup(encoder, decoder):
    """Every tensor's gradient to 2e-4 of its own largest entry (the training tests' tolerance for another order of sums through
    the encoder's backward), and the same bits on a second run.  Entries that are sums of cancelling terms are off by fp32's step
    of the terms, not of themselves: 2^-23 of the largest gradient of all is added."""
    args = _args(encoder=encoder, decoder=decoder)
    model, (V, R, train, valid, test, tl) = _model(args)
    model.train()
    graphs = cli.GraphCache(V, R, DEV)
    glist = [graphs(s) for s in tl[:2]]
    triples = torch.from_numpy(np.asarray(tl[2], dtype=np.int64)).to(DEV)
    runs = []
    for on in (False, True, True):
        training.use_sorted_lookup(model, on)
        model.zero_grad()
        torch.manual_seed(1)
        le, lr, _, lrad = model.get_loss(glist, triples, None, True, query_time=2)
        (le + lr + lrad).backward()
        runs.append({n: p.grad.clone() for n, p in model.named_parameters() if p.grad is not None})
    plain, once, twice = runs
    assert plain.keys() == once.keys() == twice.keys()
    largest = max(float(g.abs().max()) for g in plain.values())
    for n, g in plain.items():
        top = float(g.abs().max())
        off = float((g - once[n]).abs().max())
        assert off <= 2e-4 * top + 2.0 ** -23 * largest, n
        assert torch.equal(once[n], twice[n]), n


@pytest.mark.parametrize("encoder,decoder", [("lgcn", "roth"), ("hyperbolic_uvrgcn", "murp")])
@pytest.mark.parametrize("extra", [["--optimizer", "muon"], ["--sorted-lookup"], ["--optimizer", "muon", "--sorted-lookup"]])
def test_replayed_steps_train_as_eager_ones(tmp_path, encoder, decoder, extra):
    """--hip-graph with Muon, with the sorted lookup and with both: the eager run's losses bit for bit, its parameters to 1e-6."""
    _graph_vs_eager(tmp_path, encoder, decoder, extra, epochs=3, every=100)
