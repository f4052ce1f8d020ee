"""The lookup, the Muon optimiser and sampled forecasts in the paths that call them, one by one and in one run.

Muon's step is checked against the formula in 64 bits.  The tolerance, 1e-5 of the parameter's Frobenius norm
(28 to 78 here: 2.8e-4 and more), by arithmetic: three steps of lr sqrt(rows / cols) <= 0.064 times an update that is off
by less than 1e-4 (the bound of test_gpu_orthogonalize.reference at these sizes), and three fp32 roundings a
step of a parameter of norm <= 78: 3 * 0.064 * 1e-4 + 9 * 2^-24 * 78 < 6.2e-5."""
import math

import numpy as np
import pytest
import torch

from regcn_amd import cli, muon, ranking, training

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def _args(*extra, encoder="lgcn", decoder="roth"):
    return cli.build_parser().parse_args(
        ["-d", "synthetic:icews14s_lgcn_roth", "--gpu", "0", "--encoder", encoder, "--decoder", decoder, "--n-hidden",
         "64", "--n-bases", "32", "--synthetic-snapshots", "8", "--train-history-len", "2", "--test-history-len", "2",
         "--relation-prediction", "--entity-prediction", "--seed", "0", "--dropout", "0.0", *extra])


def _model(args):
    torch.manual_seed(0)
    V, R, train, valid, test = cli.load_dataset(args)
    tl = ranking.split_by_time(train)
    return cli.build_model(args, V, R, tl, DEV), (V, R, train, valid, test, tl)


@pytest.mark.parametrize("encoder,decoder", [("lgcn", "roth"), ("hyperbolic_uvrgcn", "murp"),
                                             ("hyperbolic_uvrgcn", "atth"), ("hyperbolic_uvrgcn", "hyperbolic_convtranse")])
def test_sorted_lookup_gives_the_same_gradients(encoder, decoder):
    """Each looked-up row's gradient is an fp32 sum of the same terms in another order; through the encoder's
    backward both sides keep the tolerance of the training tests: 2e-4 of the largest entry."""
    args = _args(encoder=encoder, decoder=decoder)
    model, (V, R, train, valid, test, tl) = _model(args)
    model.train()
    graphs = cli.GraphCache(V, R, DEV)
    glist = [graphs(s) for s in tl[:2]]
    triples = torch.from_numpy(np.asarray(tl[2], dtype=np.int64)).to(DEV)
    grads = []
    for on in (False, True, True):
        training.use_sorted_lookup(model, on)
        model.zero_grad()
        torch.manual_seed(1)
        le, lr, _, lrad = model.get_loss(glist, triples, None, True, query_time=2)
        (le + lr + lrad).backward()
        grads.append((float(le.detach()), {n: p.grad.clone() for n, p in model.named_parameters() if p.grad is not None}))
    assert abs(grads[0][0] - grads[1][0]) <= 1e-5 * max(1.0, abs(grads[0][0]))
    assert grads[0][1].keys() == grads[1][1].keys()
    for n, g in grads[0][1].items():
        scale = max(1.0, float(g.abs().max()))
        assert float((g - grads[1][1][n]).abs().max()) <= 2e-4 * scale, n
    training.use_sorted_lookup(model, False)
    assert not any(getattr(m, "sorted_lookup", False) for m in model.modules())


def _ortho64(G, steps=5, eps=1e-7):
    a, b, c = muon.COEFFS
    X = G.double()
    flip = X.shape[0] > X.shape[1]
    X = X.t() if flip else X
    X = X / (X.norm() + eps)
    for _ in range(steps):
        A = X @ X.t()
        X = a * X + (b * A + c * (A @ A)) @ X
    return X.t() if flip else X


@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_step_against_the_formula(nesterov):
    shapes = [(40, 64), (64, 40), (64, 64), (20, 300)]
    g = torch.Generator().manual_seed(0)
    ps = [torch.randn(*s, generator=g).to(DEV).requires_grad_(True) for s in shapes]
    frozen = torch.randn(8, 8, device=DEV).requires_grad_(True)  # never gets a gradient
    ref = [p.detach().cpu().double() for p in ps]
    buf = [torch.zeros_like(r) for r in ref]
    kept = frozen.detach().clone()
    opt = muon.Muon([{"params": ps + [frozen]}], lr=0.05, momentum=0.9, nesterov=nesterov, weight_decay=0.1)
    for _ in range(3):
        opt.zero_grad()
        for p, r, b in zip(ps, ref, buf):
            p.grad = torch.randn(*p.shape, generator=g).to(DEV)
            gr = p.grad.cpu().double()
            b.mul_(0.9).add_(gr)
            d = gr + 0.9 * b if nesterov else b
            r.mul_(1 - 0.05 * 0.1).add_(_ortho64(d) * math.sqrt(max(1.0, p.shape[0] / p.shape[1])), alpha=-0.05)
        opt.step()
        for p, r in zip(ps, ref):
            assert float((p.detach().cpu().double() - r).norm()) <= 1e-5 * float(r.norm())
    assert torch.equal(frozen.detach(), kept) and frozen not in opt.state
    state = opt.state_dict()
    again = muon.Muon([{"params": ps + [frozen]}], lr=0.05, momentum=0.9)
    again.load_state_dict(state)
    for p in ps:
        assert torch.equal(again.state[p]["momentum_buffer"], opt.state[p]["momentum_buffer"])


@pytest.mark.parametrize("dt,half_step", [(torch.bfloat16, 2.0 ** -8), (torch.float16, 2.0 ** -11)])
def test_muon_step_of_16_bit_parameters(dt, half_step):
    """The momentum and the step are fp32, the parameter is rounded once: half a step of its type, beside the
    1e-5 of the update's norm that the fp32 step is allowed."""
    g = torch.Generator().manual_seed(1)
    p = torch.randn(40, 64, generator=g).to(DEV).to(dt).requires_grad_(True)
    opt = muon.Muon([p], lr=0.05, momentum=0.9, weight_decay=0.1)
    buf = torch.zeros(40, 64, dtype=torch.float64)
    for step in range(4):
        p.grad = (torch.randn(40, 64, generator=g) * 0.01).to(DEV).to(dt)
        gr = p.grad.cpu().double()
        buf.mul_(0.9).add_(gr)
        want = p.detach().cpu().double() * (1 - 0.05 * 0.1) - 0.05 * _ortho64(gr + 0.9 * buf)
        opt.step()
        off = (p.detach().cpu().double() - want).abs()
        assert float((off - half_step * 1.01 * want.abs()).max()) <= 1e-5 * 0.05 * 64 ** 0.5
        m = opt.state[p]["momentum_buffer"]
        assert m.dtype == torch.float32
        assert float((m.cpu().double() - buf).abs().max()) <= 2 * (step + 1) * 2.0 ** -24 * 0.5
        if step == 1:  # a resumed run goes on with the same bits
            again = muon.Muon([p], lr=0.05, momentum=0.9, weight_decay=0.1)
            again.load_state_dict(opt.state_dict())
            assert torch.equal(again.state[p]["momentum_buffer"], m) and again.state[p]["momentum_buffer"].dtype == m.dtype
            opt = again


def test_split_parameters():
    model, _ = _model(_args())
    mats, rest = muon.split_parameters(model)
    names = {id(p): n for n, p in model.named_parameters()}
    got = {names[id(p)] for p in mats}
    assert "time_gate_weight" in got and "relation_gru.weight_ih" in got and "decoder_ob.rot_proj.weight" in got
    assert not {"dynamic_emb", "emb_rel", "temporal_radius_evolution.radius_mlp.weight"} & got
    assert len(mats) + len(rest) == len(names)


@pytest.mark.parametrize("graph", [False, True])
def test_training_run_with_both(graph, tmp_path):
    """--optimizer muon --sorted-lookup, eager and replayed from HIP graphs: every epoch's loss is finite and
    every matrix has moved."""
    args = _args("--optimizer", "muon", "--sorted-lookup", "--n-epochs", "3", "--evaluate-every", "10",
                 *(["--hip-graph"] if graph else []))
    model, (V, R, train, valid, test, tl) = _model(args)
    mats, _ = muon.split_parameters(model)
    before = [p.detach().clone() for p in mats]
    out = cli.train_model(args, model, tl, valid, V, R, DEV, str(tmp_path / "m.pth"))
    assert len(out["epoch_loss"]) == 3 and all(np.isfinite(out["epoch_loss"]))
    moved = [not torch.equal(p.detach(), b) for p, b in zip(mats, before)]
    used = [p.grad is not None for p in mats]
    assert all(m for m, u in zip(moved, used) if u) and sum(moved) >= 8
    assert all(bool(torch.isfinite(p).all()) for p in model.parameters())


def test_snapshots_from_drawn_answers():
    torch.manual_seed(0)
    V, R, B = 50, 4, 6
    score = torch.randn(B, V, device=DEV)
    tri = torch.tensor([[1, 0, 2], [3, 2, 4], [5, 3, 6], [2, 4, 1], [4, 6, 3], [6, 7, 5]], device=DEV)
    u = torch.rand(B, 9, device=DEV, dtype=torch.float64)
    got = ranking.construct_snap_sampled(tri, V, R, score, 9, u=u, temperature=0.7, top_k=5)
    ids = ranking.sample(score, u, temperature=0.7, top_k=5).cpu().numpy()
    want = [[h, r, o] if r < R else [o, r - R, h] for (h, r, _), row in zip(tri.tolist(), ids) for o in sorted(set(row.tolist()))]
    np.testing.assert_array_equal(got, np.array(want))
    # one draw from the best one is the top-1 snapshot
    np.testing.assert_array_equal(ranking.construct_snap_sampled(tri, V, R, score, 3, top_k=1),
                                  ranking.construct_snap(tri, V, R, score, 1))
    rel = ranking.construct_snap_sampled(tri, V, R, score[:, : 2 * R], 4, relation=True, temperature=0.0)
    np.testing.assert_array_equal(rel, ranking.construct_snap_r(tri, V, R, score[:, : 2 * R].contiguous(), 1))
    score[2] = -float("inf")  # a query without an answer adds none
    assert not any(h == 5 for h, _, _ in ranking.construct_snap_sampled(tri, V, R, score, 4).tolist())


def test_train_then_forecast_in_one_command(tmp_path):
    """python -m regcn_amd.cli with the lookup, Muon and sampled multi-step forecasts together."""
    res = cli.main(["-d", "synthetic:icews14s_lgcn_roth", "--gpu", "0", "--encoder", "lgcn", "--decoder", "roth",
                    "--n-hidden", "64", "--n-bases", "32", "--synthetic-snapshots", "14", "--train-history-len", "2",
                    "--test-history-len", "2", "--relation-prediction", "--entity-prediction", "--seed", "0",
                    "--n-epochs", "2", "--optimizer", "muon", "--sorted-lookup", "--multi-step", "--sample-draws", "8",
                    "--sample-temperature", "0.8", "--sample-top-p", "0.9", "--sample-top-k", "50", "--sample-min-p",
                    "0.001", "--checkpoint", str(tmp_path / "m.pth")])
    assert all(0.0 < m <= 1.0 for m in res)


def test_topk_forecast_is_as_before():
    """Without --sample-draws the next snapshot is the reference's top-k one."""
    args = _args("--multi-step", "--topk", "3")
    score = torch.randn(4, 30, device=DEV)
    tri = torch.tensor([[1, 0, 2], [3, 2, 4], [5, 3, 6], [2, 240, 1]], device=DEV)
    np.testing.assert_array_equal(cli._next_snap(args, tri, 30, 230, score, None),
                                  ranking.construct_snap(tri, 30, 230, score, 3))
