"""Sums of captured training steps against the same step run eagerly, on inputs that change between the replays (a
sum whose workgroups' tickets are not cleared leaves its result of the replay before)."""
import numpy as np
import pytest
import torch

from regcn_amd import _lib
from regcn_amd import autograd as A
from regcn_amd import cli, muon, ranking, training
from regcn_amd import hyperbolic_decoder as D
from regcn_amd.weights import bump_versions

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def replays_as_eager(step, leaves, times=4):
    """step() -> tensors that follow from `leaves`: captured once and replayed, the leaves changed in place and eager
    work done between the replays; every replay gives the eager bits."""
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = [o.detach() for o in step()]
    for k in range(times):
        with torch.no_grad():
            for x in leaves:
                x.mul_(1.0 + 0.01 * (k + 1))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            want = [o.detach().clone() for o in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.randn(300000, device=DEV).sum()
        torch.cuda.synchronize()
        for i, (o, w) in enumerate(zip(outs, want)):
            assert torch.equal(o, w), "replay %d, output %d: off by %.3g of %.3g" % (
                k, i, float((o - w).abs().max()), float(w.abs().max()))


@pytest.mark.parametrize("n", [4097, 32768, 32769, 131072, 1000003])
def test_totals(n):
    x = torch.randn(n, 3, device=DEV)
    replays_as_eager(lambda: [A.total(x), A.total(x[:, 1]), A.sum_last(x.t())], [x])


@pytest.mark.parametrize("B,N", [(8, 200001), (300, 9000)])
def test_cross_entropy_gradients(B, N):
    g = torch.Generator().manual_seed(N)
    q = (torch.randn(B, 16, generator=g) * 0.3).to(DEV).requires_grad_(True)
    cand = (torch.randn(N, 16, generator=g) * 0.3).to(DEV).requires_grad_(True)
    bias = torch.randn(N, generator=g).to(DEV).requires_grad_(True)
    scale, margin = (torch.tensor(v, device=DEV).requires_grad_(True) for v in (1.5, 0.25))
    target = torch.randint(0, N, (B,), generator=g).to(DEV)
    leaves = [q, cand, bias, scale, margin]

    def step():
        loss = A.hyp_ce_loss(q, cand, target, 0.01, bias=bias, scale=scale, margin=margin)
        return [loss.detach(), *torch.autograd.grad(loss, leaves)]
    replays_as_eager(step, leaves)


@pytest.mark.parametrize("batch", [None, 20])
def test_step_with_many_entities(batch):
    """140,000 entities: the losses and gradients of a whole step, its radius loss among them."""
    V, R = 140000, 12
    args = cli.build_parser().parse_args(
        ["-d", "synthetic:icews14s_lgcn_roth", "--gpu", "0", "--encoder", "hyperbolic_uvrgcn", "--decoder", "roth",
         "--n-hidden", "32", "--n-bases", "16", "--relation-prediction", "--entity-prediction", "--dropout", "0",
         "--input-dropout", "0", "--hidden-dropout", "0", "--feat-dropout", "0"])
    rng = np.random.default_rng(0)
    snaps = [np.stack([rng.integers(0, V, 900), rng.integers(0, R, 900), rng.integers(0, V, 900)], 1) for _ in range(3)]
    torch.manual_seed(0)
    model = cli.build_model(args, V, R, snaps, DEV)
    model.train()
    graphs = cli.GraphCache(V, R, DEV)
    glist = [graphs(s) for s in snaps[:2]]
    triples = torch.from_numpy(snaps[2][:50].astype(np.int64)).to(DEV)
    params = [p for p in model.parameters() if p.requires_grad]

    def step():
        for p in params:
            p.grad = None
        if batch is None:
            losses = model.get_loss(glist, triples, None, True, query_time=2)
            sum(l.sum() for l in losses).backward()
        else:
            parts = model.get_loss_batches(glist, triples, None, True, batch, query_time=2)
            losses = [l for part in parts for l in part]
        bump_versions(params)  # as after an optimizer step: caches made of the parameters are made again
        return [l.detach() for l in losses] + [p.grad for p in params if p.grad is not None]
    replays_as_eager(step, params)


@pytest.mark.parametrize("rows", [7, 460, 512, 3000])
def test_gru_cell(rows):
    """torch's own cell to the bit but for the order of the bias gradients' sums: at most `rows` additions of fp32 terms,
    rows 2^-24 of the sum of their magnitudes."""
    torch.manual_seed(rows)
    cell = torch.nn.GRUCell(80, 40).to(DEV)
    x, h = (torch.randn(rows, n, device=DEV).requires_grad_(True) for n in (80, 40))
    g = torch.randn(rows, 40, device=DEV)
    leaves = [x, h, *cell.parameters()]
    out = A.gru_cell(cell, x, h)
    want = cell(x, h)
    assert torch.equal(out, want)
    got, ref = torch.autograd.grad(out, leaves, g), torch.autograd.grad(want, leaves, g)
    for (name, _), a, b in zip([("x", 0), ("h", 0), *cell.named_parameters()], got, ref):
        if name.startswith("bias"):  # |g| <= 6 and a gate's factors are below 1
            assert float((a - b).abs().max()) <= 2 * rows * 2.0 ** -24 * rows * 6.0
        else:
            assert torch.equal(a, b), name
    del out, want
    replays_as_eager(lambda: [*torch.autograd.grad(A.gru_cell(cell, x, h), leaves, g)], leaves + [g])


@pytest.mark.parametrize("B", [64, 3080])
@pytest.mark.parametrize("turn", [D.givens_rotation, D.givens_reflection])
def test_angles_that_all_rows_share(B, turn):
    x, angles = torch.randn(B, 200, device=DEV).requires_grad_(True), torch.randn(100, device=DEV).requires_grad_(True)
    g = torch.randn(B, 200, device=DEV)
    replays_as_eager(lambda: [*torch.autograd.grad(turn(x, angles), [x, angles], g)], [x, angles, g])
    rows = angles.detach().expand(B, 100).contiguous()
    assert torch.equal(turn(x.detach(), angles.detach()), turn(x.detach(), rows))


@pytest.mark.parametrize("B,N", [(3080, 460), (70, 9000)])
def test_distance_cross_entropy_gradients(B, N):
    g = torch.Generator().manual_seed(B)
    q, cand = ((torch.randn(n, 8, generator=g) * 0.3).to(DEV).requires_grad_(True) for n in (B, N))
    c, bias = ((torch.rand(n, generator=g) + 0.05).to(DEV).requires_grad_(True) for n in (B, N))
    scale, margin = (torch.tensor(v, device=DEV).requires_grad_(True) for v in (1.5, 0.25))
    target = torch.randint(0, N, (B,), generator=g).to(DEV)
    leaves = [q, cand, c, bias, scale, margin]

    def step():
        loss = A.hyp_dist_ce_loss(q, cand, target, c, bias=bias, scale=scale, margin=margin)
        return [loss.detach(), *torch.autograd.grad(loss, leaves)]
    replays_as_eager(step, leaves)


def test_convolutional_relation_scores_bias():
    torch.manual_seed(0)
    dec = D.HyperbolicConvTransR(256, 40).to(DEV)
    ent, rel = torch.randn(50, 40, device=DEV) * 0.1, torch.randn(512, 40, device=DEV) * 0.1
    tri = torch.randint(0, 50, (3080, 3), device=DEV)
    g = torch.randn(3080, 512, device=DEV)
    replays_as_eager(lambda: [*torch.autograd.grad(dec(ent, rel, tri), [dec.b], g)], [g])


def test_steps_whose_graph_would_not_replay_run_eagerly(caplog):
    """A sum over several workgroups in a step: right on every run, where a replay would not be; the other keys replay."""
    x = torch.ones(1 << 20, device=DEV)
    steps, calls = training.GraphedSteps(DEV), {"sum": 0, "total": 0}

    def step(name):
        calls[name] += 1
        return x.sum() if name == "sum" else A.total(x)
    for k in range(1, 5):
        x.fill_(float(k))
        for name in calls:
            assert float(steps.run(name, lambda: step(name))) == float(k << 20)
    assert calls == {"sum": 5, "total": 2}  # the capture's own call among them
    assert sum("memset" in r.message for r in caplog.records) == 1


@pytest.mark.parametrize("encoder,decoder,extra", [
    ("lgcn", "roth", []), ("hyperbolic_uvrgcn", "roth", ["--no-reuse-encoder"]), ("hyperbolic_uvrgcn", "atth", []),
    ("hyperbolic_uvrgcn", "murp", ["--sorted-lookup"]), ("hyperbolic_uvrgcn", "hyperbolic_convtranse", []),
    ("lgcn", "roth", ["--plus-relation-specific-curvature"])])
def test_training_steps_hold_no_memset_nodes(encoder, decoder, extra):
    """Whole steps of 3,080 queries over 23,033 entities and 512 relations, both optimisers among them: --hip-graph
    replays them."""
    args = cli.build_parser().parse_args(
        ["-d", "synthetic:icews18_roth", "--gpu", "0", "--encoder", encoder, "--decoder", decoder, "--n-hidden", "200",
         "--synthetic-snapshots", "5", "--relation-prediction", "--entity-prediction", "--optimizer", "muon", *extra])
    torch.manual_seed(0)
    V, R, train, _, _ = cli.load_dataset(args)
    tl = ranking.split_by_time(train)
    model = training.use_sorted_lookup(cli.build_model(args, V, R, tl, DEV), args.sorted_lookup)
    model.train()
    graphs = cli.GraphCache(V, R, DEV)
    glist = [graphs(s) for s in tl[:2]]
    triples = torch.from_numpy(np.asarray(tl[2], dtype=np.int64)).to(DEV)
    mats, rest = muon.split_parameters(model)
    optimizer = cli.Optimizers(muon.Muon(mats), torch.optim.Adam(rest, capturable=True, fused=True))

    def step():
        optimizer.zero_grad()
        if args.reuse_encoder:
            model.get_loss_batches(glist, triples, None, True, args.triple_batch_size, query_time=2)
        else:
            sum(l.sum() for l in model.get_loss(glist, triples, None, True, query_time=2)).backward()
        torch.nn.utils.clip_grad_norm_(model.parameters(), 1.0)
        optimizer.step()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph, stream=side):
        step()
    assert _lib.graph_memset_nodes(graph) == 0


def test_replayed_steps_draw_new_dropout_masks():
    """A step's random numbers are the generator's next ones on every replay."""
    x = torch.ones(4000, device=DEV)
    steps = training.GraphedSteps(DEV)
    masks = [steps.run("key", lambda: torch.nn.functional.dropout(x, 0.5) * 1.0).clone() for _ in range(5)]
    torch.cuda.synchronize()
    assert all(1500 < int((m > 0).sum()) < 2500 for m in masks)
    assert not any(torch.equal(a, b) for i, a in enumerate(masks) for b in masks[:i])


def test_loss_of_many_queries():
    """The mean over 140,000 queries of 40 candidates."""
    g = torch.Generator().manual_seed(0)
    q, cand = ((torch.randn(n, 8, generator=g) * 0.3).to(DEV).requires_grad_(True) for n in (140000, 40))
    target = torch.randint(0, 40, (140000,), generator=g).to(DEV)
    one = torch.ones((), device=DEV)

    def step():
        loss = A.hyp_ce_loss(q, cand, target, 0.01, scale=one, margin=one)
        return [loss.detach(), *torch.autograd.grad(loss, [q, cand])]
    replays_as_eager(step, [q, cand])


def test_muon_refuses_its_first_step_in_a_capture():
    """A momentum buffer made there would be cleared by every replay; after an eager step the capture carries it on."""
    p, ref = (torch.randn(40, 30, generator=torch.Generator().manual_seed(1)).to(DEV).requires_grad_(True) for _ in range(2))
    grad = torch.randn(40, 30, device=DEV)
    opt, ref_opt = muon.Muon([p]), muon.Muon([ref])
    p.grad, ref.grad = grad.clone(), grad.clone()
    side = torch.cuda.Stream()
    with pytest.raises(RuntimeError, match="first Muon step"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            opt.step()
    torch.cuda.synchronize()
    assert not opt.state[p]
    for _ in range(5):
        ref_opt.step()
    with torch.cuda.stream(side):
        opt.step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        opt.step()
    for _ in range(4):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(p, ref) and torch.equal(opt.state[p]["momentum_buffer"], ref_opt.state[ref]["momentum_buffer"])
