"""Performance cases of the training and forecasting operators.

Three operators of one train-and-forecast run:

  lookup   embedding rows by token, scaled, and the table's gradient summed by token
  orth     an update orthogonalised by Newton-Schulz products (the Muon optimiser's step)
  sample   ids drawn from scores with temperature, top-k, top-p and min-p, from given random numbers

`run` computes a case in elementary torch operations (`own` false) or through regcn_amd's entry
points (`own` true); `exact` computes it once more in 64 bits from the operator's definition.
"""
import importlib
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
COEFFS = (3.4445, -4.7750, 2.0315)
EPS = 1e-7
FILTERED = -1e7  # what the evaluation writes over the other true answers of a query


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one query's entity row at serving time: latency only
        dict(name="lookup_one", op="lookup", vocab=7128, dim=200, tokens=1, zipf=0.0, pad=0.0, scale=1.0,
             dtype="f32", grad=False),
        # the relation rows of a snapshot's triples in both directions: few rows, each many times
        dict(name="lookup_relations", op="lookup", vocab=512, dim=200, tokens=3080, zipf=0.0, pad=0.0, scale=1.0,
             dtype="f32", grad=True),
        # odd sizes in 16 bits, a padded batch
        dict(name="lookup_odd_f16", op="lookup", vocab=10007, dim=333, tokens=4999, zipf=1.1, pad=0.25,
             scale=18.25, dtype="f16", grad=True),
        # a wide table of word pieces in bf16, scaled by the root of its width
        dict(name="lookup_wide_bf16", op="lookup", vocab=131072, dim=1024, tokens=16384, zipf=1.1, pad=0.0,
             scale=32.0, dtype="bf16", grad=True),
        # a million entities, hub entities in a large share of the tokens
        dict(name="lookup_million", op="lookup", vocab=1000000, dim=200, tokens=262144, zipf=1.1, pad=0.0,
             scale=1.0, dtype="f32", grad=True),
        # the two-dimensional weights of the encoder and its decoders: one optimiser step
        dict(name="orth_model", op="orth", shapes="200x200*11,600x400,600x200,100x200,460x400", spectrum="decay",
             steps=5, dtype="f32"),
        # the convolutional decoders' projections: short and very long
        dict(name="orth_long", op="orth", shapes="200x10000*2", spectrum="flat", steps=5, dtype="f32"),
        # odd sizes, taller than wide
        dict(name="orth_odd_bf16", op="orth", shapes="1333x777", spectrum="decay", steps=5, dtype="bf16"),
        # a large square weight
        dict(name="orth_large", op="orth", shapes="4096x4096", spectrum="flat", steps=5, dtype="f32"),
        # one query's answer among the entities, from the ten best
        dict(name="sample_one", op="sample", rows=1, cols=7128, draws=1, temperature=1.0, top_k=10, top_p=1.0,
             min_p=0.0, filtered=0.01, masked=0.0, spread=3.0, dtype="f32"),
        # a snapshot's queries in both directions, ten facts each, from the bulk of the distribution
        dict(name="sample_snapshot", op="sample", rows=3080, cols=23033, draws=10, temperature=0.8, top_k=0,
             top_p=0.9, min_p=0.0, filtered=0.001, masked=0.0, spread=2.0, dtype="f32"),
        # few queries over a million entities, all three limits
        dict(name="sample_million", op="sample", rows=16, cols=1000000, draws=16, temperature=1.3, top_k=5000,
             top_p=0.95, min_p=0.001, filtered=0.0, masked=0.2, spread=2.5, dtype="f32"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["lookup", "orth", "sample"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "lookup":
        vocab, tokens, dim = _log_int(rng, 1, 1000000), _log_int(rng, 1, 262144), _log_int(rng, 1, 1024)
        dim = max(1, min(dim, 250000000 // (vocab + tokens)))
        return dict(op=op, vocab=vocab, dim=dim, tokens=tokens, zipf=rng.choice([0.0, 1.1, 1.6]),
                    pad=rng.choice([0.0, 0.0, 0.3]), scale=rng.choice([1.0, round(math.sqrt(dim), 3)]), dtype=dtype,
                    grad=rng.random() < 0.75)
    if op == "orth":
        left, shapes = 1.5e12, []
        for _ in range(rng.choice([1, 1, 2, 4, 8])):
            m, n = _log_int(rng, 1, 4096), _log_int(rng, 1, 4096)
            cost = 5 * (3.0 * min(m, n) ** 2 * max(m, n) + min(m, n) ** 3)
            if cost <= left:
                left -= cost
                shapes.append("%dx%d" % (m, n))
        return dict(op=op, shapes=",".join(shapes), spectrum=rng.choice(["flat", "decay"]),
                    steps=rng.choice([3, 4, 5, 5]), dtype=dtype)
    cols = _log_int(rng, 1, 1000000)
    rows = _log_int(rng, 1, max(1, min(4096, 60000000 // cols)))
    return dict(op=op, rows=rows, cols=cols, draws=rng.choice([1, 1, 4, 10]),
                temperature=round(rng.uniform(0.3, 2.0), 3), top_k=rng.choice([0, 1, _log_int(rng, 1, cols)]),
                top_p=rng.choice([1.0, round(rng.uniform(0.05, 0.99), 3)]),
                min_p=rng.choice([0.0, 0.0, round(rng.uniform(0.0, 0.3), 3)]), filtered=rng.choice([0.0, 0.01]),
                masked=rng.choice([0.0, 0.3, 0.9]), spread=round(rng.uniform(0.5, 5.0), 2), dtype=dtype)


def _shapes(case):
    out = []
    for part in case["shapes"].split(","):
        size, _, times = part.partition("*")
        m, _, n = size.partition("x")
        out += [(int(m), int(n))] * int(times or 1)
    return out


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "lookup":
        V, d, n = case["vocab"], case["dim"], case["tokens"]
        moved, flops = 8 * n + (min(n, V) + n) * d * e, n * d
        if case["grad"]:
            moved, flops = moved + (n + V) * d * e, flops + n * d
        return {"bytes": moved, "flops": flops}
    if case["op"] == "orth":
        moved = flops = 0
        for m, n in _shapes(case):
            m, n = min(m, n), max(m, n)
            moved += 2 * m * n * e
            # X X^T and A A are symmetric: half their products
            flops += case["steps"] * (m * m * n + m * m * m + 2 * m * m * n)
        return {"bytes": moved, "flops": flops}
    B, N, S = case["rows"], case["cols"], case["draws"]
    return {"bytes": B * N * e + B * S * 20, "flops": 4 * B * N}


# ----------------------------------------------------------------------------------------- inputs
def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dev, dt = torch.device("cuda"), DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    def uniform(*shape, dtype=torch.float32):
        return torch.rand(*shape, generator=g, device=dev, dtype=dtype)

    if case["op"] == "lookup":
        V, d, n, a = case["vocab"], case["dim"], case["tokens"], case["zipf"]
        u = uniform(n, dtype=torch.float64)
        if a:  # Zipf ranks by inverting the truncated law, dealt over the table by a permutation
            rank = ((V ** (1 - a) - 1) * u + 1) ** (1 / (1 - a)) - 1
            idx = torch.randperm(V, generator=g, device=dev)[rank.long().clamp(0, V - 1)]
        else:
            idx = (u * V).long().clamp(0, V - 1)
        pad = None
        if case["pad"]:
            pad = V // 2
            idx = torch.where(uniform(n) < case["pad"], torch.full_like(idx, pad), idx)
        table = (normal(V, d) * 0.1).to(dt)
        gout = (normal(n, d) * 0.01).to(dt) if case["grad"] else None
        return dict(table=table, idx=idx, pad=pad, gout=gout)
    if case["op"] == "orth":
        mats = []
        for m, n in _shapes(case):
            x = normal(m, n)
            if case["spectrum"] == "decay":  # a few strong directions over noise, as gradients have
                r = max(1, min(m, n) // 16)
                x = x * 0.05 + normal(m, r) @ normal(r, n) / math.sqrt(r)
            mats.append((x * 1e-3).to(dt))
        return dict(mats=mats)
    B, N = case["rows"], case["cols"]
    score = normal(B, N) * case["spread"]
    if case["filtered"]:
        score = torch.where(uniform(B, N) < case["filtered"], torch.full_like(score, FILTERED), score)
    score = score.to(dt)
    if case["masked"]:
        score = torch.where(uniform(B, N) < case["masked"], torch.full_like(score, -math.inf), score)
    return dict(score=score, u=uniform(B, case["draws"], dtype=torch.float64))


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=dict(case))
    if own:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "re-gcn_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        module, name = {"lookup": ("autograd", "embedding"), "orth": ("muon", "orthogonalize"),
                        "sample": ("ranking", "sample")}[case["op"]]
        state["call"] = getattr(importlib.import_module("regcn_amd." + module), name)
        if case["op"] == "lookup" and case["grad"]:
            state["table"].requires_grad_(True)
    return state


# ------------------------------------------------------------------------------------------- runs
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(st):
    case, call = st["case"], st["call"]
    if case["op"] == "lookup":
        if not case["grad"]:
            with torch.no_grad():
                return [call(st["table"], st["idx"], case["scale"], padding_idx=st["pad"])]
        out = call(st["table"], st["idx"], case["scale"], padding_idx=st["pad"])
        return [out.detach(), torch.autograd.grad(out, st["table"], st["gout"])[0]]
    if case["op"] == "orth":
        return call(st["mats"], steps=case["steps"], coeffs=COEFFS, eps=EPS)
    return list(call(st["score"], st["u"], temperature=case["temperature"], top_k=case["top_k"], top_p=case["top_p"],
                     min_p=case["min_p"], return_logp=True))


def _run_plain(st):
    case = st["case"]
    return {"lookup": _plain_lookup, "orth": _plain_orth, "sample": _plain_sample}[case["op"]](case, st)


def _plain_lookup(case, st):
    table, idx, scale = st["table"], st["idx"], case["scale"]
    out = [(table[idx].float() * scale).to(table.dtype)]
    if case["grad"]:
        grad = torch.zeros(table.shape, device=table.device, dtype=torch.float32)
        g = st["gout"].float()
        if st["pad"] is not None:
            g = torch.where((idx == st["pad"]).unsqueeze(1), torch.zeros_like(g), g)
        grad.index_add_(0, idx, g)
        out.append((grad * scale).to(table.dtype))
    return out


def _plain_orth(case, st):
    a, b, c = COEFFS
    out = []
    for G in st["mats"]:
        X = G.float()
        if G.shape[0] > G.shape[1]:
            X = X.t()
        X = X / (X.norm() + EPS)
        for _ in range(case["steps"]):
            A = X @ X.t()
            B = b * A + c * (A @ A)
            X = a * X + B @ X
        if G.shape[0] > G.shape[1]:
            X = X.t()
        out.append(X.to(G.dtype).contiguous())
    return out


def _plain_sample(case, st):
    # weights and running sums in 64 bits: a sum of many weights is compared with a drawn border
    s = st["score"].double()
    B, N = s.shape
    s = torch.where(torch.isnan(s), torch.full_like(s, -math.inf), s)
    order = torch.sort(s, dim=1, descending=True, stable=True)
    top = order.values[:, :1]
    w = torch.where(order.values == top, torch.ones_like(s), torch.exp((order.values - top) / case["temperature"]))
    w = torch.where(order.values == -math.inf, torch.zeros_like(w), w)
    if 0 < case["top_k"] < N:
        w[:, case["top_k"]:] = 0
    run_w = torch.cumsum(w, 1)
    keep = w >= case["min_p"]
    if case["top_p"] < 1:
        keep &= run_w - w < case["top_p"] * run_w[:, -1:]
    kept = torch.zeros_like(w).scatter_(1, order.indices, w * keep)
    run_k = torch.cumsum(kept, 1)
    ids = torch.searchsorted(run_k, st["u"].double() * run_k[:, -1:], right=True)
    last = (torch.arange(N, device=s.device) * (kept > 0)).amax(1, keepdim=True)
    ids = torch.minimum(ids, last)
    logp = torch.log(kept.gather(1, ids) / run_k[:, -1:])
    none = (top == -math.inf).expand_as(ids)
    return [torch.where(none, torch.full_like(ids, -1), ids),
            torch.where(none, torch.full_like(logp, -math.inf), logp).float()]


# ------------------------------------------------------------------------------------------ exact
def exact(case, seed):
    st = _inputs(case, seed)
    if case["op"] == "lookup":
        t = st["table"].double()
        out = [torch.index_select(t, 0, st["idx"]).mul_(case["scale"])]
        if case["grad"]:
            idx, g = st["idx"], st["gout"].double()
            if st["pad"] is not None:
                g, idx = g[idx != st["pad"]], idx[idx != st["pad"]]
            # the rows of one token lie next to each other: each row's sum is a difference of running sums
            token, order = torch.sort(idx, stable=True)
            grad = torch.zeros_like(t)
            for c0 in range(0, t.shape[1], 64):
                run_g = torch.cumsum(g[order, c0:c0 + 64], 0)
                end = torch.ones_like(token, dtype=torch.bool)
                end[:-1] = token[1:] != token[:-1]
                total = run_g[end]
                grad[token[end], c0:c0 + 64] = torch.diff(total, dim=0, prepend=torch.zeros_like(total[:1]))
            out.append(grad.mul_(case["scale"]))
        return out
    if case["op"] == "orth":
        a, b, c = COEFFS
        out = []
        for G in st["mats"]:
            X = G.double()
            X = X / (torch.linalg.vector_norm(X) + EPS)
            eye = torch.eye(min(X.shape), device=X.device, dtype=torch.float64)
            for _ in range(case["steps"]):  # the polynomial on the shorter side
                if X.shape[0] <= X.shape[1]:
                    A = X @ X.t().contiguous()
                    X = (a * eye + b * A + c * (A @ A)) @ X
                else:
                    A = X.t().contiguous() @ X
                    X = X @ (a * eye + b * A + c * (A @ A))
            out.append(X)
        return out
    # one row at a time, by thresholds: a candidate stands before another when its score is larger,
    # or equal with the lower index
    B, N = st["score"].shape
    ids = torch.full((B, case["draws"]), -1, device="cuda", dtype=torch.int64)
    logp = torch.full(ids.shape, -math.inf, device="cuda", dtype=torch.float64)
    k = case["top_k"] if 0 < case["top_k"] < N else N
    for r in range(B):
        s = st["score"][r].double()
        place = torch.nonzero(s > -math.inf).flatten()  # drops NaN and masked scores
        if not place.numel():
            continue
        s = s[place]
        best = torch.argsort(-s, stable=True)[:k]
        w = torch.exp((s[best] - s[best[0]]) / case["temperature"])
        before = torch.cumsum(w, 0) - w
        count = int((before < case["top_p"] * w.sum()).sum()) if case["top_p"] < 1 else len(w)
        count = min(count, int((w >= case["min_p"]).sum()))
        chosen, at = torch.sort(place[best[:count]])
        w = w[:count][at]
        run_w = torch.cumsum(w, 0)
        hit = torch.searchsorted(run_w, st["u"][r] * run_w[-1], right=True).clamp(max=count - 1)
        ids[r] = chosen[hit]
        logp[r] = torch.log(w[hit]) - torch.log(w.sum())
    return [ids, logp]
