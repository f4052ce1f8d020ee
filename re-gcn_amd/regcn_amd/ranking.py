"""Evaluation ranking with time-aware filtering (mirror of rgcn/utils.py:21-305, SURVEY.md
§8(f) row f2).

`get_total_rank(test_triples, score, all_ans, eval_bz, rel_predict=0)` keeps the reference
signature and returns `(filter_mrr, mrr, rank, filter_rank)`, but instead of two full
`torch.sort`s per batch and a host loop writing -1e7 into the filtered answers it runs one
HIP kernel (`regcn_rank_f32`): rank = 1 + #{candidates scoring strictly above the target},
and the filtered rank additionally excludes the other true answers of the same snapshot
(a CSR list built once on the host).  Without score ties against the target this equals
the reference's sort position + 1; with ties the reference's order is whatever
`torch.sort` returns (unspecified), the kernel counts the tie as not above (the optimistic
rank).  As in the reference (filter_score / filter_score_r write into a view of `score`,
rgcn/utils.py:51-75), `score` leaves get_total_rank with the other true answers set to
-1e7, so `construct_snap` under --multi-step picks its top-k from the filtered scores.
"""
import ctypes

import numpy as np
import torch

from . import _lib


def _filter_csr(test_triples, all_ans, rel_predict):
    """Per query, the other true answers (reference filter_score / filter_score_r)."""
    tri = test_triples.detach().cpu().numpy()
    ptr = [0]
    idx = []
    for h, r, t in tri.tolist():
        if all_ans is None:
            ans = ()
        elif rel_predict:
            ans = set(all_ans.get(h, {}).get(t, ())) - {r}
        else:
            ans = set(all_ans.get(h, {}).get(r, ())) - {t}
        idx.extend(sorted(ans))
        ptr.append(len(idx))
    return np.asarray(ptr, dtype=np.int32), np.asarray(idx, dtype=np.int32)


def ranks(score, target, filt_ptr=None, filt_idx=None):
    """(rank, filtered rank), 1-based int64, one HIP launch."""
    B, N = score.shape
    s = score.detach().contiguous().float()
    dev = s.device
    tgt = target.to(device=dev, dtype=torch.int32).contiguous()
    raw = torch.empty(B, device=dev, dtype=torch.int32)
    flt = torch.empty(B, device=dev, dtype=torch.int32)
    fp = torch.from_numpy(filt_ptr).to(dev) if filt_ptr is not None else None
    fi = torch.from_numpy(filt_idx).to(dev) if filt_idx is not None and len(filt_idx) else None
    if fp is not None and fi is None:  # no other answers anywhere: empty lists
        fi = torch.zeros(1, device=dev, dtype=torch.int32)
    _lib.call("regcn_rank_f32", _lib.fptr(s, "score"), B, N, _lib.iptr(tgt, "target"), _lib.iptr(fp), _lib.iptr(fi),
              _lib.iptr(raw), _lib.iptr(flt), _lib.stream())
    return raw.long(), flt.long()


FILTERED_SCORE = -10000000.0  # rgcn/utils.py:60, :74


def apply_filter_(score, filt_ptr, filt_idx):
    """Write -1e7 into `score[b, filt_idx[filt_ptr[b]:filt_ptr[b+1]]]` in place, as
    filter_score / filter_score_r do (rgcn/utils.py:51-75): one device index_put."""
    if filt_idx is None or len(filt_idx) == 0:
        return score
    counts = np.diff(filt_ptr).astype(np.int64)
    rows = torch.from_numpy(np.repeat(np.arange(len(counts), dtype=np.int64), counts)).to(score.device)
    cols = torch.from_numpy(filt_idx.astype(np.int64)).to(score.device)
    score[rows, cols] = FILTERED_SCORE
    return score


def sort_and_rank(score, target):
    """rgcn/utils.py:21-25: 0-based position of the target among the candidates."""
    return ranks(score, target)[0] - 1


def get_total_rank(test_triples, score, all_ans, eval_bz, rel_predict=0):
    """rgcn/utils.py:136-166.  eval_bz only batched the reference's sorts; one launch here."""
    col = {1: 1, 2: 0}.get(int(rel_predict), 2)
    target = test_triples[:, col]
    fp, fi = _filter_csr(test_triples, all_ans, bool(rel_predict))
    rank, filter_rank = ranks(score, target, fp, fi)
    apply_filter_(score, fp, fi)
    mrr = torch.mean(1.0 / rank.float())
    filter_mrr = torch.mean(1.0 / filter_rank.float())
    return filter_mrr.item(), mrr.item(), rank, filter_rank


_SAMPLE_MAX_COLS = 1 << 24
_SAMPLE_MAX_DRAWS = 1 << 30


def _row_limits(value, whole):
    """A limit's values per row as the kernel reads them, none narrowed: whole numbers clamped to int32, others in fp32
    where that holds their type, else fp64."""
    if whole:
        if value.is_floating_point():
            value = value.nan_to_num(0.0).clamp(0.0, 2.0 ** 30)
        if value.dtype != torch.int32:
            value = value.to(torch.int64).clamp(0, 2 ** 31 - 1).to(torch.int32)
    elif value.dtype in (torch.bfloat16, torch.float16):
        value = value.float()
    elif value.dtype != torch.float32:
        value = value.double()
    return value.contiguous()


def _limit(value, name, rows, device, whole, low, high, high_in=True):
    """(number, device tensor of one per row or None) of a sampling limit."""
    if isinstance(value, torch.Tensor) and value.dim() > 0:
        if value.shape != (rows,) or value.device != device:
            raise ValueError("%s must be one number or a tensor of %d on %s (got %s on %s)"
                             % (name, rows, device, tuple(value.shape), value.device))
        return 0, _row_limits(value, whole)
    v = float(value)
    if not (low <= v < high or high_in and v == high):
        raise ValueError("%s must lie between %g and %g (got %r)" % (name, low, high, value))
    return v, None


def sample(score, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, return_logp=False):
    """Ids drawn from scores (B x N, or N for one row; fp32, bf16 or fp16) at the numbers u in [0, 1)
    (B, or B x S for S draws a row; fp32 or fp64), one HIP launch a call (regcn_sample).  Per row, with
    weights w = exp((score - max) / temperature): in the order "larger score first, ties by lower id" are
    kept the first `top_k` (0: all), of those the shortest prefix holding `top_p` of their weight, and of
    those w >= `min_p` (the first is always kept); a draw is the lowest id whose running sum, by id, of kept
    weights exceeds u times their sum.  Weights are rounded to multiples of 2^-S, S = min(51, 63 - ceil(log2 N)), and
    their sums are exact, so equal inputs give equal ids on every call.  The rounding moves at most N 2^-(S+1) of
    probability: 2^-33 at 32,768 scores, 2^-24 at a million, 2^-16 at the most, 2^24, where scores 28 T below the largest
    are never drawn.

    NaN and -inf scores are never drawn and a row of them gives -1; temperature 0 takes the best id.
    temperature, top_k, top_p and min_p may each be a tensor of one value per row, fp64 ones in full (not checked: a
    temperature that is not above 0 takes the best id, top_k <= 0, top_p >= 1 and min_p <= 0 are off).
    Returns int64 ids in u's shape, with return_logp also the log of each draw's probability among the
    kept (fp32, -inf where the id is -1)."""
    if not isinstance(score, torch.Tensor) or not isinstance(u, torch.Tensor):
        raise TypeError("sample takes tensors (score: %s, u: %s)" % (type(score).__name__, type(u).__name__))
    if score.dim() not in (1, 2) or u.dim() > score.dim():
        raise ValueError("score is B x N with u of B or B x S, or N with u of S or one number (got %s, %s)"
                         % (tuple(score.shape), tuple(u.shape)))
    if score.dtype not in _lib.DTYPES:
        raise TypeError("score must be float32, bfloat16 or float16 (got %s)" % score.dtype)
    if u.dtype not in (torch.float32, torch.float64):
        raise TypeError("u must be float32 or float64 (got %s)" % u.dtype)
    rows = score.shape[0] if score.dim() == 2 else 1
    if score.dim() == 2 and (u.dim() == 0 or u.shape[0] != rows):
        raise ValueError("u has %s, score %d rows" % (tuple(u.shape), rows))
    cols = score.shape[-1]
    if cols > _SAMPLE_MAX_COLS:
        raise ValueError("rows of up to %d scores (got %d)" % (_SAMPLE_MAX_COLS, cols))
    if rows > 2 ** 31 - 1 or rows and u.numel() // rows > _SAMPLE_MAX_DRAWS:
        raise ValueError("fewer than 2^31 rows and up to %d draws a row (got %d, %d)"
                         % (_SAMPLE_MAX_DRAWS, rows, u.numel() // rows))
    dev = score.device
    t, t_rows = _limit(temperature, "temperature", rows, dev, False, 0.0, float("inf"), False)
    k, k_rows = _limit(top_k, "top_k", rows, dev, True, 0, 2 ** 31 - 1)
    p, p_rows = _limit(top_p, "top_p", rows, dev, False, 0.0, 1.0)
    m, m_rows = _limit(min_p, "min_p", rows, dev, False, 0.0, 1.0)
    if not score.is_cuda or u.device != dev:
        raise ValueError("score and u must live on one HIP device (got %s, %s); the HIP path has no CPU fallback"
                         % (dev, u.device))
    score, u = score.detach(), u.detach().contiguous()
    if cols > 1 and score.stride(-1) != 1 or rows > 1 and score.stride(0) < cols:
        score = score.contiguous()
    ids = torch.empty(u.shape, device=dev, dtype=torch.int64)
    logp = torch.empty(u.shape, device=dev, dtype=torch.float32) if return_logp else None
    draws = u.numel() // rows if rows else 0
    if cols == 0:
        ids.fill_(-1)
        if return_logp:
            logp.fill_(-float("inf"))
    elif draws:
        d = _lib.SampleDesc()
        d.score, d.ld, d.rows, d.cols, d.draws = score.data_ptr(), score.stride(0) if rows > 1 else cols, rows, cols, draws
        d.dtype, d.u, d.u_wide, d.top_k = _lib.DTYPES[score.dtype], u.data_ptr(), u.dtype == torch.float64, int(k)
        d.temperature, d.top_p, d.min_p, d.ids = t, p, m, ids.data_ptr()
        for name, v in (("temperature_rows", t_rows), ("top_k_rows", k_rows), ("top_p_rows", p_rows),
                        ("min_p_rows", m_rows), ("logp", logp)):
            if v is not None:
                setattr(d, name, v.data_ptr())
        d.rows_wide = sum(b for b, v in ((1, t_rows), (2, p_rows), (4, m_rows)) if v is not None and v.dtype == torch.float64)
        d.ws_bytes = _lib.lib().regcn_sample_workspace_bytes(rows, cols, d.dtype)
        if d.ws_bytes:
            ws = torch.empty(d.ws_bytes, device=dev, dtype=torch.uint8)
            d.workspace = ws.data_ptr()
        _lib.launch("regcn_sample", dev, ctypes.byref(d))
    return (ids, logp) if return_logp else ids


def stat_ranks(rank_list, method):
    """rgcn/utils.py:169-178."""
    total_rank = torch.cat(rank_list)
    mrr = torch.mean(1.0 / total_rank.float())
    print("MRR ({}): {:.6f}".format(method, mrr.item()))
    for hit in (1, 3, 10):
        print("Hits ({}) @ {}: {:.6f}".format(method, hit, torch.mean((total_rank <= hit).float()).item()))
    return mrr


def construct_snap(test_triples, num_nodes, num_rels, final_score, topK):
    """rgcn/utils.py:367-381: the top-k predicted objects as next-history triples."""
    _, idx = torch.sort(final_score, dim=1, descending=True)
    top = idx[:, :topK].cpu().numpy()
    tri = test_triples.cpu().numpy()
    out = []
    for (h, r, _), cand in zip(tri.tolist(), top.tolist()):
        for o in cand:
            out.append([h, r, o] if r < num_rels else [o, r - num_rels, h])
    return np.array(out, dtype=int).reshape(-1, 3)


def construct_snap_r(test_triples, num_nodes, num_rels, final_score, topK):
    """rgcn/utils.py:383-406: the top-k predicted relations as next-history triples."""
    _, idx = torch.sort(final_score, dim=1, descending=True)
    top = idx[:, :topK].cpu().numpy()
    tri = test_triples.cpu().numpy()
    out = []
    for (h, _, t), cand in zip(tri.tolist(), top.tolist()):
        for r in cand:
            out.append([h, r, t] if r < num_rels else [t, r - num_rels, h])
    return np.array(out, dtype=int).reshape(-1, 3)


def construct_snap_sampled(test_triples, num_nodes, num_rels, final_score, draws, u=None, relation=False, **limits):
    """`construct_snap` (relation: `construct_snap_r`) with drawn answers in place of the top k: the
    distinct ids of `draws` draws a query (`sample` with its limits, at the numbers u, B x draws, or fresh
    uniform ones) as next-history triples, in increasing id.  A query without an answer adds none."""
    B = final_score.shape[0]
    if u is None:
        u = torch.rand(B, draws, device=final_score.device, dtype=torch.float64)
    ids = sample(final_score, u.reshape(B, draws), **limits).cpu().numpy()
    tri = test_triples.cpu().numpy()
    out = []
    for (h, r, t), drawn in zip(tri.tolist(), ids):
        for x in np.unique(drawn[drawn >= 0]).tolist():
            if relation:
                out.append([h, x, t] if x < num_rels else [t, x - num_rels, h])
            else:
                out.append([h, r, x] if r < num_rels else [x, r - num_rels, h])
    return np.array(out, dtype=int).reshape(-1, 3)


def load_all_answers_for_filter(total_data, num_rel, rel_p=False):
    """rgcn/utils.py:264-283: {s: {r: {o}}, o: {r + R: {s}}} (or {s: {o: {r}}} for
    relation prediction) over one snapshot's triples."""
    all_ans = {}
    for s, r, o in np.asarray(total_data)[:, :3].tolist():
        if rel_p:
            all_ans.setdefault(s, {}).setdefault(o, set()).add(r)
            all_ans.setdefault(o, {}).setdefault(s, set()).add(r + num_rel)
        else:
            all_ans.setdefault(o, {}).setdefault(r + num_rel, set()).add(s)
            all_ans.setdefault(s, {}).setdefault(r, set()).add(o)
    return all_ans


def split_by_time(data):
    """rgcn/utils.py:306-339: consecutive runs of equal time (column 3; the data is in time
    order, as the reference requires) as (s, r, o) snapshots."""
    data = np.asarray(data)
    if len(data) == 0:
        return []
    cuts = np.nonzero(np.diff(data[:, 3]))[0] + 1
    return [chunk[:, :3].copy() for chunk in np.split(data, cuts)]


def load_all_answers_for_time_filter(total_data, num_rels, num_nodes, rel_p=False):
    """rgcn/utils.py:286-303: one filter dict per snapshot."""
    return [load_all_answers_for_filter(snap, num_rels, rel_p) for snap in split_by_time(total_data)]
