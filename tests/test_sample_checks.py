"""Refusals of ranking.sample and its C entry (no GPU: every call raises before it reaches one)."""
import ctypes

import pytest
import torch

from regcn_amd import _lib, ranking

S, U = torch.zeros(3, 10), torch.zeros(3)


@pytest.mark.parametrize("args,kw,err", [
    ((S, U), {}, ValueError), ((S.numpy(), U), {}, TypeError), ((S, 0.5), {}, TypeError), ((S.double(), U), {}, TypeError),
    ((S, U.half()), {}, TypeError), ((S[None], U), {}, ValueError), ((S, U[:2]), {}, ValueError), ((S[0], S), {}, ValueError),
    ((S, torch.tensor(0.5)), {}, ValueError), ((S, U), dict(temperature=-1.0), ValueError),
    ((S, U), dict(temperature=float("nan")), ValueError), ((S, U), dict(temperature=float("inf")), ValueError),
    ((S, U), dict(top_k=-1), ValueError), ((S, U), dict(top_p=1.5), ValueError), ((S, U), dict(top_p=-0.1), ValueError),
    ((S, U), dict(min_p=2.0), ValueError), ((S, U), dict(min_p=float("nan")), ValueError),
    ((S, U), dict(top_p=torch.ones(2)), ValueError),
    ((torch.zeros(1, 1).expand(1, (1 << 24) + 1), U[:1]), {}, ValueError)])
def test_sample_refuses(args, kw, err):
    with pytest.raises(err):
        ranking.sample(*args, **kw)


def test_c_entry_refuses():
    lib = _lib.lib()
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.addressof(buf)

    def call(**kw):
        d = _lib.SampleDesc()
        d.score, d.u, d.ids, d.ld, d.rows, d.cols, d.draws, d.temperature, d.top_p = p, p, p, 10, 3, 10, 1, 1.0, 1.0
        for k, v in kw.items():
            setattr(d, k, v)
        return lib.regcn_sample(ctypes.byref(d), None)

    for kw in (dict(score=None), dict(u=None), dict(ids=None), dict(rows=-1), dict(cols=-2), dict(draws=-1), dict(dtype=3),
               dict(dtype=-1), dict(ld=9), dict(cols=(1 << 24) + 1, ld=1 << 25)):
        assert call(**kw) < 0, kw
    assert b"sample" in lib.regcn_last_error_string()
    assert call(rows=0) == 0 and call(draws=0) == 0
    assert lib.regcn_sample(None, None) < 0
    assert lib.regcn_sample_workspace_bytes(0, 0, 0) >= 0


@pytest.mark.parametrize("flag,value", [("--sample-draws", "-1"), ("--sample-temperature", "-0.5"), ("--sample-temperature", "inf"),
                                        ("--sample-temperature", "nan"), ("--sample-top-k", "-2"), ("--sample-top-p", "1.5"),
                                        ("--sample-top-p", "-0.1"), ("--sample-min-p", "2")])
def test_the_command_refuses(flag, value):
    """Before it loads anything."""
    from regcn_amd import cli
    with pytest.raises(ValueError, match="--sample"):
        cli.main(["-d", "synthetic:icews14s_lgcn_roth", "--test", "--multi-step", "--sample-draws", "4", flag, value])


def test_limits_per_row_are_not_narrowed():
    limit = lambda v, whole: ranking._limit(v, "it", len(v), v.device, whole, 0, 1)[1]  # noqa: E731
    got = limit(torch.tensor([2 ** 32 + 5, -2 ** 40, 2 ** 31 - 1, -1, 7]), True)
    assert got.dtype == torch.int32 and got.tolist() == [2 ** 31 - 1, 0, 2 ** 31 - 1, 0, 7]
    assert limit(torch.tensor([5, 100], dtype=torch.int8), True).tolist() == [5, 100]
    assert limit(torch.tensor([float("nan"), float("inf"), 3.0, -2.0]), True).tolist() == [0, 2 ** 30, 3, 0]
    fine = torch.tensor([0.9, 1e-50], dtype=torch.float64)
    assert torch.equal(limit(fine, False), fine) and limit(fine, False).dtype == torch.float64
    for dt in (torch.float32, torch.float16, torch.bfloat16):
        assert limit(fine.to(dt), False).dtype == torch.float32 and torch.equal(limit(fine.to(dt), False), fine.to(dt).float())
    assert limit(torch.tensor([2 ** 24 + 1]), False).tolist() == [2 ** 24 + 1]


def test_sizes_past_int32_are_refused():
    """Not passed on as what is left of them in 32 bits."""
    one = torch.zeros(1, 1)
    for score, u in ((one.expand(1 << 31, 1), torch.zeros(1).expand(1 << 31)), (one, one.expand(1, (1 << 30) + 1)),
                     (one, one.expand(1, (1 << 32) + 1)), (one[0], one[0].expand((1 << 30) + 1))):
        with pytest.raises(ValueError, match="2\\^31"):
            ranking.sample(score, u)
    lib = _lib.lib()
    p = ctypes.addressof(ctypes.create_string_buffer(4096))
    d = _lib.SampleDesc(score=p, u=p, ids=p, ld=10, rows=1, cols=10, draws=(1 << 30) + 1, temperature=1.0, top_p=1.0)
    assert lib.regcn_sample(ctypes.byref(d), None) < 0
