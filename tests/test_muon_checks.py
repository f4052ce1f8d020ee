"""Refusals of muon.orthogonalize and its C entries (no GPU: every call raises before it reaches one)."""
import ctypes

import pytest
import torch

from regcn_amd import _lib, muon

G = torch.zeros(4, 8)


@pytest.mark.parametrize("g,kw,err", [
    (G, {}, ValueError), (G.double(), {}, TypeError), (G[0], {}, ValueError), (G.numpy(), {}, TypeError),
    ([G, None], {}, TypeError), (G, dict(steps=0), ValueError), (G, dict(steps=2000), ValueError),
    (G, dict(coeffs=(3.0, 0.0, 0.0)), ValueError), (G, dict(coeffs=(1.0, 2.0)), ValueError),
    (G, dict(coeffs=(float("nan"), 0.0, 0.0)), ValueError), (G, dict(coeffs=(20.0, -40.0, 20.0)), ValueError), (G, dict(eps=-1.0), ValueError),
    (G, dict(eps=float("inf")), ValueError), ([G.view(2, 2, 8)], {}, ValueError)])
def test_orthogonalize_refuses(g, kw, err):
    with pytest.raises(err):
        muon.orthogonalize(g, **kw)


def test_c_entries_refuse():
    lib = _lib.lib()
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.cast(buf, ctypes.c_void_p)

    def mats(**kw):
        m = (_lib.Matrix * 1)()
        m[0].x, m[0].out, m[0].rows, m[0].cols, m[0].dtype = p, p, 4, 8, 0
        for k, v in kw.items():
            setattr(m[0], k, v)
        return m

    need = lib.regcn_orthogonalize_workspace_bytes(mats(), 1)
    assert need > 0
    call = lambda m, n=1, steps=5, ws=p, size=need: lib.regcn_orthogonalize(m, n, steps, 1.5, -0.5, 0.0, 0.0, ws, size, None)  # noqa: E731
    assert call(mats(), size=need - 1) < 0 and call(mats(), ws=None) < 0 and call(None) < 0
    assert call(mats(), steps=0) < 0 and call(mats(), n=-1) < 0
    for kw in (dict(x=None), dict(out=None), dict(rows=0), dict(cols=-3), dict(rows=1 << 21), dict(dtype=7)):
        assert call(mats(**kw)) < 0, kw
    assert b"orthogonalize" in lib.regcn_last_error_string()
    assert call(mats(), n=0) == 0  # no matrices: nothing to do
    assert lib.regcn_orthogonalize_workspace_bytes(None, 1) == 0
    assert lib.regcn_orthogonalize_workspace_bytes(mats(rows=0), 1) == 0


def test_workspace_is_that_of_the_largest_set():
    """32 matrices go through one set of launches; the sets follow one another in the same workspace."""
    lib = _lib.lib()

    def size(shapes):
        m = (_lib.Matrix * len(shapes))()
        for d, (r, c) in zip(m, shapes):
            d.rows, d.cols = r, c
        return lib.regcn_orthogonalize_workspace_bytes(m, len(shapes))

    one = size([(200, 200)])
    assert size([(200, 200)] * 32) == 32 * one == size([(200, 200)] * 70)
    assert size([(200, 200), (4096, 4096)]) == size([(4096, 4096)])  # the tile sizes are sets of their own


@pytest.mark.parametrize("kw", [dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-0.1), dict(steps=0),
                                dict(coeffs=(4.0, 0.0, 0.0))])
def test_muon_refuses_settings(kw):
    with pytest.raises(ValueError):
        muon.Muon([torch.zeros(2, 2, requires_grad=True)], **kw)


@pytest.mark.parametrize("p", [torch.zeros(3), torch.zeros(2, 2, 2), torch.zeros(2, 2, dtype=torch.float64)])
def test_muon_refuses_parameters(p):
    with pytest.raises(ValueError):
        muon.Muon([p.requires_grad_(True)])


def test_more_steps_take_fp32_operands():
    """A caller of the C entry asks for them by the matrix's type; the workspace follows."""
    lib = _lib.lib()
    p = ctypes.addressof(ctypes.create_string_buffer(4096))

    def mats(rows, dtype):
        m = (_lib.Matrix * 1)()
        m[0].x, m[0].out, m[0].rows, m[0].cols, m[0].dtype = p, p, rows, 300, dtype
        return m
    size = lambda m: lib.regcn_orthogonalize_workspace_bytes(m, 1)  # noqa: E731
    call = lambda m, steps: lib.regcn_orthogonalize(m, 1, steps, 1.5, -0.5, 0.0, 0.0, p, 0, None)  # noqa: E731
    assert call(mats(200, 0), 9) == -2  # REGCN_ENOTSUP
    assert b"REGCN_FULL_FP32" in lib.regcn_last_error_string()
    for m, steps in ((mats(200, 0), 8), (mats(200, _lib.FULL_FP32), 9), (mats(64, 0), 9)):
        assert call(m, steps) == -1 and b"workspace" in lib.regcn_last_error_string()
    assert size(mats(200, 1 | _lib.FULL_FP32)) > 0 and size(mats(200, 3 | _lib.FULL_FP32)) == 0
    assert size(mats(64, 0)) == size(mats(64, _lib.FULL_FP32))


def test_a_state_without_momentum_loads():
    """Of a parameter that has not stepped yet."""
    opt = muon.Muon([torch.zeros(2, 3, requires_grad=True)])
    opt.state[opt.param_groups[0]["params"][0]] = {}
    again = muon.Muon([torch.zeros(2, 3, requires_grad=True)])
    again.load_state_dict(opt.state_dict())
    assert not any(again.state.values())
