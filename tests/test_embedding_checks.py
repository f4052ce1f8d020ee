"""Refusals of autograd.embedding and its C entries (no GPU: every call raises before it reaches one)."""
import ctypes

import pytest
import torch

from regcn_amd import _lib
from regcn_amd import autograd as A

T = torch.zeros(4, 8)
I = torch.zeros(3, dtype=torch.int64)


@pytest.mark.parametrize("args,kw,err", [
    ((T.numpy(), I), {}, TypeError), ((T, [0, 1]), {}, TypeError), ((T[0], I), {}, ValueError),
    ((T.double(), I), {}, TypeError), ((T.to(torch.int32), I), {}, TypeError), ((T, I.float()), {}, TypeError),
    ((T, I.to(torch.int16)), {}, TypeError), ((T, I), {}, ValueError)])
def test_embedding_refuses(args, kw, err):
    with pytest.raises(err):
        A.embedding(*args, **kw)


def test_c_entries_refuse():
    lib = _lib.lib()
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.cast(buf, ctypes.c_void_p)
    assert lib.regcn_embedding(p, 8, p, 1, 4, 16, -1, 0, 1.0, p, None) < 0
    assert lib.regcn_embedding(p, 8, p, 1, -4, 16, 8, 0, 1.0, p, None) < 0
    assert lib.regcn_embedding(p, 8, p, 1, 4, 16, 8, 3, 1.0, p, None) < 0
    assert lib.regcn_embedding(p, 7, p, 1, 4, 16, 8, 0, 1.0, p, None) < 0       # rows overlap
    assert lib.regcn_embedding(p, 8, None, 1, 4, 16, 8, 0, 1.0, p, None) < 0
    assert lib.regcn_embedding(None, 8, p, 1, 4, 16, 8, 0, 1.0, p, None) < 0
    assert lib.regcn_embedding(p, 8, p, 1, 1 << 31, 16, 8, 0, 1.0, p, None) < 0
    assert lib.regcn_embedding(p, 8, p, 1, 0, 16, 8, 0, 1.0, None, None) == 0    # no tokens: nothing to do
    need = lib.regcn_embedding_grad_workspace_bytes(4, 16, 8)
    assert need > 0
    assert lib.regcn_embedding_grad(p, p, 1, 4, 16, 8, -1, 0, 1.0, p, p, need - 1, None) < 0
    assert lib.regcn_embedding_grad(p, p, 1, 4, 16, 8, -1, 0, 1.0, p, None, need, None) < 0
    assert lib.regcn_embedding_grad(p, p, 1, 4, 1 << 31, 8, -1, 0, 1.0, p, p, need, None) < 0
    assert lib.regcn_embedding_grad(p, p, 1, 4, 16, 0, -1, 0, 1.0, p, p, need, None) < 0
    assert b"embedding" in lib.regcn_last_error_string()


@pytest.mark.parametrize("n,V,d", [(0, 1, 1), (1, 1, 1), (63, 5, 3), (16384, 10, 200), (16385, 10, 200),
                                   (1 << 20, 1 << 20, 1024)])
def test_workspace_grows(n, V, d):
    f = _lib.lib().regcn_embedding_grad_workspace_bytes
    assert 0 < f(n, V, d) <= f(n + 1, V, d) <= f(n + 1, V + 100, d + 8)


@pytest.mark.parametrize("shape,n", [((1, 1 << 31), 3), ((1 << 31, 1), 3), ((4, 8), 1 << 31), ((1, (1 << 32) + 5), 3)])
def test_sizes_past_int32_are_refused(shape, n):
    """Not passed on as what is left of them in 32 bits."""
    with pytest.raises(ValueError, match="fewer than 2\\^31"):
        A.embedding(torch.zeros(1, 1).expand(shape), torch.zeros(1, dtype=torch.int64).expand(n))


def test_c_entries_refuse_wide_rows():
    lib = _lib.lib()
    p = ctypes.addressof(ctypes.create_string_buffer(4096))
    assert lib.regcn_embedding(p, 0x7fffffff, p, 1, 4, 16, 0x7fffffff, 0, 1.0, p, None) < 0
    assert lib.regcn_embedding_grad(p, p, 1, 4, 16, 0x7fffffff, -1, 0, 1.0, p, p, 1 << 62, None) < 0
