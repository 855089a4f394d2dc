"""Refusals of the C entries that look at a token's indices in both tables, without a GPU."""
import ctypes

import pytest

from mk_iii_technologies_tsrn_b200 import _lib

P = ctypes.c_void_p(4096)


@pytest.fixture
def lib():
    lib = _lib.load()
    old = lib.tp_set_pointer_checks(0)
    yield lib
    lib.tp_set_pointer_checks(old)


def test_embedding_gradients_of_both_tables_refuse(lib):
    need = lib.tp_embedding_bwd_workspace_bytes(4, 5, 8)

    def bwd(N=4, V=5, other=P, rows=3, dw=P, ws=P, n=need, bits=64):
        return lib.tp_embedding_bwd_both(0, bits, N, 8, P, P, V, 1.0, -1, other, rows, dw, ws, n,
                                         None)

    assert bwd(rows=-1) == -1 and bwd(bits=8) == -1 and bwd(V=2 ** 31) == -5
    assert bwd(dw=None) == -2 and bwd(n=need - 1) == -7 and bwd(V=0, dw=None) == 0

    def pos(T=2, L=3, ids=P, bits=64, V=5, dp=P):
        return lib.tp_embedding_pos_bwd_both(0, 4, T, 8, P, L, ids, bits, V, dp, None)

    assert pos(V=-1) == -1 and pos(bits=8) == -1 and pos(T=3) == -1 and pos(L=1) == -1
    assert pos(dp=None) == -2 and pos(L=0, T=0) == -1
    assert lib.tp_embedding_pos_bwd(0, 2 ** 31, 1, 8, P, 3, P, None) == -5


def test_padding_of_the_table_gradient_is_checked():
    import torch

    from mk_iii_technologies_tsrn_b200 import ops
    ids, dout = torch.zeros(2, dtype=torch.int64), torch.randn(2, 4)
    for bad in (5, -6):
        with pytest.raises(ValueError, match="padding_idx"):
            ops.embedding_bwd(ids, dout, 5, padding_idx=bad)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.embedding_bwd(ids, dout, 5, padding_idx=-5)
