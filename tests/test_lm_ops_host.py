"""Refusals of ops.embedding, gated_scan, gated_scan_step and residual_norm, and of their C entry
points, on a host without a GPU."""
import ctypes

import pytest
import torch

from mk_iii_technologies_tsrn_b200 import _lib, ops


def test_cpu_tensors_are_refused():
    w, ids = torch.randn(5, 4), torch.zeros(2, 3, dtype=torch.int64)
    x = torch.randn(1, 3, 4)
    for call in (lambda: ops.embedding(ids, w), lambda: ops.embedding_bwd(ids, x, 5),
                 lambda: ops.gated_scan(x, x), lambda: ops.residual_norm(x, x),
                 lambda: ops.gated_scan_step(x[0], x[0], x[0])):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_choices_are_checked_first():
    x = torch.randn(1, 3, 4)
    with pytest.raises(ValueError, match="form"):
        ops.gated_scan(x, x, form="tanh")
    with pytest.raises(ValueError, match="form"):
        ops.gated_scan_step(x[0], x[0], x[0], form="tanh")
    with pytest.raises(ValueError, match="padding_idx"):
        ops.embedding(torch.zeros(2, dtype=torch.int64), torch.randn(5, 4), padding_idx=5)


@pytest.fixture
def lib():
    lib = _lib.load()
    old = lib.tp_set_pointer_checks(0)
    yield lib
    lib.tp_set_pointer_checks(old)


P = ctypes.c_void_p(4096)


def _res_fwd(lib, dtype=0, pd=0, norm=0, rows=2, D=8, x=P, ldx=8, gate=None, ldg=0, bn=0, bw=None,
             eps=1e-5, y=P, stats=None):
    return lib.tp_residual_norm_fwd(dtype, pd, norm, rows, D, x, ldx, P, 8, gate, ldg, None, 0, bn,
                                    bw, None, None, None, eps, y, None, stats, None)


def test_residual_norm_entry_refuses(lib):
    assert _res_fwd(lib, rows=-1) == -1 and _res_fwd(lib, D=0) == -1
    assert _res_fwd(lib, dtype=2) == -4 and _res_fwd(lib, pd=5) == -4
    assert _res_fwd(lib, D=8193) == -4 and _res_fwd(lib, norm=2) == -1
    assert _res_fwd(lib, eps=-1.0) == -1 and _res_fwd(lib, eps=float("nan")) == -1
    assert _res_fwd(lib, ldx=-8) == -1 and _res_fwd(lib, gate=P, ldg=-1) == -1
    assert _res_fwd(lib, bw=P) == -1                      # a branch weight without a branch norm
    assert _res_fwd(lib, x=None) == -2 and _res_fwd(lib, y=None) == -2
    assert _res_fwd(lib, stats=ctypes.c_void_p(4100)) == -3
    assert _res_fwd(lib, rows=0, x=None, y=None) == 0
    assert lib.tp_residual_norm_bwd_workspace_bytes(-1, 8) == -1
    assert lib.tp_residual_norm_bwd_workspace_bytes(4, 9000) == -1
    need = lib.tp_residual_norm_bwd_workspace_bytes(4, 8)
    assert need > 0

    def bwd(gate=None, dgate=None, dscale=None, dbw=None, dx=P, stats=P, ws=P, n=need):
        return lib.tp_residual_norm_bwd(0, 0, 0, 4, 8, P, 8, P, 8, gate, 8, None, 0, 0, None, None,
                                        None, None, 1e-5, stats, P, P, dx, P, dgate, dscale, dbw,
                                        None, None, None, ws, n, None)

    assert bwd(ws=None) == -7 and bwd(n=need - 1) == -7
    assert bwd(dgate=P) == -1 and bwd(dscale=P) == -1 and bwd(dbw=P) == -1
    assert bwd(gate=P) == -2 and bwd(dx=None) == -2 and bwd(stats=None) == -2


def test_gated_scan_entries_refuse(lib):
    def fwd(dtype=0, form=0, B=1, T=2, C=4, gate=P, sb=8, h=P):
        return lib.tp_gated_scan_fwd(dtype, form, B, T, C, gate, sb, 4, P, 8, 4, None, None, h,
                                     None, None, None, 0, None)

    assert fwd(B=-1) == -1 and fwd(T=-1) == -1 and fwd(C=-1) == -1 and fwd(sb=-1) == -1
    assert fwd(dtype=2) == -4 and fwd(form=2) == -1 and fwd(gate=None) == -2 and fwd(h=None) == -2
    assert fwd(B=0, gate=None, h=None) == 0 and fwd(C=0, gate=None, h=None) == 0
    assert fwd(B=2 ** 40) == -5
    # one row of few channels over a long time is cut in time: runs in a workspace
    need = lib.tp_gated_scan_workspace_bytes(1, 65536, 8)
    assert need > 0 and need % (2 * 8 * 4) == 0
    assert lib.tp_gated_scan_workspace_bytes(64, 1024, 640) == 0
    assert lib.tp_gated_scan_workspace_bytes(-1, 1, 1) == -1
    assert fwd(T=65536, C=8) == -7

    def bwd(states=P, dgate=P, form=1):
        return lib.tp_gated_scan_bwd(0, form, 1, 2, 4, P, 8, 4, P, 8, 4, None, states, None, None,
                                     dgate, P, None, None, 0, None)

    assert bwd(states=None) == -2 and bwd(dgate=None) == -2 and bwd(form=-1) == -1

    def step(dtype=0, form=0, B=2, C=4, lds=4, state=P):
        return lib.tp_gated_scan_step(dtype, form, B, C, P, 4, P, 4, state, lds, P, None)

    assert step(lds=3) == -1 and step(lds=0) == -1 and step(state=None) == -2
    assert step(dtype=7) == -4 and step(form=3) == -1 and step(B=-2) == -1
    assert step(B=0, state=None) == 0
    assert lib.tp_gated_scan_states_floats(2, 65, 3) == 2 * 2 * 3
    assert lib.tp_gated_scan_states_floats(2, 0, 3) == 0
    assert lib.tp_gated_scan_states_floats(-1, 0, 3) == -1


def test_embedding_entries_refuse(lib):
    def fwd(dtype=0, bits=64, N=4, T=2, D=8, ids=P, V=5, pw=None, L=0, ldp=0, pos=None, out=P):
        return lib.tp_embedding_fwd(dtype, bits, N, T, D, ids, P, V, 8, 1.0, pw, L, ldp, pos, out,
                                    None)

    assert fwd(N=-1) == -1 and fwd(V=-1) == -1 and fwd(bits=16) == -1 and fwd(dtype=2) == -4
    assert fwd(ids=None) == -2 and fwd(out=None) == -2
    assert fwd(pos=P) == -1                                    # positions without a table
    assert fwd(pw=P, L=1, ldp=8, T=2) == -1                    # more positions than rows
    assert fwd(pw=P, L=4, ldp=-8) == -1 and fwd(pw=P, L=4, ldp=8, T=0) == -1
    assert fwd(N=0, ids=None, out=None) == 0

    need = lib.tp_embedding_bwd_workspace_bytes(4, 5, 8)
    assert need > 0 and lib.tp_embedding_bwd_workspace_bytes(4, 2 ** 31, 8) == -1

    def bwd(dtype=0, bits=64, N=4, V=5, ids=P, dw=P, ws=P, n=need):
        return lib.tp_embedding_bwd(dtype, bits, N, 8, ids, P, V, 1.0, -1, dw, ws, n, None)

    assert bwd(dtype=2) == -4 and bwd(bits=8) == -1 and bwd(N=2 ** 31) == -5
    assert bwd(V=2 ** 31) == -5 and bwd(dw=None) == -2 and bwd(ids=None) == -2
    assert bwd(ws=None) == -7 and bwd(n=need - 1) == -7 and bwd(ws=ctypes.c_void_p(4104)) == -3
    assert bwd(V=0, dw=None, ws=None) == 0

    def pos(N=4, T=2, L=3, dp=P):
        return lib.tp_embedding_pos_bwd(0, N, T, 8, P, L, dp, None)

    assert pos(T=3) == -1 and pos(T=0) == -1 and pos(L=1) == -1 and pos(dp=None) == -2
    assert pos(L=0, N=0) == 0 and pos(L=2 ** 31) == -5


def test_sorted_order_of_the_item_list():
    """The gradient's item list (the tokens of row 0, the end of row 0, the tokens of row 1, ...):
    token j is item keys[j] + j, so the tokens among the first d items are found by bisection."""
    import bisect
    import random
    rng = random.Random(0)
    for _ in range(50):
        V, n = rng.randint(1, 12), rng.randint(0, 30)
        keys = sorted(rng.randint(0, V) for _ in range(n))     # V: not in the table
        items, j = [], 0
        for v in range(V + 1):
            while j < n and keys[j] == v:
                items.append("token")
                j += 1
            if v < V:
                items.append("end")
        assert len(items) == n + V
        at = [k + i for i, k in enumerate(keys)]
        for d in range(n + V + 1):
            assert bisect.bisect_left(at, d) == items[:d].count("token")


def test_pointer_checks_of_one_thread():
    import threading
    lib = _lib.load()
    assert lib.tp_set_thread_pointer_checks(0) == 1
    other = []
    t = threading.Thread(target=lambda: other.append(lib.tp_set_thread_pointer_checks(1)))
    t.start()
    t.join()
    assert other == [1]                                   # another thread's are on
    assert lib.tp_set_thread_pointer_checks(1) == 0
