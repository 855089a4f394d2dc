"""Two host threads that call the same C entry points at once, on streams of their own, with sizes
whose launches of one kernel need different amounts of dynamic shared memory.  (ctypes calls run
without the interpreter lock, as the autograd engine's thread does.)"""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

CALLS = 20000


def _both(works):
    """Runs every call of `works` CALLS times, a thread and a stream for each; the statuses seen."""
    seen, go = [set() for _ in works], threading.Barrier(len(works))

    def loop(i, work, stream):
        torch.cuda.set_device(0)
        go.wait()
        for _ in range(CALLS):
            seen[i].add(work(stream.cuda_stream))
        stream.synchronize()

    threads = [threading.Thread(target=loop, args=(i, w, torch.cuda.Stream()))
               for i, w in enumerate(works)]
    torch.cuda.synchronize()
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    return seen


@pytest.mark.parametrize("sizes", [((256, 32), (600, 32)), ((40, 768), (40, 1024))],
                         ids=["sort", "sum"])
def test_embedding_gradient(cuda, sizes):
    from mk_iii_technologies_tsrn_b200 import _lib
    lib, g, N = _lib.load(), torch.Generator(device=cuda).manual_seed(1), 2000
    works, results = [], []
    for V, D in sizes:
        ids = torch.randint(0, V, (N,), device=cuda, generator=g)
        dout = torch.randint(-8, 9, (N, D), device=cuda, generator=g).float()    # sums are exact
        dw = torch.empty(V, D, device=cuda)
        need = lib.tp_embedding_bwd_workspace_bytes(N, V, D)
        ws = torch.empty(need, device=cuda, dtype=torch.uint8)
        results.append((dw, torch.zeros(V, D, device=cuda).index_add_(0, ids, dout)))
        works.append(lambda s, a=(ids, dout, dw, ws), V=V, D=D, need=need: lib.tp_embedding_bwd(
            0, 64, N, D, a[0].data_ptr(), a[1].data_ptr(), V, 1.0, -1, a[2].data_ptr(),
            a[3].data_ptr(), need, s))
    assert _both(works) == [{0}, {0}]
    for got, want in results:
        assert torch.equal(got, want)


def test_residual_backward(cuda):
    from mk_iii_technologies_tsrn_b200 import _lib, ops
    lib, g, R = _lib.load(), torch.Generator(device=cuda).manual_seed(2), 64
    D = 640      # one block for both calls; the sums of four parameters, or of five
    x, b, dy, dn = (torch.randn(R, D, device=cuda, generator=g) for _ in range(4))
    w, bias, scale, bw, bb = (torch.randn(D, device=cuda, generator=g) for _ in range(5))
    stats = ops.residual_norm_fwd(x, b, w, bias, scale=scale, branch_norm=True, branch_weight=bw,
                                  branch_bias=bb, need_stats=True)[2]
    need = lib.tp_residual_norm_bwd_workspace_bytes(R, D)
    works, outs = [], []
    for last in (True, False):
        o = [torch.empty(R, D, device=cuda) for _ in range(2)] + [torch.empty(D, device=cuda)
                                                                  for _ in range(5)]
        ws = torch.empty(need, device=cuda, dtype=torch.uint8)
        outs.append(o)
        works.append(lambda s, o=o, ws=ws, last=last: lib.tp_residual_norm_bwd(
            0, 0, 0, R, D, x.data_ptr(), D, b.data_ptr(), D, None, 0, scale.data_ptr(), 1, 1,
            bw.data_ptr(), bb.data_ptr(), w.data_ptr(), bias.data_ptr(), 1e-5, stats.data_ptr(),
            dy.data_ptr(), dn.data_ptr(), o[0].data_ptr(), o[1].data_ptr(), None, o[2].data_ptr(),
            o[3].data_ptr(), o[4].data_ptr(), o[5].data_ptr(), o[6].data_ptr() if last else None,
            ws.data_ptr(), need, s))
    assert _both(works) == [{0}, {0}]
    want = ops.residual_norm_bwd(stats, dy, dn, x, b, w, bias, scale=scale, branch_norm=True,
                                 branch_weight=bw, branch_bias=bb)
    names = ("x", "branch", "scale", "branch_weight", "branch_bias", "weight", "bias")
    for o, n in zip(outs, (7, 6)):
        for got, k in zip(o[:n], names):
            assert torch.equal(got, want[k]), k
