"""ops.embedding (scaled token embedding with position rows) and its gradient by sorted tokens.

Forward: the kernel rounds the product and the sum one by one in fp32 (bf16: once more at the
end), as the torch expression below does, so the bits are equal.  Gradient: a sum of n rows in
fp32, scaled once and rounded to the table's type: with u = 2^-24 each of at most n + 1 additions
and the product lose at most u of a partial sum, so the error is at most (n + 2) u scale sum|d|,
plus half a step of the type of the result."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
TYPES = [torch.float32, torch.bfloat16]


def _gen(dev, seed=0):
    return torch.Generator(device=dev).manual_seed(seed)


def _plain(ids, w, scale, pos=None, positions=None):
    out = w.float()[ids.long()] * scale
    if pos is not None:
        at = positions.long() if positions is not None else torch.arange(ids.shape[-1],
                                                                         device=ids.device)
        out = out + pos.float()[at]
    return out.to(w.dtype)


def _check_grad(got, ids, dout, rows, scale, padding_idx=None):
    """Against the sum in 64 bits with the bound of the docstring."""
    D = dout.shape[-1]
    flat, d = ids.reshape(-1).long().cpu(), dout.reshape(-1, D).double().cpu()
    keep = (flat >= 0) & (flat < rows)
    if padding_idx is not None:
        keep &= flat != padding_idx
    flat, d = flat[keep], d[keep]
    ref = torch.zeros(rows, D, dtype=torch.float64).index_add_(0, flat, d) * scale
    mag = torch.zeros(rows, D, dtype=torch.float64).index_add_(0, flat, d.abs()) * abs(scale)
    n = torch.bincount(flat, minlength=rows).double()[:, None]
    tol = (n + 2) * U * mag * 1.01 + HALF[got.dtype] * ref.abs() * 1.01
    err = (got.double().cpu() - ref).abs()
    assert torch.all(err <= tol), float((err - tol).max())
    absent = torch.bincount(flat, minlength=rows) == 0
    assert torch.all(got.cpu()[absent] == 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,V,D", [((1, 1), 1, 1), ((3, 5), 7, 8), ((2, 33), 300, 40),
                                       ((64, 1), 1000, 512), ((4, 129), 50, 129),
                                       ((5, 7), 11, 1028), ((2, 600), 97, 640), ((9,), 5, 3)])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_forward_bits(cuda, dtype, shape, V, D, index):
    from mk_iii_technologies_tsrn_b200 import ops
    g = _gen(cuda)
    ids = torch.randint(0, V, shape, device=cuda, generator=g, dtype=index)
    w = torch.randn(V, D, device=cuda, generator=g).to(dtype)
    T = shape[-1]
    pos = torch.randn(T + 3, D, device=cuda, generator=g).to(dtype)
    at = torch.randint(0, T + 3, shape, device=cuda, generator=g)
    s = D ** 0.5
    assert torch.equal(ops.embedding(ids, w, s), _plain(ids, w, s))
    assert torch.equal(ops.embedding(ids, w, s, pos_weight=pos), _plain(ids, w, s, pos))
    assert torch.equal(ops.embedding(ids, w, s, pos_weight=pos, positions=at),
                       _plain(ids, w, s, pos, at))


def test_forward_strides_and_broadcast_positions(cuda):
    from mk_iii_technologies_tsrn_b200 import ops
    g = _gen(cuda, 1)
    ids = torch.randint(0, 40, (6, 10), device=cuda, generator=g)
    table = torch.randn(40, 100, device=cuda, generator=g)
    pos = torch.randn(50, 64, device=cuda, generator=g)
    for w in (table[:, 4:68], table[:, 3:67], table[::2][:, :64], torch.randn(
            64, 40, device=cuda, generator=g).t()):
        i = ids % w.shape[0]
        assert torch.equal(ops.embedding(i.t(), w, 2.5), _plain(i.t(), w, 2.5))
        at = torch.tensor([[7], [0], [49], [3], [3], [21]], device=cuda, dtype=torch.int32)
        assert torch.equal(ops.embedding(i, w, 2.5, pos_weight=pos, positions=at),
                           _plain(i, w, 2.5, pos, at.expand(6, 10)))


def test_empty(cuda):
    from mk_iii_technologies_tsrn_b200 import ops
    w = torch.randn(5, 8, device=cuda, requires_grad=True)
    p = torch.randn(4, 8, device=cuda, requires_grad=True)
    ids = torch.empty(3, 0, device=cuda, dtype=torch.int64)
    out = ops.embedding(ids, w, 2.0, pos_weight=p)
    assert out.shape == (3, 0, 8)
    gw, gp = torch.autograd.grad(out, (w, p), torch.empty_like(out))
    assert torch.all(gw == 0) and torch.all(gp == 0)


def test_out_of_range_ids(cuda):
    from mk_iii_technologies_tsrn_b200 import ops
    g = _gen(cuda, 2)
    w = torch.randn(10, 12, device=cuda, generator=g, requires_grad=True)
    ids = torch.tensor([[3, -1, 9], [10, 0, 2 ** 40]], device=cuda)
    out = ops.embedding(ids, w, 2.0)
    with pytest.raises(ops.DeviceIndexError):
        ops.check_device_error(cuda)
    bad = torch.tensor([[False, True, False], [True, False, True]], device=cuda)
    assert torch.all(out[bad].isnan()) and torch.equal(out[~bad], w[ids[~bad]] * 2.0)
    dout = torch.randn_like(out)
    _check_grad(torch.autograd.grad(out, w, dout)[0], ids, dout, 10, 2.0)
    pos = torch.randn(4, 12, device=cuda)
    out = ops.embedding(torch.zeros(2, 1, device=cuda, dtype=torch.int64), w.detach(), 1.0,
                        pos_weight=pos, positions=torch.tensor([[4], [3]], device=cuda))
    with pytest.raises(ops.DeviceIndexError):
        ops.check_device_error(cuda)
    assert torch.all(out[0].isnan()) and torch.equal(out[1, 0], w[0] + pos[3])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V,D", [(1, 1, 1), (1, 100000, 8), (40, 3, 24), (256, 256, 33),
                                   (2047, 2047, 16), (2049, 2048, 16), (5000, 70000, 20),
                                   (30000, 5, 12), (9001, 256, 640), (700, 4200000, 4),
                                   (4100, 300, 1500)])
def test_gradient(cuda, dtype, N, V, D):
    from mk_iii_technologies_tsrn_b200 import ops
    g = _gen(cuda, N + V)
    # a third of the tokens share one id, the others are spread
    ids = torch.randint(0, V, (N,), device=cuda, generator=g)
    ids = torch.where(torch.rand(N, device=cuda, generator=g) < 0.33, V // 2, ids)
    dout = torch.randn(N, D, device=cuda, generator=g).to(dtype)
    dw = ops.embedding_bwd(ids, dout, V, 1.7)
    _check_grad(dw, ids, dout, V, 1.7)
    assert torch.equal(dw, ops.embedding_bwd(ids, dout, V, 1.7))
    if V > 1:
        _check_grad(ops.embedding_bwd(ids.int(), dout, V, 1.0, padding_idx=V // 2), ids, dout, V,
                    1.0, V // 2)


@pytest.mark.parametrize("ids_of", ["same", "sorted", "reversed", "last", "first"])
def test_gradient_of_skewed_ids(cuda, ids_of):
    from mk_iii_technologies_tsrn_b200 import ops
    N, V, D = 20000, 30000, 36
    ids = {"same": torch.full((N,), 12345), "sorted": torch.arange(N),
           "reversed": torch.arange(N).flip(0), "last": torch.full((N,), V - 1),
           "first": torch.zeros(N, dtype=torch.int64)}[ids_of].to(cuda)
    dout = torch.randn(N, D, device=cuda, generator=_gen(cuda, 3))
    _check_grad(ops.embedding_bwd(ids, dout, V), ids, dout, V, 1.0)


def test_gradient_keeps_the_order_of_tokens(cuda):
    # 1 + 2^-24 steps are lost one by one after a large row, and kept before it: only the order of
    # the tokens gives these sums
    from mk_iii_technologies_tsrn_b200 import ops
    d = torch.ones(9, 1, device=cuda) * 2.0 ** -24
    up, down = d.clone(), d.clone()
    up[0], down[-1] = 1.0, 1.0
    ids = torch.full((9,), 2, device=cuda)
    assert ops.embedding_bwd(ids, up, 4)[2].item() == 1.0
    assert ops.embedding_bwd(ids, down, 4)[2].item() == 1.0 + 8 * 2.0 ** -24


def test_gradient_with_non_finite_rows(cuda):
    from mk_iii_technologies_tsrn_b200 import ops
    dout = torch.ones(4, 8, device=cuda)
    dout[1], dout[2] = float("inf"), float("nan")
    dw = ops.embedding_bwd(torch.tensor([0, 3, 9, 0], device=cuda), dout, 5)
    assert torch.all(dw[0] == 2) and torch.all(dw[3].isinf()) and torch.all(dw[[1, 2, 4]] == 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,T,D,L", [(1, 1, 1, 1), (3, 17, 40, 20), (65, 9, 33, 9), (2, 5, 640, 8)])
def test_autograd(cuda, dtype, B, T, D, L):
    from mk_iii_technologies_tsrn_b200 import ops
    g = _gen(cuda, B)
    V = 23
    ids = torch.randint(0, V, (B, T), device=cuda, generator=g)
    w = torch.randn(V, D, device=cuda, generator=g).to(dtype).requires_grad_()
    p = torch.randn(L, D, device=cuda, generator=g).to(dtype).requires_grad_()
    dout = torch.randn(B, T, D, device=cuda, generator=g).to(dtype)
    rows = torch.arange(T, device=cuda).expand(B, T)
    gw, gp = torch.autograd.grad(ops.embedding(ids, w, 3.0, pos_weight=p, padding_idx=-1), (w, p),
                                 dout)
    _check_grad(gw, ids, dout, V, 3.0, V - 1)
    _check_grad(gp, rows, dout, L, 1.0)
    at = torch.randint(0, L, (B, 1), device=cuda, generator=g)
    gp, = torch.autograd.grad(ops.embedding(ids, w.detach(), 3.0, pos_weight=p, positions=at), p,
                              dout)
    _check_grad(gp, at.expand(B, T), dout, L, 1.0)


def test_gradient_against_differences(cuda):
    # the operator is linear in its tables: a step along v changes it by the gradient's product
    # with v exactly, up to the rounding of the two forwards (a few u of the outputs each)
    from mk_iii_technologies_tsrn_b200 import ops
    g = _gen(cuda, 5)
    ids = torch.randint(0, 50, (4, 30), device=cuda, generator=g)
    w = torch.randn(50, 16, device=cuda, generator=g, requires_grad=True)
    v = torch.randn(50, 16, device=cuda, generator=g)
    dout = torch.randn(4, 30, 16, device=cuda, generator=g)
    gw, = torch.autograd.grad(ops.embedding(ids, w, 2.0), w, dout)
    with torch.no_grad():
        diff = (ops.embedding(ids, w + v, 2.0).double() - ops.embedding(ids, w - v, 2.0).double())
    want = (diff * dout.double()).sum() / 2
    size = ((w.abs() + v.abs()).detach()[ids].double() * 2 * dout.abs().double()).sum()
    assert abs(float((gw.double() * v.double()).sum() - want)) <= 64 * U * float(size)


def test_captured_and_replayed(cuda):
    from mk_iii_technologies_tsrn_b200 import ops
    g = _gen(cuda, 6)
    ids = torch.randint(0, 500, (8, 300), device=cuda, generator=g)
    dout = torch.randn(8, 300, 64, device=cuda, generator=g)
    side = torch.cuda.Stream(cuda)
    with torch.cuda.stream(side):
        ops.embedding_bwd(ids, dout, 500)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dw = ops.embedding_bwd(ids, dout, 500)
    for seed in (7, 8):
        ids.copy_(torch.randint(0, 500, (8, 300), device=cuda, generator=_gen(cuda, seed)))
        graph.replay()
        assert torch.equal(dw, ops.embedding_bwd(ids, dout, 500))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [33, 40, 1095, 2056])
def test_every_row_of_a_sparse_gradient_is_written(cuda, dtype, D):
    # runs of absent rows of all lengths, before, between and behind the tokens' rows, over a
    # buffer of NaN; one id very often, so that some shares hold tokens alone
    from mk_iii_technologies_tsrn_b200 import _lib
    lib = _lib.load()
    g = torch.Generator(device=cuda).manual_seed(3)
    V, rows = 4000, torch.tensor([3, 4, 6, 9, 13, 18, 30, 700, 701, 3990], device=cuda)
    ids = torch.cat((rows, rows[4].expand(3000), rows[torch.randint(0, 10, (90,), device=cuda,
                                                                    generator=g)]))
    N = ids.numel()
    dout = torch.randint(-8, 9, (N, D), device=cuda, generator=g).to(dtype)    # sums are exact
    dw = torch.full((V * D + 8,), float("nan"), device=cuda, dtype=dtype)
    need = lib.tp_embedding_bwd_workspace_bytes(N, V, D)
    ws = torch.full((need,), 255, device=cuda, dtype=torch.uint8)
    st = lib.tp_embedding_bwd(0 if dtype == torch.float32 else 1, 64, N, D, ids.data_ptr(),
                              dout.data_ptr(), V, 1.0, -1, dw.data_ptr(), ws.data_ptr(), need,
                              torch.cuda.current_stream().cuda_stream)
    assert st == 0
    want = torch.zeros(V, D, device=cuda, dtype=torch.float64).index_add_(0, ids, dout.double())
    assert torch.equal(dw[:V * D].view(V, D), want.to(dtype)) and torch.all(dw[V * D:].isnan())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("B,T,D", [(2, 3, 12), (5, 40, 33), (12, 7, 8), (70, 60, 16),
                                   (1100, 250, 4)])
def test_token_outside_one_table_adds_to_neither_gradient(cuda, dtype, index, B, T, D):
    # bad ids at good positions and good ids at bad positions, with the NaN that their rows of the
    # output send back; the tokens left in sum as if the others were not there
    from mk_iii_technologies_tsrn_b200 import ops
    g = _gen(cuda, B)
    V, L, scale = 19, T + 2, 2.0
    ids = torch.randint(0, V, (B, T), device=cuda, generator=g).to(index)
    at = torch.randint(0, L, (B, T), device=cuda, generator=g).to(index)
    bad_id = torch.rand(B, T, device=cuda, generator=g) < 0.2
    bad_at = torch.rand(B, T, device=cuda, generator=g) < 0.2
    bad_id[0, 1], bad_at[0, 0], bad_id[0, 0] = True, True, False
    ids[bad_id] = torch.where(ids[bad_id] % 2 == 0, -1, V).to(index)
    w = torch.randn(V, D, device=cuda, generator=g).to(dtype).requires_grad_()
    p = torch.randn(L, D, device=cuda, generator=g).to(dtype).requires_grad_()
    dout = torch.randn(B, T, D, device=cuda, generator=g).to(dtype)
    rows = torch.arange(T, device=cuda).expand(B, T)
    for positions, where, bad in ((None, rows, bad_id),
                                  (torch.where(bad_at, L + 3, at.long()).to(index), at,
                                   bad_id | bad_at)):
        out = ops.embedding(ids, w, scale, pos_weight=p, positions=positions)
        with pytest.raises(ops.DeviceIndexError):
            ops.check_device_error(cuda)
        assert torch.equal(out.isnan().any(-1), bad)
        d = torch.where(bad[..., None], float("nan"), dout)
        gw, gp = torch.autograd.grad(out, (w, p), d)
        _check_grad(gw, torch.where(bad, -1, ids.long()), dout, V, scale)
        _check_grad(gp, torch.where(bad, -1, where.long()), dout, L, 1.0)


def test_padding_counted_from_the_end(cuda):
    from mk_iii_technologies_tsrn_b200 import ops
    g = _gen(cuda, 8)
    ids = torch.randint(0, 6, (50,), device=cuda, generator=g)
    dout = torch.randn(50, 8, device=cuda, generator=g)
    for p in (-1, -6, -2):
        _check_grad(ops.embedding_bwd(ids, dout, 6, padding_idx=p), ids, dout, 6, 1.0, p + 6)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V", [(40000, 300), (40000, 70000), (40000, 4200000), (262144, 1023),
                                 (262145, 1023), (300000, 300), (300000, 70000),
                                 (300000, 4200000)])
def test_gradient_of_many_tokens(cuda, dtype, N, V):
    # sorts of one, two and three digits, by a cluster of 16 blocks and by two kernels a digit
    from mk_iii_technologies_tsrn_b200 import ops
    g = _gen(cuda, N + V)
    ids = torch.randint(0, V, (N,), device=cuda, generator=g)
    ids = torch.where(torch.rand(N, device=cuda, generator=g) < 0.25, V // 2, ids)
    ids[::1001] = V + 5                                       # in no table
    dout = torch.randn(N, 4, device=cuda, generator=g).to(dtype)
    dw = ops.embedding_bwd(ids, dout, V, 1.7)
    _check_grad(dw, ids, dout, V, 1.7)
    assert torch.equal(dw, ops.embedding_bwd(ids.int(), dout, V, 1.7))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [2367, 2368, 40001])
@pytest.mark.parametrize("D", [37, 40, 512, 1028])
def test_forward_of_many_tokens(cuda, dtype, N, D):
    # four rows at a time, four vectors of a longer row, single channels
    from mk_iii_technologies_tsrn_b200 import ops
    g = _gen(cuda, D)
    ids = torch.randint(0, 999, (N,), device=cuda, generator=g)
    at = torch.randint(0, 50, (N,), device=cuda, generator=g)
    w = torch.randn(999, D, device=cuda, generator=g).to(dtype)
    pos = torch.randn(50, D, device=cuda, generator=g).to(dtype)
    assert torch.equal(ops.embedding(ids, w, 1.5), _plain(ids, w, 1.5))
    assert torch.equal(ops.embedding(ids, w, 1.5, pos_weight=pos, positions=at),
                       _plain(ids, w, 1.5, pos, at))


def test_gradient_of_a_table_of_2_to_the_30_rows(cuda):
    # keys of 31 bits: more digits than the cluster's sort takes, with few tokens too
    from mk_iii_technologies_tsrn_b200 import ops
    g = _gen(cuda, 9)
    for N in (1500, 5000):
        V = 2 ** 30 + 3
        ids = torch.randint(0, V, (N,), device=cuda, generator=g)
        ids[::3] = V - 1
        dout = torch.randint(-8, 9, (N, 1), device=cuda, generator=g).bfloat16()
        dw = ops.embedding_bwd(ids, dout, V)
        rows, where = torch.unique(ids, return_inverse=True)
        want = torch.zeros(len(rows), device=cuda).index_add_(0, where, dout[:, 0].float())
        assert torch.equal(dw[rows, 0], want.bfloat16())
        assert int(torch.count_nonzero(dw)) == int(torch.count_nonzero(want))
        del dw
