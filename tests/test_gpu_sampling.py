"""Sampling against the definition in 64 bits on the host.  Tokens are whole numbers: the random
numbers keep off the borders of the running sums by 1e-9 of the whole (the kernel's weights are
rounded to 2^-45 of the best's, 2^17 of them to 4e-9 at the very most and 1e-11 in the mean), so that
both sides must give the same one."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _rule(x, u, T, k, p, m):
    """(token, log of its share, distance of the choices from their borders) of one row."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    if x.max() == -np.inf:
        return -1, math.nan, 1.0
    order = np.argsort(-x, kind="stable")
    if not T > 0:
        return int(order[0]), 0.0, 1.0
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == x.max(), 1.0, np.exp((x[order] - x.max()) / T))
    w[x[order] == -np.inf] = 0.0
    far = 1.0
    n = len(w) if k <= 0 else min(len(w), k)
    if p < 1:
        sums = np.cumsum(w[:n]) / w[:n].sum()
        far = np.abs(sums[:-1] - p).min() if n > 1 else 1.0
        n = max(1, int((np.concatenate(([0.0], sums[:-1])) < p).sum()))
    n = max(1, min(n, int((w >= m).sum())))
    kept = np.sort(order[:n])
    with np.errstate(invalid="ignore"):
        q = np.where(x[kept] == x.max(), 1.0, np.exp((x[kept] - x.max()) / T))
    sums = np.cumsum(q) / q.sum()
    far = min(far, np.abs(sums[:-1] - u).min() if n > 1 else 1.0)
    i = min(int((sums <= u).sum()), int(np.flatnonzero(q)[-1]))
    return int(kept[i]), math.log(q[i] / q.sum()), far


def _check(logits, u, T=1.0, k=0, p=1.0, m=0.0, **kw):
    from mk_iii_technologies_tsrn_b200 import ops
    token, logprob = ops.sample_tokens(logits, u, temperature=T, top_k=k, top_p=p, min_p=m, return_logprob=True)
    assert torch.equal(token, ops.sample_tokens(logits, u, temperature=T, top_k=k, top_p=p, min_p=m))
    x, un = logits.float().cpu().numpy(), u.double().cpu().numpy()
    row = lambda c, b: float(c[b]) if isinstance(c, torch.Tensor) else c
    close = 0
    for b in range(len(x)):
        want, lp, far = _rule(x[b], un[b], row(T, b), int(row(k, b)), row(p, b), row(m, b))
        if far < 1e-9:
            close += 1
            continue
        assert int(token[b]) == want, (b, int(token[b]), want)
        # rounded once to float32; weights to 2^-45 of the best's
        if want >= 0:
            assert abs(float(logprob[b]) - lp) <= abs(lp) * 2.0 ** -23 + 1e-9
        else:
            assert math.isnan(float(logprob[b]))
    assert close <= 1 + len(x) // 8
    return token


def _logits(dev, B, V, dtype, seed=0, spread=3.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (spread * torch.randn(B, V, device=dev, generator=g)).to(dtype), torch.rand(B, device=dev, generator=g)


CHOICES = [
    dict(),
    dict(T=0.7),
    dict(T=0.0),
    dict(k=1),
    dict(k=5),
    dict(k=50, p=0.9),
    dict(k=50, p=0.9, m=0.05),
    dict(p=0.5),
    dict(p=0.95, T=1.3),
    dict(m=0.1),
    dict(p=0.9999),
    dict(k=1500),                  # more than are sorted
    dict(k=1200, p=0.97),
    dict(T=30.0, p=0.8),           # flat: the threshold is searched for
    dict(T=30.0, k=1100, p=0.3, m=0.5),
    dict(T=0.01, p=0.9),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(3, 1), (5, 7), (4, 256), (2, 5001), (3, 49999), (1, 131072), (2, 200001)], ids=str)
def test_matches_the_rule(cuda, shape, dtype):
    for i, c in enumerate(CHOICES):
        _check(*_logits(cuda, *shape, dtype, seed=i), **c)


def test_every_request_its_own(cuda):
    B = 24
    for dtype in (torch.float32, torch.bfloat16):
        x, u = _logits(cuda, B, 3001, dtype)
        i = torch.arange(B, device=cuda)
        T = torch.where(i % 5 == 0, 0.0, 0.3 + 0.05 * i)
        k = torch.where(i % 3 == 0, 0, 3 + 70 * i)
        p = torch.where(i % 2 == 0, 1.0, 0.3 + 0.02 * i)
        m = torch.where(i % 4 == 0, 0.0, 0.001 * i)
        _check(x, u, T, k.int(), p, m)
        _check(x, u, T, k, p, m)                           # 64-bit counts too
        _check(x, u, 0.8, k.int(), 0.9, m)


def test_many_rows(cuda):
    _check(*_logits(cuda, 700, 300, torch.float32), k=20, p=0.8)


def test_ties_go_to_the_lowest_index(cuda):
    from mk_iii_technologies_tsrn_b200 import ops
    x = torch.zeros(1, 5000, device=cuda)
    x[0, 100:4000:3] = 2.0                                 # 1300 equals
    first = list(range(100, 4000, 3))
    u = torch.tensor([0.9999], device=cuda)
    assert int(ops.sample_tokens(x, u, top_k=7)) == first[6]
    assert int(ops.sample_tokens(x, u, top_k=1200)) == first[1199]
    assert int(ops.sample_tokens(x, u * 0, top_k=1200)) == first[0]
    assert int(ops.sample_tokens(x, u, top_k=1250, top_p=0.5)) == first[624]
    assert int(ops.sample_tokens(x, u, temperature=0)) == first[0]
    assert int(ops.sample_tokens(x, u, top_p=1e-6)) == first[0]
    # (0.7 of 600 equal weights is a border in 64 bits too: 420 tokens have less before them)
    nine = torch.arange(9, device=cuda) / 9 + 0.01
    want = [first[int(t * 420)] for t in nine.double().tolist()]
    assert ops.sample_tokens(x.expand(9, -1), nine, top_k=600, top_p=0.7).tolist() == want
    half = torch.randn(4, 3000, device=cuda).mul(2).round().div(2).bfloat16()
    for c in (dict(k=100), dict(k=2000, p=0.9), dict(p=0.3), dict(k=100, p=0.6, m=0.2)):
        _check(half, torch.rand(4, device=cuda, generator=torch.Generator(device=cuda).manual_seed(1)), **c)


def test_masked_tokens_and_rows(cuda):
    x, u = _logits(cuda, 6, 4000, torch.float32)
    x[0] = float("-inf")
    x[1] = float("nan")
    x[2, 5:] = float("-inf")
    x[3, ::2] = float("nan")
    x[4, 17] = x[4, 3000] = float("inf")
    x[5] = torch.finfo(torch.float32).min
    x[5, 9] = 0.0
    for c in (dict(), dict(k=3), dict(p=0.9), dict(k=2000), dict(m=0.3), dict(T=0.0), dict(T=40.0, p=0.99)):
        t = _check(x, u, **c)
        assert t[0] == -1 and t[1] == -1 and int(t[2]) < 5 and int(t[3]) % 2 == 1
        assert int(t[4]) in (17, 3000) and int(t[5]) == 9


def test_random_numbers_at_the_ends(cuda):
    from mk_iii_technologies_tsrn_b200 import ops
    x = torch.zeros(6, 10, device=cuda)
    x[:, 8:] = float("-inf")
    u = torch.tensor([0.0, 0.9999999, 1.0, 1.5, -0.5, float("nan")], device=cuda)
    for c in (dict(), dict(top_p=0.99), dict(min_p=0.5)):
        assert ops.sample_tokens(x, u, **c).tolist() == [0, 7, 7, 7, 0, 7]
    assert ops.sample_tokens(x, u.double(), top_k=4).tolist() == [0, 3, 3, 3, 0, 3]


def test_strided_logits(cuda):
    from mk_iii_technologies_tsrn_b200 import ops
    big, u = _logits(cuda, 4, 1003, torch.bfloat16)
    for x in (big[:, 1:1000], big[::2, 3:], big[:, ::2], big[:1].expand(3, -1)):
        _check(x, u[:len(x)].contiguous(), k=30, p=0.9)
    two = torch.stack((u, u), 1)[:, 0]
    assert torch.equal(ops.sample_tokens(big, two), ops.sample_tokens(big, u))


def test_counts_follow_the_weights(cuda):
    # 2^17 even random numbers give every token its share of them, up to the one at each end
    from mk_iii_technologies_tsrn_b200 import ops
    w = torch.tensor([0.5, 0.125, 0.25, 0.0625, 0.0625], device=cuda)
    n = 2 ** 17
    u = (torch.arange(n, device=cuda, dtype=torch.float64) + 0.5) / n
    t = ops.sample_tokens(w.log().expand(n, -1).contiguous(), u)
    assert ((torch.bincount(t, minlength=5) - w * n).abs() <= 1).all()


def test_best_tokens_next_to_one_another(cuda):
    # the best tokens lie in a few threads' parts of the row, or in one part of it
    for V, n in ((131072, 700), (50000, 300), (8192, 2000)):
        for dtype in (torch.float32, torch.bfloat16):
            x, u = _logits(cuda, 3, V, dtype, seed=V)
            x[0, 1000:1000 + n] += 30.0
            x[1, ::2] = float("-inf")
            x[1, 40:] = float("-inf")                     # twenty tokens
            x[2, :n] = 9.0                                # and equal ones
            for c in (dict(k=100), dict(k=30, p=0.8), dict(k=900), dict(p=0.9), dict(p=0.5, T=3.0), dict(k=250, m=0.1)):
                _check(x, u, **c)


def test_flat_rows(cuda):
    # logits of an untrained model: every token in the nucleus, the border between close values
    for dtype in (torch.float32, torch.bfloat16):
        for spread in (1e-3, 0.05, 0.5):
            x, u = _logits(cuda, 3, 40000, dtype, spread=spread)
            for c in (dict(p=0.9), dict(p=0.3, m=0.999), dict(k=5000), dict(k=5000, p=0.5), dict(k=40)):
                _check(x, u, **c)
