"""Eviction against a loop over sequences and heads: whole numbers and moved rows, so equal bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _case(dev, B, Hkv, D, L, page, dtype, layout, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    per = -(-L // page)
    pages = B * per + 1
    table = torch.randperm(pages, device=dev, generator=g)[:B * per].view(B, per).int()
    shape = (pages, page, Hkv, D) if layout == "slots" else (pages, Hkv, page, D)
    k, v = (torch.randn(shape, device=dev, generator=g).to(dtype) for _ in range(2))
    if layout == "heads":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    mass = torch.exp(2 * torch.randn(B, Hkv, per * page, device=dev, generator=g))
    n = torch.randint(0, L + 1, (B,), device=dev, generator=g, dtype=torch.int32)
    n[-1] = L
    return k, v, table, mass, n


def _want(k, v, table, mass, n, keep, recent):
    B, Hkv = mass.shape[:2]
    page = k.shape[1]
    k2, v2, out = k.clone(), v.clone(), mass.clone()
    kept = torch.full((B, Hkv, keep), -1, dtype=torch.int32)
    host = mass.cpu()
    tab = table.tolist()
    for b in range(B):
        m = int(n[b])
        for h in range(Hkv):
            if m <= keep:
                take = list(range(m))
            else:
                old = m - min(recent, m)
                val = [float("inf") if x != x else x for x in host[b, h, :old].tolist()]
                nan = [x != x for x in host[b, h, :old].tolist()]
                best = sorted(range(old), key=lambda j: (not nan[j], -val[j], j))[:keep - (m - old)]
                take = sorted(best) + list(range(old, m))
            src = torch.tensor(take, dtype=torch.long, device=k.device)
            kept[b, h, :len(take)] = torch.tensor(take, dtype=torch.int32)
            if len(take) == 0:
                continue
            row = torch.tensor(tab[b], device=k.device)
            to = torch.arange(len(take), device=k.device)
            hs = torch.full_like(to, h)
            k2[row[to // page], to % page, hs] = k[row[src // page], src % page, hs]
            v2[row[to // page], to % page, hs] = v[row[src // page], src % page, hs]
            out[b, h, :len(take)] = mass[b, h, src]
    return kept.to(k.device), k2, v2, out


CASES = [
    # B, Hkv, D, L, page, keep, recent, layout
    (3, 2, 64, 100, 16, 40, 10, "slots"),
    (2, 3, 33, 77, 5, 30, 0, "heads"),
    (1, 1, 8, 5, 1, 1, 1, "slots"),
    (2, 2, 128, 3000, 64, 1024, 1024, "slots"),      # the recent ones alone
    (2, 4, 80, 2500, 24, 2499, 7, "heads"),
    (4, 1, 16, 50, 16, 60, 20, "slots"),             # room for all
    (1, 2, 256, 1025, 16, 512, 100, "slots"),
    (1, 1, 4, 9000, 16, 100, 3, "slots"),
    (1, 2, 4, 70000, 64, 40000, 1000, "slots"),      # more than stays in a block's registers
    (1, 1, 1, 33000, 100, 32900, 0, "slots"),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_matches_the_loop(cuda, case, dtype):
    from mk_iii_technologies_tsrn_b200 import ops
    B, Hkv, D, L, page, keep, recent, layout = case
    k, v, table, mass, n = _case(cuda, B, Hkv, D, L, page, dtype, layout)
    kept, k2, v2, out = _want(k, v, table, mass, n, keep, recent)
    apart = torch.full_like(mass, 7.0)
    ka, va = k.clone(), v.clone()
    got = ops.cache_evict(ka, va, table, n, mass, keep, recent, out=apart)
    assert torch.equal(got, kept) and torch.equal(ka, k2) and torch.equal(va, v2)
    live = torch.arange(mass.shape[2], device=cuda) < n.clamp(max=keep)[:, None, None]
    assert torch.equal(torch.where(live, apart, out), out) and bool((apart[~live.expand_as(apart)] == 7).all())
    got = ops.cache_evict(k, v, table, n.long(), mass, keep, recent)           # mass in place
    assert torch.equal(got, kept) and torch.equal(k, k2) and torch.equal(v, v2) and torch.equal(mass, out)


@pytest.mark.parametrize("values", ["equal", "few", "nan", "zeros", "negative"])
def test_ties_and_special_weights(cuda, values):
    from mk_iii_technologies_tsrn_b200 import ops
    k, v, table, mass, n = _case(cuda, 2, 2, 16, 2100, 16, torch.float32, "slots", seed=3)
    if values == "equal":
        mass.fill_(0.5)
    elif values == "few":
        mass.copy_((mass * 2).floor().clamp(max=3))
    elif values == "nan":
        mass[:, :, 10:900:7] = float("nan")
        mass[:, :, 11] = float("inf")
        mass[:, :, 12] = float("-inf")
    elif values == "zeros":
        mass.zero_()
        mass[:, :, ::2] = -0.0                            # equal to 0: the lower slot of them
    else:
        mass.neg_()
    kept, k2, v2, out = _want(k, v, table, mass, n, 1000, 50)
    got = ops.cache_evict(k, v, table, n, mass, 1000, 50)
    assert torch.equal(got, kept) and torch.equal(k, k2) and torch.equal(v, v2)
    assert torch.equal(mass.view(torch.int32), out.view(torch.int32))


def test_bad_lengths_and_pages(cuda):
    from mk_iii_technologies_tsrn_b200 import ops
    k, v, table, mass, n = _case(cuda, 3, 2, 64, 96, 16, torch.float32, "slots")
    n = torch.tensor([96, 97, -2], device=cuda, dtype=torch.int32)
    keepers = torch.tensor([96, 0, 0], device=cuda, dtype=torch.int32)
    kept, k2, v2, out = _want(k, v, table, mass, keepers, 32, 8)
    got = ops.cache_evict(k, v, table, n, mass, 32, 8)
    with pytest.raises(ops.DeviceIndexError):
        ops.check_device_error(cuda)
    assert torch.equal(got, kept) and torch.equal(k, k2) and torch.equal(mass, out)
    k, v, table, mass, n = _case(cuda, 1, 1, 64, 96, 16, torch.float32, "slots")
    before = k.clone()
    table[0, 0], table[0, 1] = -1, k.shape[0]             # where the rows would go
    ops.cache_evict(k, v, table, n, mass, 32, 8)
    with pytest.raises(ops.DeviceIndexError):
        ops.check_device_error(cuda)
    assert torch.equal(k, before)
