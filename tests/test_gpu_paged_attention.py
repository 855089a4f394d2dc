"""Paged attention of one new token, and the writing of prompts, against the definition in 64 bits.

Tolerance of the attention, counted in roundings (u = 2^-24): a score in units of its exponent is a
sum of D products, each rounded, and four more steps, so it is off by at most
(D + 6) u * scale / tau * sum_f |q_f k_f| (the tropical part by less: a sum and a maximum); its base-2
form by 2 u |s|; the exponential by 2^-22 relative.  A softmax weight is then off by a factor of
exp(2 d) for scores off by d, and sums of n weights by n u more; the output by that times the
largest |v|, and a bf16 output by half a step, 2^-8 of its value, more.

bf16 weights are multiplied with V as two bf16 parts: rounding p to the first leaves at most 2^-8 p,
rounding that rest to the second at most 2^-8 of it, so 2^-16 p is lost; over a row that is at most
2^-16 sum p |v| <= 2^-16 max |v|."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _cache(dev, B, L, Hkv, D, page, dtype, layout="slots", seed=0, spare=2, wide=0):
    """Random caches and a table of scattered pages; `wide`: rows lie that many channels apart."""
    g = torch.Generator(device=dev).manual_seed(seed)
    per = max(1, -(-L // page))
    pages = B * per + spare
    table = torch.randperm(pages, device=dev, generator=g)[:B * per].view(B, per).int()
    shape = (pages, page, Hkv, D + wide) if layout == "slots" else (pages, Hkv, page, D + wide)
    k, v = (torch.randn(shape, device=dev, generator=g).to(dtype)[..., :D] for _ in range(2))
    if layout == "heads":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    return k, v, table, g


def _rows(cache, table, b, n):
    page = cache.shape[1]
    return cache[table[b, :-(-n // page)].long()].flatten(0, 1)[:n].double()


def _reference(q, k, v, table, lengths, scale, gate=None, tau=None):
    """(out, weights [B][H, n], largest error of a score in its exponent's units) in 64 bits."""
    B, H, D = q.shape
    G = H // k.shape[2]
    out = torch.zeros(B, H, D, dtype=torch.float64, device=q.device)
    weights, off = [], torch.zeros(B, H, device=q.device, dtype=torch.float64)
    for b, n in enumerate(lengths.tolist()):
        if n == 0:
            weights.append(None)
            continue
        kb, vb = (_rows(c, table, b, n).transpose(0, 1).repeat_interleave(G, 0) for c in (k, v))
        qb = q[b].double()[:, None]
        s = (kb * qb).sum(-1)
        if gate is not None:
            t = (kb + qb).amax(-1)
            g = gate[b].double()[:, None]
            s = g * t + (1 - g) * s
        f = scale / (tau.double() if tau is not None else torch.ones(H, device=q.device).double())
        s = s * f[:, None]
        w = torch.softmax(s, -1)
        out[b] = (w[..., None] * vb).sum(1)
        weights.append(w)
        off[b] = ((D + 6) * U * f * (kb * qb).abs().sum(-1).amax(-1) + 2 * U * s.abs().amax(-1) + 2.0 ** -22
                  + 0.5 * n * U)
    return out, weights, off


def _check(o, want, off, v, dtype):
    top = v.double().abs().max()
    tol = 2 * off[..., None] * top * torch.ones_like(want)
    if dtype == torch.bfloat16:
        tol = tol + want.abs() * 2.0 ** -8 + top * 2.0 ** -16
    bad = (o.double() - want).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} off, worst {(o.double() - want).abs().max():.3g}"


def _check_mass(mass, before, weights, lengths, off, H, Hkv, fresh):
    G = H // Hkv
    for b, n in enumerate(lengths.tolist()):
        want = before[b].double().clone()
        if n:
            if fresh:
                want[:, n - 1] = 0.0
            want[:, :n] += weights[b].view(Hkv, G, n).sum(1)
            tol = G * 2 * off[b].max() + (G + 2) * U * want.abs()
            assert ((mass[b].double() - want).abs() <= tol).all()
        assert torch.equal(mass[b, :, n:], before[b, :, n:])       # behind the end: as it was


CASES = [
    # B, H, Hkv, D, L, page, layout
    (1, 1, 1, 1, 1, 1, "slots"),
    (3, 8, 8, 64, 100, 16, "slots"),
    (2, 12, 4, 80, 333, 24, "heads"),
    (2, 8, 1, 128, 1000, 7, "slots"),
    (3, 6, 3, 32, 65, 16, "heads"),
    (1, 32, 8, 128, 5000, 64, "slots"),
    (2, 5, 5, 256, 129, 33, "slots"),
    (2, 9, 3, 33, 77, 5, "heads"),
    (2, 16, 1, 96, 515, 16, "slots"),
    (1, 4, 2, 250, 200, 16, "slots"),
    (40, 4, 4, 8, 50, 16, "slots"),
    (1, 34, 2, 64, 20000, 16, "slots"),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_matches_the_definition(cuda, case, gated, dtype):
    from mk_iii_technologies_tsrn_b200 import ops
    B, H, Hkv, D, L, page, layout = case
    k, v, table, g = _cache(cuda, B, L, Hkv, D, page, dtype, layout)
    lengths = torch.randint(0, L + 1, (B,), device=cuda, generator=g, dtype=torch.int32)
    lengths[-1] = L
    q = (2 * torch.randn(B, H, D, device=cuda, generator=g)).to(dtype)
    gate = tau = None
    if gated:
        gate = torch.rand(B, H, device=cuda, generator=g)
        tau = 0.5 + torch.rand(H, device=cuda, generator=g)
    mass = torch.rand(B, Hkv, table.shape[1] * page, device=cuda, generator=g)
    before = mass.clone()
    want, weights, off = _reference(q, k, v, table, lengths, D ** -0.5, gate, tau)
    o = ops.paged_attention(q, k, v, table, lengths, gate=gate, tau=tau)
    _check(o, want, off, v, dtype)
    o2 = ops.paged_attention(q, k, v, table, lengths, gate=gate, tau=tau, mass=mass)
    assert torch.equal(o, o2)
    _check_mass(mass, before, weights, lengths, off, H, Hkv, False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", [(3, 8, 8, 64, 100, 16, "slots"), (2, 12, 4, 80, 333, 24, "heads"),
                                  (2, 10, 2, 33, 40, 3, "slots"), (5, 32, 8, 128, 700, 16, "slots")], ids=str)
def test_new_token_counts_and_is_stored(cuda, case, dtype):
    from mk_iii_technologies_tsrn_b200 import ops
    B, H, Hkv, D, L, page, layout = case
    k, v, table, g = _cache(cuda, B, L, Hkv, D, page, dtype, layout)
    lengths = torch.randint(1, L + 1, (B,), device=cuda, generator=g, dtype=torch.int32)
    lengths[0] = 1
    q, key, value = (torch.randn(B, h, D, device=cuda, generator=g).to(dtype) for h in (H, Hkv, Hkv))
    wide = torch.randn(B, 2, 3 * Hkv, D, device=cuda, generator=g).to(dtype)     # (strided inputs)
    key2 = wide[:, 0, ::3].copy_(key)
    mass = torch.rand(B, Hkv, table.shape[1] * page, device=cuda, generator=g)
    before = mass.clone()
    kw, vw = k.clone(), v.clone()
    for b, n in enumerate(lengths.tolist()):
        at = int(table[b, (n - 1) // page])
        kw[at, (n - 1) % page] = key[b]
        vw[at, (n - 1) % page] = value[b]
        # what was in the slot must not matter
        k[at, (n - 1) % page] = float("nan")
        v[at, (n - 1) % page] = float("nan")
    want, weights, off = _reference(q, kw, vw, table, lengths, 0.3)
    version = k._version
    o = ops.paged_attention(q, k, v, table, lengths.long(), key=key2, value=value, scale=0.3, mass=mass)
    _check(o, want, off, vw, dtype)
    assert torch.equal(k, kw) and torch.equal(v, vw) and k._version > version
    _check_mass(mass, before, weights, lengths, off, H, Hkv, True)


def test_what_lies_behind_the_end_is_not_read(cuda):
    from mk_iii_technologies_tsrn_b200 import ops
    for dtype in (torch.float32, torch.bfloat16):
        for group in (1, 4, 8):
            k, v, table, g = _cache(cuda, 3, 300, 2, 64, 16, dtype)
            lengths = torch.tensor([0, 1, 250], device=cuda, dtype=torch.int32)
            q = torch.randn(3, 2 * group, 64, device=cuda, generator=g).to(dtype)
            want = ops.paged_attention(q, k, v, table, lengths)
            assert bool((want[0] == 0).all())
            used = torch.zeros(k.shape[:2], device=cuda, dtype=torch.bool)
            for b, n in enumerate(lengths.tolist()):
                for j in range(n):
                    used[table[b, j // 16].long(), j % 16] = True
            for junk in (float("nan"), float("inf")):
                k[~used] = junk
                v[~used] = junk
                assert torch.equal(ops.paged_attention(q, k, v, table, lengths), want)
            table2 = table.clone()                       # pages of unused slots are not looked at
            table2[0] = -5
            table2[1, 1:] = 2 ** 30
            assert torch.equal(ops.paged_attention(q, k, v, table2, lengths), want)


def test_infinities_and_nan_in_use(cuda):
    from mk_iii_technologies_tsrn_b200 import ops
    k, v, table, g = _cache(cuda, 4, 600, 1, 64, 16, torch.float32)
    n = torch.full((4,), 600, device=cuda, dtype=torch.int32)
    q = torch.randn(4, 2, 64, device=cuda, generator=g).abs()
    k[table[0].long()] = float("-inf")                   # every score is -inf
    k[table[1, 3].long(), 5, 0, 7] = float("-inf")       # one is
    k[table[2, 30].long(), 2, 0, 9] = float("nan")
    k[table[3, 30].long(), 2, 0, 9] = float("inf")
    o = ops.paged_attention(q, k, v, table, n)
    assert bool(o[0].isnan().all()) and bool(o[2].isnan().all()) and bool(o[3].isnan().all())
    want, _, off = _reference(q[1:2], k, v, table[1:2], n[:1], 0.125)
    assert ((o[1:2].double() - want).abs() <= 2 * (65 * U * 20 + 2e-6 + 600 * U) * v.abs().max()).all()


def test_gate_of_zero_and_one(cuda):
    from mk_iii_technologies_tsrn_b200 import ops
    k, v, table, g = _cache(cuda, 2, 90, 2, 48, 16, torch.float32)
    n = torch.tensor([90, 17], device=cuda, dtype=torch.int32)
    q = torch.randn(2, 4, 48, device=cuda, generator=g)
    plain = ops.paged_attention(q, k, v, table, n)
    zero = ops.paged_attention(q, k, v, table, n, gate=torch.zeros(2, 4, device=cuda))
    torch.testing.assert_close(zero, plain, rtol=0, atol=2 * (54 * U * 20 + 1e-6) * float(v.abs().max()))
    one = torch.ones(2, 4, device=cuda)
    want, _, off = _reference(q, k, v, table, n, 48 ** -0.5, one)
    _check(ops.paged_attention(q, k, v, table, n, gate=one), want, off, v, torch.float32)


def test_bad_pages_and_lengths(cuda):
    from mk_iii_technologies_tsrn_b200 import ops
    k, v, table, g = _cache(cuda, 4, 200, 2, 64, 16, torch.float32)
    n = torch.tensor([200, 150, 209, -1], device=cuda, dtype=torch.int32)
    q = torch.randn(4, 2, 64, device=cuda, generator=g)
    key = torch.randn(4, 2, 64, device=cuda, generator=g)
    want, _, off = _reference(q[:1], k, v, table[:1], n[:1], 0.125)
    table2 = table.clone()
    table2[1, 4] = k.shape[0]
    kept = k.clone()
    o = ops.paged_attention(q, k, v, table2, n)
    with pytest.raises(ops.DeviceIndexError):
        ops.check_device_error(cuda)
    _check(o[:1], want, off, v, torch.float32)
    assert bool(o[1:].isnan().all())
    table2[1, 9] = -1                                     # the new token's page
    ops.paged_attention(q, k, v, table2, n, key=key, value=key)
    with pytest.raises(ops.DeviceIndexError):
        ops.check_device_error(cuda)
    kept[table[0, 12].long(), 7] = key[0]
    assert torch.equal(k, kept)
    # mass of fewer slots than the table is a limit too
    mass = torch.zeros(4, 2, 150, device=cuda)
    o = ops.paged_attention(q, k, v, table, torch.tensor([151, 150, 0, 3], device=cuda), mass=mass)
    with pytest.raises(ops.DeviceIndexError):
        ops.check_device_error(cuda)
    assert bool(o[0].isnan().all()) and not bool(o[1:].isnan().any())


def test_shared_pages_may_be_read_by_all(cuda):
    from mk_iii_technologies_tsrn_b200 import ops
    k, v, table, g = _cache(cuda, 2, 100, 2, 64, 16, torch.bfloat16)
    table[1] = table[0]
    n = torch.tensor([100, 40], device=cuda, dtype=torch.int32)
    q = torch.randn(2, 4, 64, device=cuda, generator=g).bfloat16()
    want, _, off = _reference(q, k, v, table, n, 0.125)
    _check(ops.paged_attention(q, k, v, table, n), want, off, v, torch.bfloat16)


def test_rows_at_any_stride(cuda):
    from mk_iii_technologies_tsrn_b200 import ops
    for wide in (1, 3, 8):                                # rows that do not begin on 16 bytes, and do
        k, v, table, g = _cache(cuda, 2, 70, 3, 64, 16, torch.bfloat16, wide=wide)
        n = torch.tensor([70, 33], device=cuda, dtype=torch.int32)
        q = torch.randn(2, 3, 2, 64, device=cuda, generator=g).bfloat16()[:, :, 1]
        want, _, off = _reference(q, k, v, table, n, 0.125)
        _check(ops.paged_attention(q, k, v, table, n), want, off, v, torch.bfloat16)


def test_offsets_beyond_32_bits(cuda):
    # a cache of more than 2^32 bytes (and of 2^31 elements); pages at its far end
    from mk_iii_technologies_tsrn_b200 import ops
    pages, page, D = 70000, 64, 128
    k = torch.empty(pages, page, 4, D, device=cuda, dtype=torch.bfloat16)
    v = torch.empty(pages, page, 4, D, device=cuda, dtype=torch.bfloat16)
    g = torch.Generator(device=cuda).manual_seed(0)
    table = torch.tensor([[pages - 1, 0, pages - 2], [pages // 2 + 1, 5, pages - 3]], device=cuda).int()
    for p in table.flatten().tolist():
        k[p] = torch.randn(page, 4, D, device=cuda, generator=g).bfloat16()
        v[p] = torch.randn(page, 4, D, device=cuda, generator=g).bfloat16()
    n = torch.tensor([192, 130], device=cuda, dtype=torch.int32)
    q = torch.randn(2, 8, D, device=cuda, generator=g).bfloat16()
    want, _, off = _reference(q, k, v, table, n, D ** -0.5)
    _check(ops.paged_attention(q, k, v, table, n), want, off, v[table.long()], torch.bfloat16)
    key = torch.randn(2, 1, 4, D, device=cuda, generator=g).bfloat16()
    ops.paged_append(key, key, k, v, table, n - 1)
    assert torch.equal(k[pages - 2, 63], key[0, 0]) and torch.equal(v[pages - 3, 1], key[1, 0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", [
    # B, H, Hkv, D, L, page, gated
    (3000, 2, 1, 64, 20, 4, False),          # many short sequences, some without a slot
    (3000, 2, 2, 64, 20, 16, True),
    (2, 300, 1, 64, 70, 16, False),          # many query heads of one key head
    (2, 70, 1, 32, 70, 8, True),
    (1, 2, 2, 128, 9000, 1, False),          # pages of one slot
    (3, 4, 4, 64, 4100, 8, True),
    (2, 4, 2, 96, 2000, 128, False),
    (2, 4, 4, 192, 500, 12, False),
], ids=str)
def test_shapes_of_the_cut(cuda, case, dtype):
    from mk_iii_technologies_tsrn_b200 import ops
    B, H, Hkv, D, L, page, gated = case
    k, v, table, g = _cache(cuda, B, L, Hkv, D, page, dtype)
    lengths = torch.randint(0, L + 1, (B,), device=cuda, generator=g, dtype=torch.int32)
    if B > 100:                              # runs of sequences without a slot, at both ends too
        lengths[:40] = 0
        lengths[500:900] = 0
        lengths[-300:] = 0
    q = torch.randn(B, H, D, device=cuda, generator=g).to(dtype)
    key, value = (torch.randn(B, Hkv, D, device=cuda, generator=g).to(dtype) for _ in range(2))
    gate = torch.rand(B, H, device=cuda, generator=g) if gated else None
    mass = torch.rand(B, Hkv, table.shape[1] * page, device=cuda, generator=g)
    some = lengths > 0
    last = (lengths.long() - 1).clamp(min=0)
    at = table.long().gather(1, (last // page)[:, None])[:, 0]
    before, k2, v2, mass2 = mass.clone(), k.clone(), v.clone(), mass.clone()
    o = ops.paged_attention(q, k, v, table, lengths, key=key, value=value, gate=gate, mass=mass)
    assert torch.equal(o, ops.paged_attention(q, k2, v2, table, lengths, key=key, value=value, gate=gate, mass=mass2))
    assert torch.equal(mass, mass2)
    assert torch.equal(k[at, last % page][some], key[some]) and torch.equal(v[at, last % page][some], value[some])
    pick = torch.randperm(B, device=cuda, generator=g)[:40]
    want, weights, off = _reference(q[pick], k, v, table[pick], lengths[pick], D ** -0.5,
                                    gate[pick] if gated else None)
    _check(o[pick], want, off, v, dtype)
    _check_mass(mass[pick], before[pick], weights, lengths[pick], off, H, Hkv, True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_lengths_around_the_tiles(cuda, dtype):
    from mk_iii_technologies_tsrn_b200 import ops
    for page in (16, 24, 64):
        for gated in (False, True):
            n = torch.tensor([1, 7, 8, 9, 15, 16, 17, 31, 32, 33, 47, 48, 49, 63, 64, 65, 96, 97], device=cuda).int()
            k, v, table, g = _cache(cuda, len(n), 97, 2, 64, page, dtype)
            q = torch.randn(len(n), 4, 64, device=cuda, generator=g).to(dtype)
            key = torch.randn(len(n), 2, 64, device=cuda, generator=g).to(dtype)
            gate = torch.rand(len(n), 4, device=cuda, generator=g) if gated else None
            o = ops.paged_attention(q, k, v, table, n, key=key, value=key, gate=gate)
            want, _, off = _reference(q, k, v, table, n, 0.125, gate)      # (the token is stored by now)
            _check(o, want, off, v, dtype)


# ----------------------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", [(3, 5, 2, 64, 16, "slots"), (2, 40, 3, 33, 7, "heads"), (4, 1, 8, 80, 16, "slots"),
                                  (2, 700, 4, 100, 64, "slots"), (1, 3, 1, 1, 1, "slots")], ids=str)
def test_append_writes_what_is_there(cuda, case, dtype):
    from mk_iii_technologies_tsrn_b200 import ops
    B, T, Hkv, D, page, layout = case
    k, v, table, g = _cache(cuda, B, T + 20, Hkv, D, page, dtype, layout)
    key, value = torch.randn(2, B, Hkv, T, D, device=cuda, generator=g).to(dtype).transpose(2, 3)   # (heads before tokens)
    starts = torch.randint(0, 20, (B,), device=cuda, generator=g, dtype=torch.int32)
    counts = torch.randint(0, T + 1, (B,), device=cuda, generator=g)
    for c in (counts, None):
        kw, vw = k.clone(), v.clone()
        for b in range(B):
            for t in range(T if c is None else int(c[b])):
                s = int(starts[b]) + t
                kw[int(table[b, s // page]), s % page] = key[b, t]
                vw[int(table[b, s // page]), s % page] = value[b, t]
        assert ops.paged_append(key, value, k, v, table, starts, c) is None
        assert torch.equal(k, kw) and torch.equal(v, vw)


def test_append_outside_is_not_written(cuda):
    from mk_iii_technologies_tsrn_b200 import ops
    k, v, table, g = _cache(cuda, 3, 32, 2, 64, 16, torch.float32)
    key = torch.randn(3, 4, 2, 64, device=cuda, generator=g)
    kw = k.clone()
    kw[int(table[0, 1]), 14:] = key[0, :2]                # the other two run over the table
    table[1, 0] = 99
    ops.paged_append(key, key, k, v, table, torch.tensor([30, 0, -4], device=cuda))
    with pytest.raises(ops.DeviceIndexError):
        ops.check_device_error(cuda)
    assert torch.equal(k, kw)
