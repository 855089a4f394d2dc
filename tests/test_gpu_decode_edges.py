"""Edges of the decoding operators: precision of the weights, clusters of blocks,
infinite values, rows without a channel."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("group", [1, 2, 3, 4])
def test_bf16_weights_keep_their_bits(cuda, group):
    """A slot of weight w and value -1 against two of weight 1 whose values make up for it, in 64 bits
    to 2^-16 or so: what is left is what the weights lost.

    Scores are single products of bf16 numbers, exact; their base-2 form is off by 2 U of a score below
    1, the exponential by 2^-22, so a weight by at most 2^-22 + 3 U of itself.  A sum of n products in
    fp32 is off by at most n 2^-23 of the sum of their sizes (steps may be cut off rather than rounded),
    in the output and in the sum of the weights.  The output is rounded by 2^-8 of its value at most."""
    from mk_iii_technologies_tsrn_b200 import ops
    B, Hkv, D, n = 64, 2, 64, 3
    g = torch.Generator(device=cuda).manual_seed(group)
    x = (0.1 + 0.8 * torch.rand(B, Hkv, device=cuda, generator=g)).bfloat16()
    k = torch.zeros(B, 16, Hkv, D, device=cuda, dtype=torch.bfloat16)
    v = torch.full_like(k, -1.0)
    k[:, 0, :, 0] = -x
    w = torch.exp(-x.double())
    v[:, 1] = w.bfloat16()[..., None]
    v[:, 2] = (w - w.bfloat16().double()).bfloat16()[..., None]
    q = torch.zeros(B, Hkv * group, D, device=cuda, dtype=torch.bfloat16)
    q[..., 0] = 1.0
    table = torch.arange(B, device=cuda, dtype=torch.int32)[:, None]
    o = ops.paged_attention(q, k, v, table, torch.full((B,), n, device=cuda), scale=1.0)
    want = (v[:, 1:3, :, 0].double().sum(1) - w) / (2 + w)
    assert float(want.abs().max()) < 2.0 ** -16
    sizes = 2 * w / (2 + w)
    tol = sizes * (2.0 ** -22 + 3 * U + 2 * n * 2.0 ** -23) + want.abs() * 2.0 ** -8
    off = (o.double().view(B, Hkv, group, D) - want[:, :, None, None]).abs()
    assert (off <= tol[:, :, None, None]).all()


@pytest.mark.parametrize("L", [4097, 9000, 33000, 40000])
def test_eviction_of_all_but_the_recent_slots_by_clusters(cuda, L):
    # nothing to choose: the blocks of a cluster meet for the counts alone
    from mk_iii_technologies_tsrn_b200 import ops
    import test_gpu_cache_evict as evict
    for B, Hkv, keep in ((1, 1, 1), (3, 2, 777), (9, 8, 4096)):
        k, v, table, mass, n = evict._case(cuda, B, Hkv, 8, L, 64, torch.bfloat16, "slots")
        kept, k2, v2, out = evict._want(k, v, table, mass, n, keep, keep)
        got = ops.cache_evict(k, v, table, n, mass, keep, keep)
        assert torch.equal(got, kept) and torch.equal(k, k2) and torch.equal(v, v2) and torch.equal(mass, out)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sampling_around_the_sizes_of_clusters(cuda, dtype):
    # rows of one block and of two, small blocks and large ones, few rows and many
    import test_gpu_sampling as sampling
    for V in (2048, 2049, 4096, 4097, 8192, 8193, 16385):
        for B in (1, 40, 160):
            for c in (dict(T=0.8), dict(k=20, p=0.9)):
                sampling._check(*sampling._logits(cuda, B, V, dtype, seed=V), **c)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("case", [(1, 64), (2, 64), (4, 128), (3, 33), (8, 80), (12, 256)], ids=str)
def test_infinite_values(cuda, case, gated, dtype):
    """An infinity in a value in use makes its channel that infinity, two of both signs or a NaN make it
    NaN, and the other channels are what they are; wherever the slot lies, the last one too.  Finite
    channels within the tolerance of test_gpu_paged_attention.py."""
    from mk_iii_technologies_tsrn_b200 import ops
    import test_gpu_paged_attention as base
    group, D = case
    inf, nan = float("inf"), float("nan")
    lengths = torch.tensor([1, 2, 7, 8, 16, 17, 250, 601, 5003], device=cuda, dtype=torch.int32)
    for store in (False, True):
        for B in (len(lengths), 1):                          # (one sequence: its segments are joined by teams)
            n = lengths[-B:].contiguous()
            k, v, table, g = base._cache(cuda, B, 5003, 2, D, 16, dtype)
            q = (0.2 * torch.randn(B, 2 * group, D, device=cuda, generator=g)).to(dtype)
            key, value = (torch.randn(B, 2, D, device=cuda, generator=g).to(dtype) for _ in range(2))
            gate = torch.rand(B, 2 * group, device=cuda, generator=g) if gated else None
            for b, m in enumerate(n.tolist()):
                for slot, channel, x in ((m - 1, 0, inf), (0, 1, -inf), (m // 2, 2, inf), (0, 3, inf), (m - 1, 3, -inf),
                                         (m // 3, 4, nan), (m - 1, D - 1, -inf), (m * 2 // 3, 9, inf)):
                    if x == -inf and channel == 3 and m == 1:
                        continue
                    v[table[b, slot // 16].long(), slot % 16, 1, channel] = x
                    if slot == m - 1:
                        value[b, 1, channel] = x
                last = m - 1
                at = table[b, last // 16].long()
                if not store:
                    key[b], value[b] = k[at, last % 16], v[at, last % 16]
            kw, vw = k.clone(), v.clone()
            for b, m in enumerate(n.tolist()):
                at = table[b, (m - 1) // 16].long()
                kw[at, (m - 1) % 16], vw[at, (m - 1) % 16] = key[b], value[b]
            new = dict(key=key, value=value) if store else {}
            o = ops.paged_attention(q, k, v, table, n, gate=gate, **new)
            want, _, off = base._reference(q, kw, vw, table, n, D ** -0.5, gate)
            o = o.double()
            assert torch.equal(o.isnan(), want.isnan()) and torch.equal(o.isinf(), want.isinf())
            assert torch.equal(o[o.isinf()], want[want.isinf()])
            fine = want.isfinite()
            top = v[v.isfinite()].double().abs().max()
            tol = 2 * off[..., None] * top + (want.abs() * 2.0 ** -8 + top * 2.0 ** -16 if dtype == torch.bfloat16 else 0)
            assert bool(((o - want).abs() <= tol)[fine].all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_eviction_without_channels(cuda, dtype):
    # no rows to move; the choice of slots and their weights are due
    from mk_iii_technologies_tsrn_b200 import ops
    import test_gpu_cache_evict as evict
    for L, keep in ((40, 16), (5000, 700), (9, 20)):
        _, _, table, mass, n = evict._case(cuda, 2, 3, 8, L, 16, dtype, "slots")
        k = torch.empty(table.numel() + 1, 16, 3, 0, device=cuda, dtype=dtype)
        kept, _, _, out = evict._want(k, k, table, mass, n, keep, 4)
        got = ops.cache_evict(k, k.clone(), table, n, mass, keep, 4)
        assert torch.equal(got, kept) and torch.equal(mass, out)
    key = torch.empty(2, 5, 3, 0, device=cuda, dtype=dtype)
    ops.paged_append(key, key, k, k.clone(), table, torch.zeros_like(n))


def test_generate_under_a_budget_beyond_all_tokens(cuda):
    import test_gpu_decode_run as decode
    m = decode._model(cuda)
    ids = torch.randint(0, 97, (2, 9), device=cuda, generator=torch.Generator(device=cuda).manual_seed(2))
    u = torch.rand(20, 2, device=cuda, generator=torch.Generator(device=cuda).manual_seed(3))
    assert torch.equal(m.generate(ids, 20, uniform=u), m.generate(ids, 20, uniform=u, keep=2 ** 40))


def test_counts_beyond_32_bits_keep_all_tokens(cuda):
    from mk_iii_technologies_tsrn_b200 import ops
    x = torch.randn(4, 900, device=cuda, generator=torch.Generator(device=cuda).manual_seed(0))
    u = torch.tensor([0.1, 0.5, 0.9, 0.99], device=cuda)
    k = torch.tensor([2 ** 32 + 1, 2 ** 32 + 5, 2 ** 31, -2 ** 32 + 1], device=cuda)
    assert torch.equal(ops.sample_tokens(x, u, top_k=k), ops.sample_tokens(x, u))
    assert torch.equal(ops.sample_tokens(x, u, top_k=2 ** 40), ops.sample_tokens(x, u))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_caches_whose_rows_overlap_are_refused(cuda, dtype):
    from mk_iii_technologies_tsrn_b200 import ops
    from test_decode_host_edges import _layouts
    n = torch.tensor([1], device=cuda, dtype=torch.int32)
    for k, apart in _layouts(dtype, cuda):
        v, heads, slots = k.clone(), k.shape[2], k.shape[1]
        table = torch.arange(max(1, k.shape[0]), device=cuda, dtype=torch.int32)[None]
        key = torch.randn(1, slots * k.shape[0], heads, 8, device=cuda).to(dtype)
        mass = torch.rand(1, heads, table.shape[1] * slots, device=cuda)
        calls = (lambda: ops.paged_append(key, key, k, v, table, n - 1),
                 lambda: ops.paged_append(key, key, v, k, table, n - 1),
                 lambda: ops.paged_attention(key[:, 0] if key.shape[1] else mass[..., :8].to(dtype), k, v, table, n * 0),
                 lambda: ops.cache_evict(k, v, table, n, mass, 1))
        if not apart:
            for call in calls:
                with pytest.raises(ValueError, match="apart"):
                    call()
            continue
        for call in calls[:2] + calls[3:]:
            call()
        if k.numel():
            assert torch.equal(k.flatten(0, 1), key[0]) and torch.equal(v.flatten(0, 1), key[0])
    k, v = torch.zeros(2, 20, 16, 2, 8, device=cuda, dtype=dtype)
    table = torch.arange(6, device=cuda, dtype=torch.int32).view(3, 2)
    flat = torch.rand(400, device=cuda)
    lengths = torch.tensor([10, 7, 0], device=cuda, dtype=torch.int32)
    for strides, apart in (((32, 96, 1), True), ((15, 10, 1), False), ((64, 32, 1), True), ((32, 32, 1), False)):
        mass = flat.as_strided((3, 2, 32), strides)
        if apart:
            ops.cache_evict(k, v, table, lengths, mass, 4)
        else:
            with pytest.raises(ValueError, match="separate"):
                ops.cache_evict(k, v, table, lengths, mass, 4)
            with pytest.raises(ValueError, match="separate"):
                ops.paged_attention(k[:3, 0], k, v, table, lengths, mass=mass)


def test_generate_runs_the_models_stack(cuda):
    # hooks on the stack of layers, and a forward of its own, count in generate as in forward
    import test_gpu_decode_run as decode
    from mk_iii_technologies_tsrn_b200 import dropin
    m = decode._model(cuda)
    ids = torch.randint(0, 97, (3, 9), device=cuda, generator=torch.Generator(device=cuda).manual_seed(2))
    plain = m.generate(ids, 4, temperature=0.0)
    calls = []
    hook = m.layers.register_forward_hook(lambda mod, a, out: calls.append(out.shape) or -out)
    got = m.generate(ids, 4, temperature=0.0)
    assert calls == [(3, 9, 64)] + [(3, 1, 64)] * 3 and not torch.equal(got, plain)
    with torch.no_grad():
        assert torch.equal(got[:, 0], m(ids)[:, -1].argmax(-1))
    hook.remove()

    class Turned(dropin.TropicalEncoder):
        def forward(self, *args, **kw):
            return -super().forward(*args, **kw)

    m.layers.__class__ = Turned
    assert torch.equal(m.generate(ids, 4, temperature=0.0), got)


def test_generate_under_autocast(cuda, monkeypatch):
    # as forward runs there; every token's attention within the tolerance of test_gpu_paged_attention.py
    import test_gpu_decode_run as decode
    import test_gpu_paged_attention as base
    import test_gpu_paged_attention_finite as finite
    from mk_iii_technologies_tsrn_b200 import dropin
    m = decode._model(cuda)
    g = torch.Generator(device=cuda).manual_seed(2)
    ids = torch.randint(0, 97, (3, 9), device=cuda, generator=g)
    mask = (torch.arange(9, device=cuda) < torch.tensor([[9], [1], [5]], device=cuda)).long()
    u = torch.rand(12, 3, device=cuda, generator=g)
    own, steps = dropin._PagedLayer.attend, []

    def attend(self, Q, K, V, scale, gate, tau):
        c, i = self.cache, self.index
        assert Q.dtype == c.k[i].dtype == torch.bfloat16
        o = own(self, Q, K, V, scale, gate, tau)
        want, _, off = base._reference(Q[:, :, 0], c.k[i], c.v[i], c.block_table, c.lengths, scale, gate.float(), tau)
        finite._check(o, want, off, c.v[i], torch.bfloat16)
        last = c.lengths.long() - 1
        at = c.block_table[torch.arange(3), last // 16].long()
        assert torch.equal(c.k[i][at, last % 16], K[:, :, 0]) and torch.equal(c.v[i][at, last % 16], V[:, :, 0])
        steps.append(i)
        return o

    with torch.autocast("cuda", dtype=torch.bfloat16):
        plain = m.generate(ids, 12, attention_mask=mask, uniform=u, top_k=20)
        short = m.generate(ids, 12, attention_mask=mask, uniform=u, keep=4, recent=1, page_size=2)
        best = m.generate(ids, 1, attention_mask=mask, temperature=0.0)[:, 0]
        with torch.no_grad():
            logits = m(ids, mask)[torch.arange(3), mask.sum(1) - 1]
        monkeypatch.setattr(dropin._PagedLayer, "attend", attend)
        assert torch.equal(m.generate(ids, 12, attention_mask=mask, uniform=u, top_k=20), plain)
    assert steps == [0, 1] * 11 and logits.dtype == torch.bfloat16
    assert torch.equal(logits.gather(1, best[:, None])[:, 0], logits.amax(1))
    for t in (plain, short):
        assert t.shape == (3, 12) and int(t.min()) >= 0 and int(t.max()) < 97


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_bad_page_shows_in_the_weights_of_its_sequence_alone(cuda, dtype):
    from mk_iii_technologies_tsrn_b200 import ops
    import test_gpu_paged_attention as base
    k, v, table, g = base._cache(cuda, 3, 200, 2, 64, 16, dtype)
    n = torch.tensor([150, 200, 203], device=cuda, dtype=torch.int32)
    q = torch.randn(3, 4, 64, device=cuda, generator=g).to(dtype)
    table[1, 4] = k.shape[0]
    n[2] = 210                                                # beyond the table: its weights stay
    mass = torch.rand(3, 2, 208, device=cuda, generator=g)
    before = mass.clone()
    ops.paged_attention(q, k, v, table, n, mass=mass)
    with pytest.raises(ops.DeviceIndexError):
        ops.check_device_error(cuda)
    assert bool(mass[1, :, :200].isnan().all()) and torch.equal(mass[1, :, 200:], before[1, :, 200:])
    assert torch.equal(mass[2], before[2]) and not bool(mass[0].isnan().any())
