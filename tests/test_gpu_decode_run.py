"""The decoding operators together, as a token model uses them: prompt, tokens one at a time,
eviction, sampling; on other streams, captured, and from two threads."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(dev, vocab=97, **kw):
    from mk_iii_technologies_tsrn_b200 import dropin
    torch.manual_seed(0)
    m = dropin.TropicalDecoderModel(vocab, d_model=64, nhead=4, num_layers=2, dim_feedforward=96, dropout=0.1,
                                    max_seq_len=80, **kw)
    with torch.no_grad():
        for p in m.parameters():
            p.add_(0.05 * torch.randn_like(p))
    return m.to(dev).eval()


def _again(m, ids, counts, new, uniform, **choices):
    """The same tokens by running the whole model on all of them every time."""
    from mk_iii_technologies_tsrn_b200 import ops
    rows = [ids[b, :n].tolist() for b, n in enumerate(counts)]
    out, gaps = [], []
    with torch.no_grad():
        for t in range(new):
            width = max(map(len, rows))
            batch = torch.zeros(len(rows), width, dtype=torch.int64, device=ids.device)
            mask = torch.zeros_like(batch)
            for b, r in enumerate(rows):
                batch[b, :len(r)] = torch.tensor(r, device=ids.device)
                mask[b, :len(r)] = 1
            logits = m(batch, mask)[torch.arange(len(rows)), [len(r) - 1 for r in rows]]
            top = logits.topk(2).values
            gaps.append(top[:, 0] - top[:, 1])
            tok = ops.sample_tokens(logits, uniform[t], **choices)
            out.append(tok)
            for r, k in zip(rows, tok.tolist()):
                r.append(k)
    return torch.stack(out, 1), torch.stack(gaps, 1)


@pytest.mark.parametrize("padded", [False, True])
def test_generate_equals_running_the_whole_model(cuda, padded):
    m = _model(cuda)
    g = torch.Generator(device=cuda).manual_seed(1)
    ids = torch.randint(0, 97, (3, 21), device=cuda, generator=g)
    counts = [21, 1, 13] if padded else [21] * 3
    mask = (torch.arange(21, device=cuda) < torch.tensor(counts, device=cuda)[:, None]).long() if padded else None
    u = torch.rand(30, 3, device=cuda, generator=g)
    # the best token: rounding (a few 1e-6 of the logits) can only turn a smaller gap than that
    got = m.generate(ids, 30, attention_mask=mask, temperature=0.0)
    want, gaps = _again(m, ids, counts, 30, u, temperature=0.0)
    for b in range(3):
        clear = int((gaps[b] > 1e-4).long().cumprod(0).sum())
        assert clear > 0 and torch.equal(got[b, :clear], want[b, :clear])
    # sampled from the same numbers: a row goes on as long as it agrees, and rounding moves a border
    # of the running sum (96 of them) by some 1e-5: hardly one token in a thousand
    got = m.generate(ids, 30, attention_mask=mask, uniform=u, top_k=40, top_p=0.9)
    want, _ = _again(m, ids, counts, 30, u, top_k=40, top_p=0.9)
    assert int((got == want).all(1).sum()) >= 2
    assert torch.equal(got, m.generate(ids, 30, attention_mask=mask, uniform=u, top_k=40, top_p=0.9))


def test_budget_that_is_never_reached_changes_nothing(cuda):
    m = _model(cuda)
    ids = torch.randint(0, 97, (2, 9), device=cuda, generator=torch.Generator(device=cuda).manual_seed(2))
    u = torch.rand(20, 2, device=cuda, generator=torch.Generator(device=cuda).manual_seed(3))
    assert torch.equal(m.generate(ids, 20, uniform=u), m.generate(ids, 20, uniform=u, keep=40))


def test_budget_holds(cuda):
    m = _model(cuda)
    ids = torch.randint(0, 97, (2, 40), device=cuda, generator=torch.Generator(device=cuda).manual_seed(2))
    u = torch.rand(40, 2, device=cuda, generator=torch.Generator(device=cuda).manual_seed(3))
    for kw in (dict(keep=16), dict(keep=5, recent=5), dict(keep=1, recent=0, page_size=3)):
        t = m.generate(ids, 40, uniform=u, **kw)
        assert t.shape == (2, 40) and int(t.min()) >= 0 and int(t.max()) < 97


def test_prompt_tokens_and_eviction_step_by_step(cuda):
    # one layer of the module against its plain expressions in 64 bits over the slots that stayed
    from mk_iii_technologies_tsrn_b200 import dropin
    torch.manual_seed(4)
    B, D, H, T = 2, 48, 4, 30
    att = dropin.TropicalMultiHeadAttention(D, H, dropout=0.0, init_temp=0.7).to(cuda)
    with torch.no_grad():
        att.score_gate.weight.normal_()
    x = torch.randn(B, T + 12, D, device=cuda)
    counts = torch.tensor([T, 17], device=cuda, dtype=torch.int32)
    cache = dropin.TropicalPagedKVCache(1, B, H, D // H, T + 16, page_size=4, collect_mass=True, device=cuda)
    att64 = dropin.TropicalMultiHeadAttention(D, H, dropout=0.0).to(cuda).double()
    att64.load_state_dict({k: v.double() for k, v in att.state_dict().items()})

    def plain(b, xq, slots):
        """The module's expressions for one query; slots: [H] lists of cached inputs."""
        q = att64.q_proj(xq).view(H, -1)
        gate, tau = torch.sigmoid(att64.score_gate(xq)), att64.maslov.temperatures
        o, ws = [], []
        for h in range(H):
            xs = torch.stack(slots[h])
            k = att64.k_proj(xs).view(len(xs), H, -1)[:, h]
            v = att64.v_proj(xs).view(len(xs), H, -1)[:, h]
            s = (gate[h] * (q[h] + k).amax(-1) + (1 - gate[h]) * (k @ q[h])) * (D // H) ** -0.5
            w = torch.softmax(s / tau[h], 0)
            o.append(w @ v)
            ws.append(w)
        return att64.out_proj(torch.cat(o)), ws

    with torch.no_grad():
        cache.begin(counts, T)
        pad = torch.arange(T, device=cuda) >= counts[:, None]
        att(x[:, :T], x[:, :T], x[:, :T], dropin.make_causal_mask(T, cuda), pad, cache=cache.layer(0))
        kept = [[[x[b, j].double() for j in range(int(counts[b]))] for _ in range(H)] for b in range(B)]
        mass = [[torch.zeros(len(kept[b][h]), device=cuda, dtype=torch.float64) for h in range(H)] for b in range(B)]
        for b in range(B):
            for i in range(int(counts[b])):
                _, ws = plain(b, kept[b][0][i], [s[:i + 1] for s in kept[b]])
                for h in range(H):
                    mass[b][h][:i + 1] += ws[h]
        for t in range(12):
            if t in (3, 8):
                cache.evict(12, 4)
                for b in range(B):
                    for h in range(H):
                        n = len(kept[b][h])
                        if n <= 12:
                            continue
                        order = torch.sort(mass[b][h][:n - 4], descending=True)
                        assert float(order.values[7] - order.values[8]) > 1e-4      # (no near ties in this case)
                        take = sorted(order.indices[:8].tolist()) + list(range(n - 4, n))
                        kept[b][h] = [kept[b][h][j] for j in take]
                        mass[b][h] = mass[b][h][take]
            cache.step()
            xt = x[:, T + t:T + t + 1]
            got, _ = att(xt, xt, xt, cache=cache.layer(0))
            for b in range(B):
                for h in range(H):
                    kept[b][h].append(xt[b, 0].double())
                    mass[b][h] = torch.cat((mass[b][h], mass[b][h].new_zeros(1)))
                want, ws = plain(b, xt[b, 0].double(), kept[b])
                for h in range(H):
                    mass[b][h] += ws[h]
                    n = len(kept[b][h])
                    assert (cache.mass[0][b, h, :n].double() - mass[b][h]).abs().max() < 1e-4
                assert (got[b, 0].double() - want).abs().max() < 1e-4
            assert cache.lengths.tolist() == [len(kept[b][0]) for b in range(B)]


def test_refusals_of_the_modules(cuda):
    from mk_iii_technologies_tsrn_b200 import dropin
    m = _model(cuda)
    ids = torch.zeros(2, 10, dtype=torch.int64, device=cuda)
    for kw, match in ((dict(max_new_tokens=0), "positions"), (dict(max_new_tokens=72), "positions"),
                      (dict(max_new_tokens=5, keep=0), "keep"), (dict(max_new_tokens=5, keep=4, recent=5), "recent"),
                      (dict(max_new_tokens=5, uniform=torch.rand(5, 3, device=cuda)), "uniform"),
                      (dict(max_new_tokens=5, attention_mask=torch.tensor([[0] + [1] * 9] * 2, device=cuda)), "right")):
        with pytest.raises(ValueError, match=match):
            m.generate(ids, **kw)
    m.train()
    with pytest.raises(RuntimeError, match="dropout"):
        m.generate(ids, 3)
    cache = dropin.TropicalPagedKVCache(1, 1, 2, 8, 4, device=cuda)
    with pytest.raises(ValueError, match="fit"):
        cache.begin(torch.tensor([5]), 5)
    with pytest.raises(ValueError, match="collect_mass"):
        cache.evict(2)
    att = dropin.TropicalMultiHeadAttention(16, 2, dropout=0.0).to(cuda)
    x = torch.randn(1, 2, 16, device=cuda)
    cache.begin(torch.tensor([2]), 2)
    with pytest.raises(RuntimeError, match="not differentiable"):
        att(x, x, x, cache=cache.layer(0))
    with torch.no_grad():
        att(x, x, x, cache=cache.layer(0))
        cache.step()
        with pytest.raises(ValueError, match="one token"):
            att(x, x, x, cache=cache.layer(0))


# ----------------------------------------------------------------------------- the operators' calls
def _inputs(dev, B=3, H=8, Hkv=2, D=64, L=700, dtype=torch.bfloat16, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    per = -(-L // 16)
    k, v = (torch.randn(B * per, 16, Hkv, D, device=dev, generator=g).to(dtype) for _ in range(2))
    table = torch.randperm(B * per, device=dev, generator=g).view(B, per).int()
    n = torch.randint(L // 2, L, (B,), device=dev, generator=g, dtype=torch.int32)
    q = torch.randn(B, H, D, device=dev, generator=g).to(dtype)
    mass = torch.rand(B, Hkv, per * 16, device=dev, generator=g)
    x, u = 3 * torch.randn(B, 5000, device=dev, generator=g), torch.rand(B, device=dev, generator=g)
    return dict(k=k, v=v, table=table, n=n, q=q, mass=mass, x=x, u=u, key=q[:, :Hkv].clone())


def _run(s, keep=300):
    from mk_iii_technologies_tsrn_b200 import ops
    o = ops.paged_attention(s["q"], s["k"], s["v"], s["table"], s["n"], key=s["key"], value=s["key"], mass=s["mass"])
    kept = ops.cache_evict(s["k"], s["v"], s["table"], s["n"], s["mass"], keep, 20)
    o2 = ops.paged_attention(s["q"], s["k"], s["v"], s["table"], s["n"].clamp(max=keep))
    ops.paged_append(o2[:, None, :s["key"].shape[1]], s["key"][:, None], s["k"], s["v"], s["table"], s["n"].clamp(max=keep) - 1)
    t, lp = ops.sample_tokens(s["x"], s["u"], top_k=40, top_p=0.9, return_logprob=True)
    return [o, kept, o2, t, lp, s["k"], s["v"], s["mass"]]


def _copy(s):
    return {k: v.clone() for k, v in s.items()}


def test_run_repeats_bit_for_bit_on_another_stream_and_captured(cuda):
    s0 = _inputs(cuda)
    want = [t.clone() for t in _run(_copy(s0))]
    other = torch.cuda.Stream(cuda)
    s = _copy(s0)
    other.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(other):
        got = _run(s)
    other.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # captured; replayed on other inputs of the same sizes; two graphs in turn
    graphs = []
    for seed in (0, 1):
        s = _copy(_inputs(cuda, seed=seed))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _run(s)
        graphs.append((graph, s, out))
    for seed in (0, 1, 2):
        for graph, s, out in graphs:
            new = _inputs(cuda, seed=seed)
            for k in s:
                s[k].copy_(new[k])
        for graph, s, out in graphs:
            graph.replay()
        fresh = _run(_inputs(cuda, seed=seed))
        for graph, s, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, fresh))


def test_two_threads_on_two_streams(cuda):
    want = [[t.clone() for t in _run(_inputs(cuda, seed=i, dtype=d))] for i, d in ((0, torch.bfloat16), (1, torch.float32))]
    torch.cuda.synchronize(cuda)
    bad = []

    def work(i, dtype):
        stream = torch.cuda.Stream(cuda)
        with torch.cuda.stream(stream):
            for _ in range(20):
                got = _run(_inputs(cuda, seed=i, dtype=dtype))
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    bad.append(i)
        stream.synchronize()

    threads = [threading.Thread(target=work, args=a) for a in ((0, torch.bfloat16), (1, torch.float32))]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


def test_refusals(cuda):
    from mk_iii_technologies_tsrn_b200 import ops
    s = _inputs(cuda)

    def att(**kw):
        args = [kw.pop(k, s[k]) for k in ("q", "k", "v", "table", "n")]
        return ops.paged_attention(*args, **kw)

    for kw in (dict(q=s["q"][:, :7]), dict(q=s["q"][..., :60]), dict(v=s["v"][:-1]), dict(table=s["table"].t()),
               dict(table=s["table"][:2]), dict(n=s["n"][:2]), dict(key=s["key"]), dict(key=s["key"][:2], value=s["key"]),
               dict(gate=torch.rand(3, 2, device=cuda)), dict(tau=torch.rand(3, device=cuda)),
               dict(mass=s["mass"].transpose(1, 2)), dict(mass=s["mass"][:, :1]),
               dict(mass=s["mass"][:1].expand(3, -1, -1)), dict(k=s["k"][:, :, :1].expand(-1, -1, 2, -1)),
               dict(k=s["k"][..., ::2], v=s["v"][..., ::2], q=s["q"][..., ::2]), dict(n=s["n"].float()),
               dict(q=s["q"].repeat(1, 1, 5), k=s["k"].repeat(1, 1, 1, 5), v=s["v"].repeat(1, 1, 1, 5))):
        with pytest.raises(ValueError):
            att(**kw)
    for kw in (dict(q=s["q"].half()), dict(mass=s["mass"].double()), dict(gate=torch.rand(3, 8, device=cuda).bfloat16()),
               dict(k=s["k"].half(), v=s["v"].half())):
        with pytest.raises((TypeError, ValueError)):
            att(**kw)
    with pytest.raises(RuntimeError, match="not differentiable"):
        att(q=s["q"].clone().requires_grad_())
    with pytest.raises(RuntimeError, match="devices|CPU"):
        att(n=s["n"].cpu())
    with pytest.raises(NotImplementedError):
        torch.func.vmap(lambda q: ops.paged_attention(q, s["k"], s["v"], s["table"], s["n"]))(s["q"][None])
    ev = lambda keep=5, recent=1, **kw: ops.cache_evict(s["k"], s["v"], s["table"], kw.pop("n", s["n"]),
                                                        kw.pop("mass", s["mass"]), keep, recent, **kw)
    for kw in (dict(keep=0), dict(recent=6), dict(recent=-1), dict(out=s["mass"][..., :4]), dict(mass=s["mass"][..., ::2]),
               dict(n=s["n"][:1])):
        with pytest.raises(ValueError):
            ev(**kw)
    key = s["q"][:, None, :2]
    for a in ((key, key[:, :, :1]), (key[:2], key[:2]), (key[..., :8], key[..., :8]), (key[0], key[0])):
        with pytest.raises(ValueError):
            ops.paged_append(*a, s["k"], s["v"], s["table"], s["n"])
    sm = lambda x=s["x"], u=s["u"], **kw: ops.sample_tokens(x, u, **kw)
    for kw in (dict(x=s["x"][0]), dict(u=s["u"][:2]), dict(top_k=torch.ones(2, device=cuda)), dict(x=s["x"][:, :0]),
               dict(temperature=torch.ones(3, 1, device=cuda)), dict(top_p=2.0), dict(u=s["u"].half())):
        with pytest.raises(ValueError):
            sm(**kw)
    with pytest.raises(TypeError):
        sm(x=s["x"].half())
    with pytest.raises(RuntimeError, match="not differentiable"):
        sm(x=s["x"].clone().requires_grad_())


def test_empty_batches(cuda):
    from mk_iii_technologies_tsrn_b200 import ops
    s = _inputs(cuda)
    none = {k: s[k][:0] for k in ("q", "table", "n", "mass", "x", "u", "key")}
    assert ops.paged_attention(none["q"], s["k"], s["v"], none["table"], none["n"], mass=none["mass"]).shape == (0, 8, 64)
    assert ops.cache_evict(s["k"], s["v"], none["table"], none["n"], none["mass"], 4).shape == (0, 2, 4)
    assert ops.sample_tokens(none["x"], none["u"]).shape == (0,)
    ops.paged_append(none["key"][:, None], none["key"][:, None], s["k"], s["v"], none["table"], none["n"])
    ops.paged_append(s["key"][:, None][:, :0], s["key"][:, None][:, :0], s["k"], s["v"], s["table"], s["n"])
    empty = s["k"][:0]
    zero = torch.zeros(3, device=cuda, dtype=torch.int32)
    assert bool((ops.paged_attention(s["q"], empty, empty, s["table"], zero) == 0).all())
    assert bool((ops.paged_attention(s["q"], s["k"], s["v"], s["table"][:, :0], zero) == 0).all())
