"""The embedding, the gated recurrence and the residual step together, as a small language model
uses them: embedding -> blocks (attention, reservoir, gated SSM with fused residual steps) -> tied
logits, trained and decoded, against the same model on the PyTorch expressions.

Both run the same attention and reservoir kernels; the rest differs in the order and number of fp32
roundings only.  Tolerances are those of the block's own fixture test (outputs 1e-4 relative, 5e-5
absolute) and of the drop-ins' gradient test (1e-3 of the largest value); top_k covers every key,
so that no rounding decides a selection."""
import numpy as np
import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu

V, D, T, B = 61, 64, 40, 3


class TinyLM(nn.Module):
    def __init__(self, fused: bool, ssm: str = "gated"):
        super().__init__()
        from mk_iii_technologies_tsrn_b200.tsrn_block import TSRNTropicalPath
        self.fused = fused
        self.embed = nn.Embedding(V, D, padding_idx=0)
        self.pos = nn.Embedding(T, D)
        self.blocks = nn.ModuleList(TSRNTropicalPath(D, top_k=T, n_heads=4, ssm=ssm,
                                                     fused_residual=fused) for _ in range(2))

    def forward(self, ids):
        from mk_iii_technologies_tsrn_b200 import ops
        # the reservoirs' power iteration starts from a drawn vector and moves it on with every
        # call: one start for both models and all calls
        for blk in self.blocks:
            v = blk.reservoir._cached_v
            v.copy_(torch.linspace(-1.0, 1.3, v.numel(), device=v.device))
        if self.fused:
            x = ops.embedding(ids, self.embed.weight, D ** 0.5, pos_weight=self.pos.weight,
                              padding_idx=0)
        else:
            at = torch.arange(ids.shape[1], device=ids.device)
            x = self.embed(ids) * D ** 0.5 + self.pos(at)
        for blk in self.blocks:
            x = blk(x)
        return x @ self.embed.weight.t()


def _pair(cuda, ssm):
    torch.manual_seed(0)
    a = TinyLM(True, ssm)
    with torch.no_grad():
        for p in a.parameters():                # zero-initialised projections would hide errors
            p.add_(0.05 * torch.randn_like(p))
    b = TinyLM(False, ssm)
    b.load_state_dict(a.state_dict())
    return a.to(cuda), b.to(cuda)


def _ids(cuda):
    g = torch.Generator(device=cuda).manual_seed(1)
    ids = torch.randint(1, V, (B, T), device=cuda, generator=g)
    ids[1, 30:] = 0                             # padding
    return ids


@pytest.mark.parametrize("ssm", ["gated", "tropical"])
def test_training_step_matches_the_unfused_model(cuda, ssm):
    a, b = _pair(cuda, ssm)
    ids = _ids(cuda)
    out = []
    for m in (a, b):
        logits = m(ids)
        loss = nn.functional.cross_entropy(logits[:, :-1].reshape(-1, V), ids[:, 1:].reshape(-1),
                                           ignore_index=0)
        loss.backward()
        out.append(logits.detach())
    torch.testing.assert_close(out[0], out[1], rtol=1e-4, atol=5e-5 * float(out[1].abs().max()))
    for (name, p), q in zip(a.named_parameters(), b.parameters()):
        assert (p.grad is None) == (q.grad is None), name
        if p.grad is not None:
            np.testing.assert_allclose(p.grad.cpu().numpy(), q.grad.cpu().numpy(), rtol=1e-3,
                                       atol=1e-3 * float(q.grad.abs().max()), err_msg=name)


def test_inference_matches_and_repeats(cuda):
    a, b = _pair(cuda, "gated")
    ids = _ids(cuda)
    with torch.no_grad():
        y = a(ids)
        torch.testing.assert_close(y, b(ids), rtol=1e-4, atol=5e-5 * float(y.abs().max()))
        assert torch.equal(y, a(ids))


def test_branch_events_of_the_fused_path(cuda):
    a, _ = _pair(cuda, "tropical")
    ev = {n: (torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True))
          for n in ("attn", "reservoir", "tropical_ssm")}
    with torch.no_grad():
        a.blocks[0](torch.randn(B, T, D, device=cuda), events=ev)
    torch.cuda.synchronize()
    assert all(s.elapsed_time(e) > 0 for s, e in ev.values())


def test_ssm_prefill_then_steps_equal_the_whole(cuda):
    # a padded prefill, then one token at a time: the same recurrence on the same fp32 states; the
    # projections' rows go through products of another size: 1e-5 of the values
    from mk_iii_technologies_tsrn_b200.ssm import GatedSSM
    torch.manual_seed(2)
    m = GatedSSM(D, 96)
    with torch.no_grad():
        for p in m.parameters():
            p.add_(0.1 * torch.randn_like(p))
    m = m.to(cuda)
    x = torch.randn(B, 30, D, device=cuda)
    n = torch.tensor([20, 1, 13], device=cuda)
    with torch.no_grad():
        whole = m(x)
        padded = x.clone()
        for i, k in enumerate(n.tolist()):
            padded[i, k:] = float("nan")        # nothing behind a row's end may matter
        _, state = m(padded, lengths=n, return_state=True)
        for t in range(8):
            at = n + t
            y = m.step(x[torch.arange(B, device=cuda), at], state)
            torch.testing.assert_close(y, whole[torch.arange(B, device=cuda), at], rtol=1e-5,
                                       atol=1e-5)
        h0 = m.init_state(B)
        assert h0.shape == (B, 96) and torch.all(h0 == 0)


def test_decoder_model_embeds_with_the_kernel(cuda):
    # the drop-in's embedding: bits of the PyTorch expression, gradients within the bound of a sum
    # of n rows in fp32; a table with a hook takes the PyTorch path
    from mk_iii_technologies_tsrn_b200 import dropin
    m = dropin.TropicalDecoderModel(V, d_model=32, nhead=4, num_layers=1, dim_feedforward=64,
                                    dropout=0.0, max_seq_len=T).to(cuda)
    ids = _ids(cuda)
    x = m._embed(ids)
    want = m.embed(ids) * m.embed_scale + m.pos_embed(torch.arange(T, device=cuda))[None]
    assert torch.equal(x, want) and "::Embedding" in x.grad_fn.name()
    d = torch.randn_like(x)
    for p, q in zip(torch.autograd.grad(x, (m.embed.weight, m.pos_embed.weight), d),
                    torch.autograd.grad(want, (m.embed.weight, m.pos_embed.weight), d)):
        n = B * T
        size = float(d.abs().sum((0, 1)).max()) * m.embed_scale
        assert float((p - q).abs().max()) <= 2 * (n + 2) * 2.0 ** -24 * size
    h = m.embed.register_forward_hook(lambda mod, i, o: o * 2)
    assert torch.equal(m._embed(ids), m.embed(ids) * m.embed_scale + m.pos_embed(
        torch.arange(T, device=cuda))[None])
    h.remove()
    assert m(ids).shape == (B, T, V)


def test_second_derivatives_are_refused(cuda):
    # the gradients are there with create_graph=True; differentiating them again raises
    from mk_iii_technologies_tsrn_b200 import ops
    w = torch.randn(7, 8, device=cuda, requires_grad=True)
    x = torch.randn(2, 3, 8, device=cuda, requires_grad=True)
    ids = torch.randint(0, 7, (2, 3), device=cuda)
    for leaf, out in ((w, ops.embedding(ids, w)), (x, ops.gated_scan(x, x, form="sigmoid")),
                      (x, ops.residual_norm(x, x)[1])):
        d = torch.randn_like(out, requires_grad=True)
        (once,) = torch.autograd.grad(out, leaf, d, create_graph=True, retain_graph=True)
        (plain,) = torch.autograd.grad(out, leaf, d.detach(), retain_graph=True)
        assert torch.equal(once, plain) and once.requires_grad
        with pytest.raises(RuntimeError, match="not differentiable"):
            once.sum().backward()
        (free,) = torch.autograd.grad(out, leaf, d.detach(), create_graph=True)
        assert torch.equal(free, plain) and not free.requires_grad


def test_a_refusal_of_the_library_is_its_error(cuda):
    from mk_iii_technologies_tsrn_b200 import _lib, ops
    x = torch.randn(4, 8, device=cuda)
    for t in (x, x.clone().requires_grad_()):
        with pytest.raises(_lib.TropicalLibraryError) as e:
            ops.residual_norm(t, t, eps=-1.0)
        assert e.value.status == -1


def test_captured_forward_and_backward(cuda):
    # whole calls with their autograd nodes in one graph, replayed on new values; an eager call of
    # the same tensors in between leaves the graph's results alone
    from mk_iii_technologies_tsrn_b200 import ops
    g = torch.Generator(device=cuda).manual_seed(11)
    B, T, V, D = 3, 70, 40, 33
    ids = torch.randint(0, V, (B, T), device=cuda, generator=g)
    w, z, s, p = (torch.randn(n, device=cuda, generator=g).requires_grad_()
                  for n in ((V, D), (B, T, D), (D,), (T, D)))
    d = torch.randn(B, T, D, device=cuda, generator=g)

    def step():
        e = ops.embedding(ids, w, 1.5, pos_weight=p)
        h = ops.gated_scan(z, e, form="sigmoid")
        y, n = ops.residual_norm(e, h, gate=z, scale=s)
        return torch.autograd.grad((y, n), (w, z, s, p), (d, d))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (1, 2):
        with torch.no_grad():
            for t in (w, z, s, d, p):
                t.copy_(torch.randn(t.shape, device=cuda, generator=g))
            ids.copy_(torch.randint(0, V, (B, T), device=cuda, generator=g))
        eager = step()
        graph.replay()
        for a, b in zip(out, eager):
            assert torch.equal(a, b)


def test_two_streams_at_once(cuda):
    from mk_iii_technologies_tsrn_b200 import ops
    g = torch.Generator(device=cuda).manual_seed(12)
    x = [torch.randn(2, 400, 96, device=cuda, generator=g).requires_grad_() for _ in range(2)]
    ids = [torch.randint(0, 50, (3000,), device=cuda, generator=g) for _ in range(2)]
    d = torch.randn(3000, 96, device=cuda, generator=g)

    def work(i):
        h = ops.gated_scan(x[i], x[i], form="sigmoid")
        y, n = ops.residual_norm(x[i], h, gate=x[i])
        return (*torch.autograd.grad((y, n), x[i], (y.detach(), n.detach())),
                ops.embedding_bwd(ids[i], d, 50))

    want = [work(0), work(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(work(i))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i]))


def test_bad_ids_stop_a_token_model(cuda):
    # the call that meets them returns NaN rows; once the device has run it, the next call raises
    from mk_iii_technologies_tsrn_b200 import dropin, ops
    m = dropin.TropicalDecoderModel(V, d_model=32, nhead=4, num_layers=1, dim_feedforward=64,
                                    dropout=0.0, max_seq_len=T).to(cuda)
    ids = _ids(cuda)
    bad = ids.clone()
    bad[1, 3] = V
    with torch.no_grad():
        want = m._embed(ids)
        assert m._embed(bad)[1, 3].isnan().all()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):                  # a capture is left alone
            m._embed(ids)
        with pytest.raises(ops.DeviceIndexError):
            m._embed(ids)
        assert torch.equal(m._embed(ids), want)


def _calls(cuda):
    """name -> (call, its differentiable arguments)"""
    from mk_iii_technologies_tsrn_b200 import ops
    g = torch.Generator(device=cuda).manual_seed(21)
    r = lambda *s: torch.randn(*s, device=cuda, generator=g)  # noqa: E731
    ids = torch.randint(0, 7, (2, 3), device=cuda, generator=g)
    return {
        "embedding": (lambda w, p: ops.embedding(ids, w, 2.0, pos_weight=p), (r(7, 8), r(4, 8))),
        "scan": (lambda z, x, h: ops.gated_scan(z, x, h, form="sigmoid"),
                 (r(2, 5, 8), r(2, 5, 8), r(2, 8))),
        "step": (lambda z, x, h: ops.gated_scan_step(z, x, h), (r(2, 8), r(2, 8), r(2, 8))),
        "residual": (lambda x, b, z, s, w, c, bw, bc: ops.residual_norm(
            x, b, w, c, gate=z, scale=s, branch_norm=True, branch_weight=bw, branch_bias=bc)[1],
            (r(3, 8), r(3, 8), r(3, 8), r(8), r(8), r(8), r(8), r(8))),
    }


@pytest.mark.parametrize("name", ["embedding", "scan", "step", "residual"])
@pytest.mark.parametrize("needs_grad", [False, True])
def test_forward_mode_is_refused(cuda, name, needs_grad):
    # a tangent of any argument, of a leaf or not, is never dropped
    from torch.autograd import forward_ad
    call, args = _calls(cuda)[name]
    for i, t in enumerate(args):
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(t.clone().requires_grad_(needs_grad), torch.ones_like(t))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(*args[:i], dual, *args[i + 1:])
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call(*args[:i], dual, *args[i + 1:])
    call(*args)


@pytest.mark.parametrize("name", ["embedding", "scan", "step", "residual"])
def test_transforms_of_torch_func_are_refused(cuda, name):
    call, args = _calls(cuda)[name]
    with pytest.raises(NotImplementedError, match="torch.func"):
        torch.func.vmap(call)(*(t[None] for t in args))
    with pytest.raises(NotImplementedError, match="torch.func|forward-mode"):
        torch.func.jvp(call, args, tuple(torch.ones_like(t) for t in args))
    with pytest.raises(NotImplementedError, match="torch.func"):
        torch.func.grad(lambda *a: call(*a).sum())(*args)


def test_token_models_keep_the_transforms_of_the_plain_embedding(cuda):
    # tangents of the tables, vmap over ids, and functional gradients, as the PyTorch expression
    from torch.autograd import forward_ad
    from mk_iii_technologies_tsrn_b200 import dropin
    m = dropin.TropicalDecoderModel(V, d_model=32, nhead=4, num_layers=1, dim_feedforward=64,
                                    dropout=0.0, max_seq_len=T).to(cuda).eval()
    ids = _ids(cuda)
    at = torch.arange(T, device=cuda)
    w, p = m.embed.weight.detach(), m.pos_embed.weight.detach()
    plain = lambda w, p, i=ids: w[i] * m.embed_scale + p[at][None]  # noqa: E731

    def functional(w, p, i=ids):
        old = m.embed.weight, m.pos_embed.weight
        del m.embed.weight, m.pos_embed.weight
        m.embed.weight, m.pos_embed.weight = w, p
        try:
            return m._embed(i)
        finally:
            del m.embed.weight, m.pos_embed.weight
            m.embed.weight, m.pos_embed.weight = old

    g = torch.Generator(device=cuda).manual_seed(22)
    tw, tp = (torch.randn(t.shape, device=cuda, generator=g) for t in (w, p))
    with forward_ad.dual_level():
        out = functional(forward_ad.make_dual(w, tw), forward_ad.make_dual(p, tp))
        tangent = forward_ad.unpack_dual(out).tangent
        assert tangent is not None
        torch.testing.assert_close(tangent, plain(tw, tp), rtol=1e-6, atol=1e-5)
    out, tangent = torch.func.jvp(functional, (w, p), (tw, tp))
    torch.testing.assert_close(tangent, plain(tw, tp), rtol=1e-6, atol=1e-5)
    got = torch.func.vmap(lambda i: m._embed(i[None])[0])(ids)
    assert torch.equal(got, plain(w, p))
    d = torch.randn_like(out)
    for a, b in zip(torch.func.grad(lambda w, p: (functional(w, p) * d).sum(), (0, 1))(w, p),
                    torch.func.grad(lambda w, p: (plain(w, p) * d).sum(), (0, 1))(w, p)):
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("kind", ["forward", "forward_pre", "full_backward", "full_backward_pre"])
def test_global_module_hooks_see_the_token_models_tables(cuda, kind):
    from mk_iii_technologies_tsrn_b200 import dropin
    from torch.nn.modules import module
    m = dropin.TropicalDecoderModel(V, d_model=32, nhead=4, num_layers=1, dim_feedforward=64,
                                    dropout=0.0, max_seq_len=T).to(cuda)
    ids, seen = _ids(cuda), []
    want = m._embed(ids)
    h = getattr(module, f"register_module_{kind}_hook")(lambda mod, *a: seen.append(mod) and None)
    try:
        x = m._embed(ids)
        x.sum().backward()
    finally:
        h.remove()
    assert torch.equal(x, want) and m.embed in seen and m.pos_embed in seen


def test_a_table_with_a_forward_of_its_own_runs_it(cuda):
    from mk_iii_technologies_tsrn_b200 import dropin
    m = dropin.TropicalDecoderModel(V, d_model=32, nhead=4, num_layers=1, dim_feedforward=64,
                                    dropout=0.0, max_seq_len=T).to(cuda)
    ids = _ids(cuda)
    plain = m.embed.forward
    m.embed.forward = lambda i: plain(i) * 3
    want = plain(ids) * 3 * m.embed_scale + m.pos_embed(torch.arange(T, device=cuda))[None]
    assert torch.equal(m._embed(ids), want)


def test_gradients_taken_as_constants_are_warned_of(cuda):
    # create_graph=True of constant incoming gradients: a gradient that depends on what requires a
    # gradient comes without its graph, and a penalty on it would add nothing without a word
    import warnings
    from mk_iii_technologies_tsrn_b200 import ops
    g = torch.Generator(device=cuda).manual_seed(23)
    shape = (2, 5, 8)

    def ask(call, args, of):
        ts = [torch.randn(s, device=cuda, generator=g).requires_grad_(k in of)
              for k, s in enumerate(args)]
        out = call(*ts)
        with warnings.catch_warnings(record=True) as seen:
            warnings.simplefilter("always")
            torch.autograd.grad(out, [t for t in ts if t.requires_grad], torch.ones_like(out),
                                create_graph=True, retain_graph=True)
            torch.autograd.grad(out, [t for t in ts if t.requires_grad][-1:],
                                torch.ones_like(out), create_graph=True, retain_graph=True)
            said = sum("first derivatives only" in str(w.message) for w in seen)
            torch.autograd.grad(out, [t for t in ts if t.requires_grad], torch.ones_like(out))
            assert said == sum("first derivatives only" in str(w.message) for w in seen)
        return said

    def scan(z, x, h):
        return ops.gated_scan(z, x, h, form="sigmoid")

    def norm(x, b, w, c):
        return ops.residual_norm(x, b, w, c)[1]

    def product(x, b, z, s):
        return ops.residual_norm(x, b, gate=z, scale=s, normalize=False)[0]

    def normed(x, b, w):
        return ops.residual_norm(x, b, branch_norm=True, branch_weight=w, normalize=False)[0]

    sizes = (shape, shape, (2, 8))
    assert ask(scan, sizes, {0}) == 2 and ask(scan, sizes, {0, 1}) == 2
    assert ask(scan, sizes, {1, 2}) == 0                     # linear in x and h0
    assert ask(norm, (shape, shape, (8,), (8,)), {0}) == 2
    assert ask(norm, (shape, shape, (8,), (8,)), {1, 3}) == 2
    assert ask(norm, (shape, shape, (8,), (8,)), {2, 3}) == 0
    sizes = (shape, shape, shape, (8,))
    assert ask(product, sizes, {2}) == 2 and ask(product, sizes, {1, 3}) == 2
    assert ask(product, sizes, {0, 1}) == 0 and ask(product, sizes, {0, 3}) == 0
    assert ask(normed, (shape, shape, (8,)), {1}) == 2 and ask(normed, (shape, shape, (8,)), {2}) == 0
    ids = torch.randint(0, 7, (2, 3), device=cuda, generator=g)
    assert ask(lambda w: ops.embedding(ids, w), ((7, 8),), {0}) == 0
