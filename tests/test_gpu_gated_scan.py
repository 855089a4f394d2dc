"""ops.gated_scan / gated_scan_step against the recurrence in 64 bits.

Error bound.  With u = 2^-24, a term u_s of h_t passes t - s products with gates; each product and
each addition on the way (a step's multiply-add, or a run's product and its application) loses at
most u of a value not above M_t = |a_t| M_{t-1} + |u_t|.  A sigmoid gate adds its own error: the
exponential 1 ulp, 1 + e half, the quotient 2, the product half: at most 4 ulp = 8 u.  Gates in bf16
take e as one power of two, and the rounded argument adds to it: the constant log2(e) is off by
0.23 u of itself and the product by u, so the exponent by 1.5 u |z| log2(e) and e by 1.5 |z| u; the
power itself 4 u, 1 + e one u, the reciprocal 2 u, the product e / (1 + e) one u: (8 + 1.5 |z|) u.
So with K = 2 (decay), 12 (sigmoid) or 12 + 1.5 |z| (sigmoid of bf16) the error stays below u N_t, N_t = |a_t| (N_{t-1} + K M_{t-1}) +
K |u_t|, computed in 64 bits beside the recurrence; the gradients' bounds follow from those of g
(the same recurrence backwards) and h.  A result is rounded once to its type: half a step more."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
TYPES = [torch.float32, torch.bfloat16]
FORMS = ["decay", "sigmoid"]


def _make(cuda, B, T, C, dtype, form, seed=0, lengths=None):
    g = torch.Generator(device=cuda).manual_seed(seed)
    z = torch.randn(B, T, C, device=cuda, generator=g) * 2 + 1
    gate = (z if form == "sigmoid" else torch.tanh(z)).to(dtype)
    x = torch.randn(B, T, C, device=cuda, generator=g).to(dtype)
    h0 = torch.randn(B, C, device=cuda, generator=g)
    dh = torch.randn(B, T, C, device=cuda, generator=g).to(dtype)
    dl = torch.randn(B, C, device=cuda, generator=g)
    n = None if lengths is None else torch.tensor(lengths, device=cuda, dtype=torch.int32)
    return gate, x, h0, dh, dl, n


def _reference(gate, x, h0, dh, dl, lengths, form):
    """Values and error bounds (before the last rounding) in 64 bits on the CPU: a dict of
    name -> (value, bound)."""
    B, T, C = x.shape
    z, xx = gate.double().cpu(), x.double().cpu()
    n = [T] * B if lengths is None else [min(max(int(k), 0), T) for k in lengths]
    live = (torch.arange(T)[None] < torch.tensor(n)[:, None])[..., None].expand(B, T, C)
    K = torch.full_like(z, 2.0)
    if form == "sigmoid":
        K = 12.0 + (1.5 * z.abs() if gate.dtype == torch.bfloat16 else 0 * z)
        a, rest = torch.sigmoid(z), torch.sigmoid(-z)
        u = rest * xx
    else:
        a, rest, u = z, torch.ones_like(z), xx
    h = h0.double().cpu()
    M, N = h.abs(), torch.zeros_like(h)
    H, HM, HN, P, PN = [], [], [], [], []
    for t in range(T):
        P.append(h), PN.append(N + 2 * M)
        aa, uu, k = a[:, t].abs(), u[:, t].abs(), K[:, t]
        hn, Nn, Mn = a[:, t] * h + u[:, t], aa * (N + k * M) + k * uu, aa * M + uu
        h, N, M = (torch.where(live[:, t], *p) for p in ((hn, h), (Nn, N), (Mn, M)))
        H.append(h), HM.append(M), HN.append(N)
    last = (h, U * (N + M))
    c, cM, cN = dl.double().cpu(), dl.double().cpu().abs(), torch.zeros_like(h)
    G, GN = [None] * T, [None] * T
    d = dh.double().cpu()
    for t in range(T - 1, -1, -1):
        g, gM = d[:, t] + c, d[:, t].abs() + cM
        gN = cN + gM
        G[t], GN[t] = g, gN
        aa, k = a[:, t].abs(), K[:, t]
        cn, cNn, cMn = a[:, t] * g, aa * (gN + k * gM), aa * gM
        c, cN, cM = (torch.where(live[:, t], *p) for p in ((cn, c), (cNn, cN), (cMn, cM)))
    out = {"last": last, "dh0": (c, U * (cN + cM))}
    if T:
        stack = lambda v: torch.stack(v, 1)   # noqa: E731
        H, HN, HM, P, PN, G, GN = (stack(v) for v in (H, HN, HM, P, PN, G, GN))
        zero = torch.zeros_like(H)
        out["h"] = (torch.where(live, H, zero), U * (HN + HM))
        dx, dxe = G * rest, U * (GN + K * G.abs()) * rest
        if form == "sigmoid":
            inner, size = rest * P - u, rest * P.abs() + u.abs()
            dz = G * a * inner
            dze = U * a * (GN * inner.abs() + G.abs() * (rest * PN + 3 * K * size))
        else:
            dz = G * P
            dze = U * (GN * P.abs() + G.abs() * (PN + P.abs()))
        out["dx"], out["dgate"] = ((torch.where(live, v, zero), e) for v, e in ((dx, dxe),
                                                                                (dz, dze)))
    return out


def _close(got, ref, what):
    value, bound = ref
    tol = bound * 1.02 + HALF[got.dtype] * (value.abs() + bound) * 1.01
    err = (got.double().cpu() - value).abs()
    assert torch.all(err <= tol), (what, float((err - tol).max()), float(err.max()))


def _check(cuda, gate, x, h0, dh, dl, n, form):
    from mk_iii_technologies_tsrn_b200 import ops
    ref = _reference(gate, x, h0, dh, dl, n, form)
    ins = [t.detach().requires_grad_() for t in (gate, x, h0)]
    h, last = ops.gated_scan(*ins, form=form, lengths=n, return_state=True)
    got = dict(zip(("dgate", "dx", "dh0"), torch.autograd.grad((h, last), ins, (dh, dl))))
    got.update(h=h.detach(), last=last.detach())
    for k, r in ref.items():
        _close(got[k], r, k)
    with torch.no_grad():
        assert torch.equal(ops.gated_scan(gate, x, h0, form=form, lengths=n), h)
    return got


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,T,C", [(1, 0, 5), (1, 1, 1), (2, 2, 3), (3, 15, 32), (2, 16, 33),
                                   (1, 63, 64), (2, 64, 66), (1, 65, 130), (2, 129, 31),
                                   (1, 1000, 48), (2, 1025, 40), (400, 70, 34), (1, 2500, 7)])
def test_against_64_bits(cuda, form, dtype, B, T, C):
    _check(cuda, *_make(cuda, B, T, C, dtype, form, seed=T + C), form)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", TYPES)
def test_lengths_and_garbage_behind_them(cuda, form, dtype):
    T = 300
    lengths = [0, 1, 63, 64, 65, 128, 299, 300, 1000, -4]
    gate, x, h0, dh, dl, n = _make(cuda, len(lengths), T, 34, dtype, form, 3, lengths)
    clean = _check(cuda, gate, x, h0, dh, dl, n, form)
    for b, k in enumerate(lengths):      # what lies behind the end is never read
        k = min(max(k, 0), T)
        gate[b, k:], x[b, k:], dh[b, k:] = float("nan"), float("inf"), float("nan")
    from mk_iii_technologies_tsrn_b200 import ops
    ins = [t.detach().requires_grad_() for t in (gate, x, h0)]
    h, last = ops.gated_scan(*ins, form=form, lengths=n.long(), return_state=True)
    got = torch.autograd.grad((h, last), ins, (dh, dl))
    for k, v in zip(("h", "last", "dgate", "dx", "dh0"), (h, last, *got)):
        assert torch.equal(v, clean[k]), k
    assert torch.equal(last[0], h0[0]) and torch.equal(got[2][0], dl[0])


@pytest.mark.parametrize("dtype", TYPES)
def test_strides(cuda, dtype):
    from mk_iii_technologies_tsrn_b200 import ops
    gate, x, h0, dh, dl, _ = _make(cuda, 3, 100, 36, dtype, "sigmoid", 4)
    ref = ops.gated_scan(gate, x, h0, form="sigmoid")
    packed = torch.stack((gate, x), -2).reshape(3, 100, 72)      # split columns of one product
    odd = torch.cat((gate[..., :1], gate, x[..., :1], x), -1)    # odd offsets
    for gv, xv in ((packed[..., :36], packed[..., 36:]), (odd[..., 1:37], odd[..., 38:]),
                   (gate.transpose(0, 1).contiguous().transpose(0, 1),
                    x.transpose(1, 2).contiguous().transpose(1, 2))):
        assert torch.equal(ops.gated_scan(gv, xv, h0, form="sigmoid"), ref)
        a, b = gv.detach().requires_grad_(), xv.detach().requires_grad_()
        ga, gb = torch.autograd.grad(ops.gated_scan(a, b, h0, form="sigmoid"), (a, b), dh)
        c, d = gate.clone().requires_grad_(), x.clone().requires_grad_()
        gc, gd = torch.autograd.grad(ops.gated_scan(c, d, h0, form="sigmoid"), (c, d), dh)
        assert torch.equal(ga, gc) and torch.equal(gb, gd)


def test_gradient_of_a_gate_shared_by_all_steps(cuda):
    # an expanded gate (strides of zero): autograd sums its gradient; the leaky recurrence
    from mk_iii_technologies_tsrn_b200 import ops
    g = torch.Generator(device=cuda).manual_seed(5)
    a = torch.rand(32, device=cuda, generator=g).requires_grad_()
    x, dh = (torch.randn(2, 90, 32, device=cuda, generator=g) for _ in range(2))
    ga, = torch.autograd.grad(ops.gated_scan(a.expand(2, 90, 32), x), a, dh)
    full = a.detach().expand(2, 90, 32).contiguous().requires_grad_()
    gf, = torch.autograd.grad(ops.gated_scan(full, x), full, dh)
    assert torch.equal(ga, gf.sum((0, 1)))


@pytest.mark.parametrize("form", FORMS)
def test_gradients_of_one_output_alone(cuda, form):
    from mk_iii_technologies_tsrn_b200 import ops
    gate, x, h0, dh, dl, _ = _make(cuda, 2, 77, 34, torch.float32, form, 6)
    ins = [t.requires_grad_() for t in (gate, x, h0)]
    zero_h, zero_l = torch.zeros_like(dh), torch.zeros_like(dl)
    h, last = ops.gated_scan(*ins, form=form, return_state=True)
    full = lambda d, l: torch.autograd.grad((h, last), ins, (d, l), retain_graph=True)  # noqa: E731
    for out, d, ref in ((h, dh, full(dh, zero_l)), (last, dl, full(zero_h, dl))):
        for p, q in zip(torch.autograd.grad(out, ins, d, retain_graph=True), ref):
            assert torch.equal(p, q)
    only, = torch.autograd.grad(h, x, dh, retain_graph=True)
    assert torch.equal(only, full(dh, zero_l)[1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("B,C", [(1, 1), (3, 33), (64, 640), (700, 129)])
def test_steps_equal_the_scan(cuda, form, dtype, B, C):
    # one step is one multiply-add on the same fp32 state, as in a scan of one step
    from mk_iii_technologies_tsrn_b200 import ops
    gate, x, h0, *_ = _make(cuda, B, 5, C, dtype, form, 7)
    pool = torch.full((B, C + 3), 9.0, device=cuda)
    state = pool[:, :C]
    state.copy_(h0)
    carry = h0
    for t in range(5):
        h = ops.gated_scan_step(gate[:, t], x[:, t], state, form=form)
        one, carry = ops.gated_scan(gate[:, t:t + 1], x[:, t:t + 1], carry, form=form,
                                    return_state=True)
        assert torch.equal(h, one[:, 0]) and torch.equal(state, carry)
    assert torch.all(pool[:, C:] == 9.0)
    _close(carry, _reference(gate, x, h0, x, h0, None, form)["last"], "last")


def test_segments_carry_the_state(cuda):
    from mk_iii_technologies_tsrn_b200 import ops
    gate, x, h0, *_ = _make(cuda, 2, 500, 40, torch.float32, "sigmoid", 8)
    ref = _reference(gate, x, h0, x, h0, None, "sigmoid")
    parts, state = [], h0
    for lo, hi in ((0, 130), (130, 131), (131, 131), (131, 500)):
        h, state = ops.gated_scan(gate[:, lo:hi], x[:, lo:hi], state, form="sigmoid",
                                  return_state=True)
        parts.append(h)
    _close(torch.cat(parts, 1), ref["h"], "h")
    _close(state, ref["last"], "last")


def test_extreme_gates(cuda):
    from mk_iii_technologies_tsrn_b200 import ops
    x = torch.randn(1, 200, 4, device=cuda, generator=torch.Generator(device=cuda).manual_seed(9))
    h0 = torch.full((1, 4), 3.0, device=cuda)
    zeros, ones = torch.zeros_like(x), torch.ones_like(x)
    assert torch.equal(ops.gated_scan(zeros, x, h0), x)                       # no memory
    assert torch.all(ops.gated_scan(ones, zeros, h0) == 3.0)                  # full memory
    z = torch.full_like(x, float("inf"))
    assert torch.all(ops.gated_scan(z, x, h0, form="sigmoid") == 3.0)
    assert torch.equal(ops.gated_scan(-z, x, h0, form="sigmoid"), x)
    big = torch.full_like(x, 200.0)
    assert torch.all(ops.gated_scan(big, x, h0, form="sigmoid") == 3.0)
    bad = x.clone()
    bad[0, 50, 1] = float("nan")
    h = ops.gated_scan(ones * 0.5, bad, h0)
    assert torch.all(h[0, 50:, 1].isnan()) and torch.all(h[0, :50].isfinite())
    assert torch.all(h[..., [0, 2, 3]].isfinite())
    # products of gates that overflow meet a zero state: the zero stays
    assert torch.all(ops.gated_scan(ones * 1e30, zeros) == 0)


def test_gradient_against_differences(cuda):
    # central differences of the recurrence in 64 bits along a random direction: their own error is
    # of order e^2 (third derivatives) and 2^-52 / e: far below the fp32 gradient's rounding, for
    # which 1e-5 of the terms' sizes allows (the bound of the docstring summed is below it)
    from mk_iii_technologies_tsrn_b200 import ops
    for form in FORMS:
        gate, x, h0, dh, dl, _ = _make(cuda, 2, 40, 5, torch.float32, form, 10)
        ins = [t.requires_grad_() for t in (gate, x, h0)]
        grads = torch.autograd.grad(ops.gated_scan(*ins, form=form, return_state=True), ins,
                                    (dh, dl))
        base = [t.detach().double().cpu() for t in ins]
        vs = [torch.randn(t.shape, dtype=torch.float64, generator=torch.Generator().manual_seed(i))
              for i, t in enumerate(base)]

        def loss(e):
            z, xx, h = (b + e * v for b, v in zip(base, vs))
            a = torch.sigmoid(z) if form == "sigmoid" else z
            u = torch.sigmoid(-z) * xx if form == "sigmoid" else xx
            total = 0.0
            for t in range(z.shape[1]):
                h = a[:, t] * h + u[:, t]
                total = total + (h * dh[:, t].double().cpu()).sum()
            return total + (h * dl.double().cpu()).sum()

        want = float((loss(1e-5) - loss(-1e-5)) / 2e-5)
        terms = [(g.double().cpu() * v) for g, v in zip(grads, vs)]
        got, size = sum(float(t.sum()) for t in terms), sum(float(t.abs().sum()) for t in terms)
        assert abs(got - want) <= 1e-5 * size


def test_repeat_bits_and_other_stream(cuda):
    from mk_iii_technologies_tsrn_b200 import ops
    gate, x, h0, dh, dl, _ = _make(cuda, 1, 3000, 64, torch.bfloat16, "sigmoid", 11)
    h, last, states = ops.gated_scan_fwd(gate, x, h0, form="sigmoid", need_states=True)
    back = ops.gated_scan_bwd(states, dh, dl, gate, x, form="sigmoid")
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        again = ops.gated_scan_fwd(gate, x, h0, form="sigmoid", need_states=True)
        back2 = ops.gated_scan_bwd(again[2], dh, dl, gate, x, form="sigmoid")
    torch.cuda.synchronize()
    for p, q in zip((h, last, states, *back), (*again, *back2)):
        assert torch.equal(p, q)


def test_captured_and_replayed(cuda):
    from mk_iii_technologies_tsrn_b200 import ops
    gate, x, h0, dh, dl, _ = _make(cuda, 2, 200, 64, torch.float32, "sigmoid", 12)

    def step():
        h, last, states = ops.gated_scan_fwd(gate, x, h0, form="sigmoid", need_states=True)
        return (h, last, *ops.gated_scan_bwd(states, dh, dl, gate, x, form="sigmoid"))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    x.copy_(torch.randn_like(x))
    graph.replay()
    for p, q in zip(out, step()):
        assert torch.equal(p, q)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,T,C", [(2, 300, 36), (3, 65, 2), (1, 2500, 70), (1, 2500, 68)])
def test_rows_that_begin_on_pairs(cuda, form, dtype, B, T, C):
    # channels of an even number that is no multiple of 16 bytes, and the same bits from buffers
    # whose rows begin elsewhere
    gate, x, h0, dh, dl, n = _make(cuda, B, T, C, dtype, form, 13, lengths=[T, T - 7, 1][:B])
    got = _check(cuda, gate, x, h0, dh, dl, n, form)
    for shift in (1, 2):
        views = []
        for t in (gate, x):
            wide = torch.full((B, T, C + 5), float("nan"), device=cuda, dtype=dtype)
            wide[..., shift:shift + C] = t
            views.append(wide[..., shift:shift + C])
        same = _check(cuda, *views, h0, dh, dl, n, form)
        assert all(torch.equal(got[k], same[k]) for k in got)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,C,per", [(64, 8, 8), (300, 33, 8), (2600, 6, 8), (3000, 7, 100)])
def test_products_of_gates_that_overflow_meet_a_zero_gate(cuda, dtype, T, C, per):
    # in every `per` steps, gates whose product leaves fp32's range, on states small enough for the
    # recurrence to stay within it, and then a gate of 0, behind which the state is the input alone.
    # The bound of the docstring counts roundings of normal numbers; dgate's products g h of two
    # values near 1e-32 are below the type's least normal number, where a rounding is off by at most
    # half of the least subnormal one (2^-149 in fp32, 2^-133 in bf16; fp32 underflow as well: twice).
    # 64 steps are whole periods in every run of 8 or 16 steps: all values are the recurrence's.  In
    # the others some runs end between the large gates and the zero: 1e10^4 > 2^128 stays infinite
    # there, and what follows is right, infinite or NaN
    from mk_iii_technologies_tsrn_b200 import ops
    gate, x, h0, dh, dl, _ = _make(cuda, 2, T, C, dtype, "decay", 14)
    n, big = (4, 1e10) if per == 8 else (39, 10.0)
    gate = torch.where(gate.abs() < 0.5, gate, 0.5)
    for k in range(per):
        if k < n:
            gate[:, k::per] = big
        elif k == n:
            gate[:, k::per] = 0
    tiny = 1e-32
    x, h0, dh, dl = x * tiny, h0 * tiny, dh * tiny, dl * tiny
    ins = [t.detach().requires_grad_() for t in (gate, x, h0)]
    h, last = ops.gated_scan(*ins, return_state=True)
    got = dict(zip(("dgate", "dx", "dh0"), torch.autograd.grad((h, last), ins, (dh, dl))))
    got.update(h=h.detach(), last=last.detach())
    for k, (value, bound) in _reference(gate, x, h0, dh, dl, None, "decay").items():
        tol = bound * 1.02 + HALF[got[k].dtype] * (value.abs() + bound) * 1.01
        tol = tol + 2.0 ** -149 + (2.0 ** -134 if got[k].dtype == torch.bfloat16 else 0.0)
        close = (got[k].double().cpu() - value).abs() <= tol
        assert torch.all(close | ~got[k].cpu().isfinite()), k
        assert T > 64 or torch.all(close), k


@pytest.mark.parametrize("T", [64, 2600])
def test_products_of_gates_that_stay_infinite_say_so(cuda, T):
    # products that overflow before small gates bring them back: where the state behind a run is
    # not the recurrence's, it is infinite or NaN, never another number
    from mk_iii_technologies_tsrn_b200 import ops
    gate = torch.full((1, T, 8), 0.5, device=cuda)
    for k in range(4):
        gate[:, k::32], gate[:, k + 4::32] = 1e10, 1e-10
    h0 = torch.full((1, 8), 1e-32, device=cuda)
    x = torch.zeros_like(gate)
    h, last = ops.gated_scan(gate, x, h0, return_state=True)
    want, state = [], h0.double()
    for t in range(T):
        state = state * gate[:, t].double()
        want.append(state)
    want = torch.stack(want, 1)
    close = (h.double() - want).abs() <= 2 * T * U * want.abs() + 2.0 ** -149
    assert torch.all(close | ~h.isfinite())
    assert torch.all((last - h[:, -1] == 0) | ~last.isfinite())
    assert torch.all(ops.gated_scan(gate, x) == 0)


@pytest.mark.parametrize("mean", [2.0, 6.0])
@pytest.mark.parametrize("dtype", TYPES)
def test_fp32_results_have_fp32_gates(cuda, dtype, mean):
    # the state at the end and the gradient of h0 are fp32 whatever the storage: their root mean
    # square error is near that of the recurrence step by step in fp32 with fp32 sigmoids.  In units
    # of a last place the plain complement of a gate has an exponential (0.4), a sum and a quotient
    # (0.29 each, half a step at most), the kernel's a quotient of up to 2 (0.5) and a product (0.29)
    # more: sqrt(0.58 / 0.33) = 1.33 times, less with the roundings that both share
    from mk_iii_technologies_tsrn_b200 import ops
    B, T, C = 4, 1536, 320
    g = torch.Generator(device=cuda).manual_seed(15)
    gate = (torch.randn(B, T, C, device=cuda, generator=g) + mean).to(dtype)
    x, dh = (torch.randn(B, T, C, device=cuda, generator=g).to(dtype) for _ in range(2))
    h0 = torch.randn(B, C, device=cuda, generator=g).requires_grad_()
    h, last = ops.gated_scan(gate, x, h0, form="sigmoid", return_state=True)
    dh0, = torch.autograd.grad(h, h0, dh)

    def plain(to):
        f, r = torch.sigmoid(gate.to(to)), torch.sigmoid(-gate.to(to))
        u, d, s = r * x.to(to), dh.to(to), h0.detach().to(to)
        c = torch.zeros_like(s)
        for t in range(T):
            s = f[:, t] * s + u[:, t]
        for t in range(T - 1, -1, -1):
            c = f[:, t] * (d[:, t] + c)
        return s, c

    rms = lambda v, e: float((v.detach().double() - e).square().mean().sqrt())  # noqa: E731
    for got, one, exact in zip((last, dh0), plain(torch.float32), plain(torch.float64)):
        assert rms(got, exact) <= 1.4 * rms(one, exact)
