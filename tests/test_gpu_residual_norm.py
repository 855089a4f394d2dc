"""ops.residual_norm (branch norm, gate, residual scale and sum, next norm) against the formulas in
64 bits.

Error bounds, u = 2^-24.  A row sum adds at most 24 values in a thread, five pairs in a warp and 16
warps: 45 additions.  A mean is off by at most 45 u mean|v|, so a normalised value by about
(45 + 4) u (c + |v^|), c = 1 + mean|v| / deviation, from the mean and as much again from the
deviation; the affine part, the gate (8 u), the scale and the sum add a few u of the terms:
K = 128 u covers them, relative to the sum of the terms' sizes and to c.  In the backward every
factor is such a value and the two row means cost 45 u of the mean sizes again: 2 K of the terms'
sizes.  Where c is large (rows far from zero mean) so is the bound.  A column sum over R rows adds
at most R u more.  A result is rounded once to its type: half a step more."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
K = 128 * U
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
TYPES = [torch.float32, torch.bfloat16]
EPS = 1e-5
NAMES = ("x", "branch", "gate", "scale", "weight", "bias", "branch_weight", "branch_bias")


def _make(cuda, R, D, dtype, *, norm="layer", gate=True, scale="channel", branch_norm=True,
          affine=True, normalize=True, params=torch.float32, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed)

    def randn(*s, mean=0.0, std=1.0, dt=dtype):
        return (torch.randn(*s, device=cuda, generator=g) * std + mean).to(dt)

    t = {"x": randn(R, D, std=2.0), "branch": randn(R, D, mean=0.3), "gate": None, "scale": None,
         "weight": None, "bias": None, "branch_weight": None, "branch_bias": None}
    if gate:
        t["gate"] = randn(R, D, std=2.0)
    if scale:
        t["scale"] = randn(*((D,) if scale == "channel" else (1,)), mean=0.7, std=0.2, dt=params)
    if affine and normalize:
        t["weight"], t["bias"] = randn(D, mean=1, std=.3, dt=params), randn(D, std=.3, dt=params)
    if affine and branch_norm:
        t["branch_weight"] = randn(D, mean=1, std=.3, dt=params)
        t["branch_bias"] = randn(D, std=.3, dt=params)
    how = dict(norm=norm, branch_norm=branch_norm, normalize=normalize)
    return t, how, randn(R, D), (randn(R, D) if normalize else None)


def _norm64(v, norm):
    m = v.mean(-1, keepdim=True) if norm == "layer" else torch.zeros_like(v[:, :1])
    r = 1.0 / ((v - m).square().mean(-1, keepdim=True) + EPS).sqrt()
    return (v - m) * r, r, 1.0 + v.abs().mean(-1, keepdim=True) * r


def _reference(t, how, dy, dn):
    """name -> (value, error bound before the last rounding), by the formulas in 64 bits."""
    v = {k: (a.double().cpu() if a is not None else None) for k, a in t.items()}
    dy, dn = (a.double().cpu() if a is not None else None for a in (dy, dn))
    R, D = v["x"].shape
    norm, out = how["norm"], {}
    one = torch.ones(D, dtype=torch.float64)
    w, bw = (v[k] if v[k] is not None else one for k in ("weight", "branch_weight"))
    b, bb = (v[k] if v[k] is not None else 0 * one for k in ("bias", "branch_bias"))
    c1 = torch.ones(R, 1, dtype=torch.float64)
    phat = v["branch"]
    if how["branch_norm"]:
        phat, r1, c1 = _norm64(v["branch"], norm)
    p, psize = phat * bw + bb, phat.abs() * bw.abs() + bb.abs()
    perr = K * c1 * (psize + (bw.abs() if how["branch_norm"] else 0))
    sg = torch.sigmoid(v["gate"]) if v["gate"] is not None else torch.ones_like(p)
    sc = v["scale"] if v["scale"] is not None else one[:1]
    branch = sc * sg * p
    y = v["x"] + branch
    yerr = (sc * sg).abs() * (perr + 16 * U * psize) + 2 * U * (y.abs() + branch.abs())
    out["y"] = (y, yerr)
    yh, c2 = y, c1
    if how["normalize"]:
        yh, r2, c2 = _norm64(y, norm)
        rel = r2 * (yerr + yerr.mean(-1, keepdim=True) * (1 + yh.abs()))
        yherr = rel + K * c2 * (1 + yh.abs())
        out["n"] = (yh * w + b, yherr * w.abs() + 4 * U * ((yh * w).abs() + b.abs()))
    if dy is None and dn is None:
        return out
    g = dy if dy is not None else torch.zeros_like(y)
    gsize = g.abs()
    gerr = torch.zeros_like(g)
    mean = lambda a: a.mean(-1, keepdim=True)   # noqa: E731
    col = lambda val, size, err: (val.sum(0), err.sum(0) + R * U * size.sum(0))   # noqa: E731
    c = c1 * c2
    if dn is not None:
        out["weight"] = col(dn * yh, (dn * yh).abs(), dn.abs() * yherr)
        out["bias"] = col(dn, dn.abs(), 0 * dn)
        q = dn * w
        layer = 1.0 if norm == "layer" else 0.0
        g = g + r2 * (q - layer * mean(q) - yh * mean(q * yh))
        size = r2 * (q.abs() + layer * mean(q.abs()) + yh.abs() * mean((q * yh).abs()))
        gerr = 2 * K * c * size + r2 * (yherr * mean((q * yh).abs()) + yh.abs() * mean(
            q.abs() * yherr))
        gsize = gsize + size
    gerr = gerr + 2 * U * gsize
    out["x"] = (g, gerr)
    t1 = sg * p
    terr = sg * (perr + 16 * U * psize)
    out["scale"] = col(g * t1, gsize * (t1.abs() + terr), gsize * terr + gerr * t1.abs() +
                       4 * U * gsize * t1.abs())
    if v["scale"] is not None and v["scale"].numel() == 1 and D > 1:
        val, err = out["scale"]
        out["scale"] = (val.sum(0, keepdim=True), (err.sum() + (D + 64) * U * (
            gsize * t1.abs()).sum()).reshape(1))
    gs, gserr, gssize = g * sc, gerr * sc.abs(), gsize * sc.abs()
    om = 1 - sg if v["gate"] is None else torch.sigmoid(-v["gate"])
    f = p * sg * om
    out["gate"] = (gs * f, gserr * f.abs() + gssize * sg * om * (perr + 40 * U * psize))
    d, derr, dsize = gs * sg, gserr * sg + 16 * U * gssize * sg, gssize * sg
    if how["branch_norm"]:
        pherr = K * c1 * (1 + phat.abs())
        out["branch_weight"] = col(d * phat, dsize * phat.abs(), derr * phat.abs() + dsize * pherr)
        out["branch_bias"] = col(d, dsize, derr)
        q, qerr, qsize = d * bw, derr * bw.abs(), dsize * bw.abs()
        layer = 1.0 if norm == "layer" else 0.0
        d = r1 * (q - layer * mean(q) - phat * mean(q * phat))
        size = r1 * (qsize + layer * mean(qsize) + phat.abs() * mean(qsize * phat.abs()))
        derr = r1 * (qerr + mean(qerr) + phat.abs() * mean(qerr * phat.abs())) + 2 * K * c1 * size
        derr = derr + r1 * (pherr * mean(qsize * phat.abs()) + phat.abs() * mean(qsize * pherr))
    out["branch"] = (d, derr)
    return out


def _close(got, ref, what):
    value, bound = ref
    tol = bound * 1.02 + HALF[got.dtype] * (value.abs() + bound) * 1.01
    err = (got.double().cpu() - value).abs()
    assert torch.all(err <= tol), (what, float((err - tol).max()), float(err.max()))


def _call(t, how, dy, dn):
    from mk_iii_technologies_tsrn_b200 import ops
    ins = {k: a.detach().requires_grad_() for k, a in t.items() if a is not None}
    kw = {k: ins.get(k) for k in ("gate", "scale", "branch_weight", "branch_bias")}
    y, n = ops.residual_norm(ins["x"], ins["branch"], ins.get("weight"), ins.get("bias"), EPS,
                             **kw, **how)
    outs, ds = [], []
    for o, d in ((y, dy), (n, dn)):
        if d is not None:
            outs.append(o), ds.append(d)
    grads = torch.autograd.grad(outs, list(ins.values()), ds, allow_unused=True)
    return y, n, dict(zip(ins, grads))


def _check(t, how, dy, dn):
    ref = _reference(t, how, dy, dn)
    y, n, grads = _call(t, how, dy, dn)
    _close(y.detach(), ref["y"], "y")
    if how["normalize"]:
        _close(n.detach(), ref["n"], "n")
    else:
        assert n is None
    for k, g in grads.items():
        assert g.dtype == t[k].dtype and g.shape == t[k].shape
        _close(g, ref[k], k)
    from mk_iii_technologies_tsrn_b200 import ops
    y2, n2, _ = ops.residual_norm_fwd(t["x"], t["branch"], t["weight"], t["bias"], EPS, gate=t[
        "gate"], scale=t["scale"], branch_weight=t["branch_weight"], branch_bias=t["branch_bias"],
        **how)
    assert torch.equal(y, y2) and (n is None or torch.equal(n, n2))
    for p, q in zip(_call(t, how, dy, dn)[2].values(), grads.values()):
        assert torch.equal(p, q)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,D", [(1, 1), (3, 2), (5, 33), (2, 128), (7, 132), (700, 64), (9, 640),
                                 (1, 641), (50, 1000), (3, 1024), (2, 2048), (5, 2564), (3, 5120),
                                 (2, 6152), (2, 8191), (3, 8192), (3000, 36)])
def test_against_64_bits(cuda, dtype, R, D):
    for norm in ("layer", "rms"):
        _check(*_make(cuda, R, D, dtype, norm=norm, seed=R + D))


@pytest.mark.parametrize("norm,gate,scale,branch_norm,affine,normalize", list(itertools.product(
    ("layer", "rms"), (False, True), (None, "one", "channel"), (False, True), (False, True),
    (False, True))))
def test_every_combination(cuda, norm, gate, scale, branch_norm, affine, normalize):
    for dtype in TYPES:
        _check(*_make(cuda, 37, 72, dtype, norm=norm, gate=gate, scale=scale,
                      branch_norm=branch_norm, affine=affine, normalize=normalize, seed=1))


@pytest.mark.parametrize("norm", ["layer", "rms"])
def test_parameters_in_bf16(cuda, norm):
    _check(*_make(cuda, 20, 200, torch.bfloat16, norm=norm, params=torch.bfloat16, seed=2))


@pytest.mark.parametrize("dtype", TYPES)
def test_one_gradient_alone(cuda, dtype):
    t, how, dy, dn = _make(cuda, 12, 96, dtype, seed=3)
    _check(t, how, dy, torch.zeros_like(dn))
    for a, b in ((dy, None), (None, dn)):
        _, _, alone = _call(t, how, a, b)
        _, _, both = _call(t, how, a if a is not None else torch.zeros_like(dy),
                           b if b is not None else torch.zeros_like(dn))
        for k in alone:
            assert torch.equal(alone[k], both[k]), k


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_shapes(cuda, dtype):
    from mk_iii_technologies_tsrn_b200 import ops
    t, how, dy, dn = _make(cuda, 24, 64, dtype, seed=4)
    y, n, grads = _call(t, how, dy, dn)
    wide = torch.cat((t["gate"], t["branch"], t["x"][:, :3], t["x"]), 1)
    views = dict(t, gate=wide[:, :64], branch=wide[:, 64:128], x=wide[:, 131:])
    for tt in (views, dict(t, x=t["x"].t().contiguous().t())):
        y2, n2, g2 = _call(tt, how, dy, dn)
        # another vector width may sum a row in another order
        for p, q in ((y, y2), (n, n2), *((grads[k], g2[k]) for k in grads)):
            torch.testing.assert_close(p, q, rtol=4 * HALF[p.dtype], atol=2e-5)
    three = {k: (a.view(2, 12, 64) if a is not None and a.dim() == 2 else a) for k, a in t.items()}
    y3, n3, g3 = _call(three, how, dy.view(2, 12, 64), dn.view(2, 12, 64))
    assert y3.shape == (2, 12, 64) and torch.equal(y3.reshape(24, 64), y)
    assert torch.equal(n3.reshape(24, 64), n) and torch.equal(g3["x"].reshape(24, 64), grads["x"])
    empty = {k: (a[:0] if a is not None and a.dim() == 2 else a) for k, a in t.items()}
    y0, n0, g0 = _call(empty, how, dy[:0], dn[:0])
    assert y0.shape == n0.shape == (0, 64)
    assert all(torch.all(g0[k] == 0) for k in ("scale", "weight", "bias", "branch_weight"))
    same = ops.residual_norm(t["x"], t["x"], t["weight"], t["bias"])     # one tensor twice
    copy = ops.residual_norm(t["x"], t["x"].clone(), t["weight"], t["bias"])
    assert torch.equal(same[0], copy[0]) and torch.equal(same[1], copy[1])


def test_constant_rows_and_non_finite_rows(cuda):
    from mk_iii_technologies_tsrn_b200 import ops
    x = torch.zeros(4, 40, device=cuda)
    b = torch.zeros(4, 40, device=cuda)
    x[1] = 5.0
    x[2, 3] = float("nan")
    b[3, 7] = float("inf")
    y, n = ops.residual_norm(x, b, eps=1e-5)
    assert torch.all(n[:2] == 0) and torch.all(y[1] == 5.0)      # no deviation: nothing is left
    assert torch.all(n[2].isnan()) and torch.all(n[3].isnan())   # and a bad row stays a bad row
    assert torch.all(y[2, :3] == 0) and y[3, 7].isinf()


def test_gradient_against_differences(cuda):
    # central differences in 64 bits along a random direction (error e^2 and 2^-52 / e) against the
    # fp32 gradient, whose rounding is far below 1e-4 of the terms' sizes by the bound above
    for norm in ("layer", "rms"):
        t, how, dy, dn = _make(cuda, 6, 20, torch.float32, norm=norm, seed=5)
        _, _, grads = _call(t, how, dy, dn)
        base = {k: a.double().cpu() for k, a in t.items()}
        vs = {k: torch.randn(a.shape, dtype=torch.float64,
                             generator=torch.Generator().manual_seed(i))
              for i, (k, a) in enumerate(base.items())}

        def loss(e):
            v = {k: base[k] + e * vs[k] for k in base}
            p = _norm64(v["branch"], norm)[0] * v["branch_weight"] + v["branch_bias"]
            y = v["x"] + v["scale"] * torch.sigmoid(v["gate"]) * p
            n = _norm64(y, norm)[0] * v["weight"] + v["bias"]
            return (y * dy.double().cpu()).sum() + (n * dn.double().cpu()).sum()

        want = float((loss(1e-5) - loss(-1e-5)) / 2e-5)
        terms = [grads[k].double().cpu() * vs[k] for k in base]
        got, size = sum(float(a.sum()) for a in terms), sum(float(a.abs().sum()) for a in terms)
        assert abs(got - want) <= 1e-4 * size


def test_captured_and_replayed(cuda):
    from mk_iii_technologies_tsrn_b200 import ops
    t, how, dy, dn = _make(cuda, 40, 128, torch.float32, seed=6)
    kw = dict(gate=t["gate"], scale=t["scale"], branch_weight=t["branch_weight"],
              branch_bias=t["branch_bias"], **how)

    def step():
        y, n, st = ops.residual_norm_fwd(t["x"], t["branch"], t["weight"], t["bias"],
                                         need_stats=True, **kw)
        g = ops.residual_norm_bwd(st, dy, dn, t["x"], t["branch"], t["weight"], t["bias"], **kw)
        return [y, n, *g.values()]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    t["x"].copy_(torch.randn_like(t["x"]))
    graph.replay()
    for p, q in zip(out, step()):
        assert torch.equal(p, q)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,D", [(1, 3), (2, 1), (9, 5), (3, 7), (17, 9), (50, 11), (33, 333),
                                 (2000, 101), (21, 641), (13, 767), (19, 1001), (9, 2001),
                                 (9, 4079), (5, 4081), (10, 1028)])
def test_rows_that_begin_inside_16_bytes(cuda, dtype, R, D):
    for how in (dict(), dict(norm="rms", gate=False, branch_norm=False, scale="one")):
        _check(*_make(cuda, R, D, dtype, seed=R, **how))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("more", [3, 8, 24])
def test_odd_rows_of_a_wider_buffer(cuda, dtype, more):
    for D in (43, 901):
        t, how, dy, dn = _make(cuda, 18, D, dtype, seed=7)
        for k in ("x", "branch", "gate"):
            wide = torch.full((18, D + more), float("nan"), device=cuda, dtype=dtype)
            wide[:, :D] = t[k]
            t[k] = wide[:, :D]
        _check(t, how, dy, dn)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_bad_row_leaves_its_neighbours(cuda, dtype):
    # rows of odd lengths share 16 bytes with their neighbours
    for D in (5, 333, 1001):
        t, how, dy, dn = _make(cuda, 20, D, dtype, seed=8)
        bad = {k: (a.clone() if a is not None and a.dim() == 2 else a) for k, a in t.items()}
        bdy, bdn = dy.clone(), dn.clone()
        for a, v in zip((bad["x"], bad["branch"], bad["gate"], bdy, bdn),
                        (float("nan"), float("inf"), float("nan"), float("inf"), float("nan"))):
            a[1::2] = v
        good, hit = _call(t, how, dy, dn), _call(bad, how, bdy, bdn)
        for p, q in ((good[0], hit[0]), (good[1], hit[1]),
                     *((good[2][k], hit[2][k]) for k in ("x", "branch", "gate"))):
            assert torch.equal(p[::2], q[::2])
            assert not torch.any(torch.isfinite(q[1::2]))


def test_the_single_scale_sums_rows_in_64_bits(cuda):
    # every term is 1 + 2^-10 and a row's sum of three exact: what is left is one rounding
    from mk_iii_technologies_tsrn_b200 import ops
    R = 100001
    b = torch.full((R, 3), 1 + 2.0 ** -10, device=cuda)
    scale = torch.ones(1, device=cuda, requires_grad=True)
    y, _ = ops.residual_norm(torch.zeros_like(b), b, scale=scale, normalize=False)
    y.backward(torch.ones_like(y))
    assert scale.grad.item() == torch.tensor(3 * R * (1 + 2.0 ** -10), dtype=torch.float64).float()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,D", [(12000, 72), (12000, 71), (6000, 1000), (6000, 1001), (3000, 2048),
                                 (1000, 4099), (1000, 5000)])
def test_more_rows_than_teams(cuda, dtype, R, D):
    # teams of a warp and of a block (aligned rows, rows that begin inside 16 bytes, single
    # channels) take a second row, forwards and backwards: more rows than blocks of one wave
    _check(*_make(cuda, R, D, dtype, seed=4))
