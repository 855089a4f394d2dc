"""Measured cases of the language-model operators: the scaled token embedding, the gated linear
recurrence, and the residual step with the norms around a block.

``run`` computes an operator in its plain form (elementary torch operations in 32 bits, rounded
once at the end) or, with ``own`` set, through the framework's public calls::

    ops.embedding(ids, weight, scale, pos_weight=, positions=, padding_idx=)
    ops.gated_scan(gate, x, h0, form=, lengths=, return_state=)
    ops.gated_scan_step(gate, x, state, form=)
    ops.residual_norm(x, branch, weight, bias, eps, norm=, gate=, scale=, branch_norm=, branch_weight=, branch_bias=)

Sizes are this repository's (640 channels, byte vocabulary, batch 64 of 1024 tokens; scans of
16 x 4096 x 1024; 512 channels and 2048 positions of the decoder model) and generic ones.
"""
import math

import torch

own = False

_DEV = "cuda"
_MOST_BYTES = 2.2e9  # no drawn case moves more than the largest listed one


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _esize(case):
    return 2 if case["dtype"] == "bf16" else 4


# ----------------------------------------------------------------------------- cases
def _embed(name, B, T, V, D, dtype, pos, train, pad=False):
    """pos: "none", "row" (the index in the sequence) or "given" (a tensor of positions)."""
    return {"name": name, "op": "embed", "B": B, "T": T, "V": V, "D": D, "L": max(T, 2048), "dtype": dtype,
            "pos": pos, "train": train, "pad": pad}


def _scan_case(name, B, T, C, dtype, form, train, ragged=False):
    return {"name": name, "op": "scan", "B": B, "T": T, "C": C, "dtype": dtype, "form": form, "train": train,
            "ragged": ragged}


def _res(name, R, D, dtype, norm, train, gate, scale, branch_norm):
    """scale: "none", "one" (a learnt scalar) or "channel" (one of each channel)."""
    return {"name": name, "op": "res", "R": R, "D": D, "dtype": dtype, "norm": norm, "train": train, "gate": gate,
            "scale": scale, "branch_norm": branch_norm}


def listed():
    return [
        # one token of each of 64 sequences, every one at its own position: a serving step
        _embed("embed_decode", 64, 1, 32000, 512, "f32", "given", False),
        # the TSRN language model on bytes: few rows, each met very often
        _embed("embed_train_bytes", 64, 1024, 256, 640, "f32", "none", True),
        # a subword vocabulary with learnt positions and a padded batch
        _embed("embed_train_subword", 16, 2048, 49999, 512, "bf16", "row", True, pad=True),
        # a large vocabulary, most of its rows absent from the batch
        _embed("embed_train_large", 32, 4096, 131072, 1024, "bf16", "none", True),
        # one token of 32 sequences: a serving step on the recurrent state
        {"name": "scan_step", "op": "step", "B": 32, "C": 640, "dtype": "f32", "form": "sigmoid"},
        # a padded batch of odd size
        _scan_case("scan_train_ragged", 6, 1537, 1000, "bf16", "sigmoid", True, ragged=True),
        # the scan workload's size
        _scan_case("scan_train_batch", 16, 4096, 1024, "f32", "decay", True),
        # one long document
        _scan_case("scan_train_long", 1, 65536, 640, "bf16", "sigmoid", True),
        # one token of 32 sequences between two blocks
        _res("residual_decode", 32, 640, "f32", "layer", False, True, "one", False),
        # the TSRN block's residual stream in training: gate, learnt mix, next block's LayerNorm
        _res("residual_train_block", 65536, 640, "f32", "layer", True, True, "one", False),
        # norms before and after the block, a scale of each channel
        _res("residual_train_sandwich", 16384, 2048, "bf16", "rms", True, False, "channel", True),
        # odd sizes, everything switched on
        _res("residual_train_odd", 4099, 1000, "bf16", "layer", True, True, "channel", True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _one(rng):
    dtype = rng.choice(["f32", "bf16"])
    op = rng.choice(["embed", "embed", "scan", "scan", "step", "res", "res"])
    if op == "embed":
        T = _log(rng, 1, 4096)
        c = _embed("", _log(rng, 1, 128), T, _log(rng, 200, 140000), rng.randint(16, 160) * 8 - rng.choice([0, 0, 0, 1, 4]),
                   dtype, rng.choice(["none", "row", "given"]), rng.random() < 0.8, pad=rng.random() < 0.3)
    elif op == "scan":
        c = _scan_case("", _log(rng, 1, 64), _log(rng, 2, 65536), rng.randint(8, 160) * 8 - rng.choice([0, 0, 0, 1, 4]),
                       dtype, rng.choice(["decay", "sigmoid"]), rng.random() < 0.8, ragged=rng.random() < 0.3)
    elif op == "step":
        c = {"name": "", "op": "step", "B": _log(rng, 1, 1024), "C": rng.randint(16, 2048), "dtype": dtype,
             "form": rng.choice(["decay", "sigmoid"])}
    else:
        c = _res("", _log(rng, 1, 70000), rng.randint(16, 512) * 8 - rng.choice([0, 0, 0, 1, 4]), dtype,
                 rng.choice(["layer", "rms"]), rng.random() < 0.8, rng.random() < 0.5, rng.choice(["none", "one", "channel"]),
                 rng.random() < 0.5)
    return {k: v for k, v in c.items() if k != "name"}


def draw(rng):
    c = _one(rng)
    while work(c)["bytes"] > _MOST_BYTES:
        c = _one(rng)
    return c


# ----------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=_DEV).manual_seed(int(seed) * 2654435761 % (1 << 62) + 17)


def prepare(case, seed):
    g, dt, op = _gen(seed), _dtype(case), case["op"]

    def randn(*shape, std=1.0, mean=0.0, dtype=dt):
        return torch.empty(shape, device=_DEV, dtype=torch.float32).normal_(mean, std, generator=g).to(dtype)

    s = {"case": dict(case)}
    if op == "embed":
        B, T, V, D = (case[k] for k in "BTVD")
        # token ids fall off as 1 / rank, as in text; the ranks are spread over the table
        u = torch.rand(B, T, device=_DEV, generator=g, dtype=torch.float64)
        ids = torch.exp(u * math.log(V + 1.0)).long().sub_(1).clamp_(0, V - 1)
        ids = (ids * 7919 + 13) % V
        if case["pad"]:  # right-padded with id 0
            keep = torch.randint(max(1, T // 2), T + 1, (B, 1), device=_DEV, generator=g)
            ids = torch.where(torch.arange(T, device=_DEV)[None] < keep, ids, torch.zeros_like(ids))
        s.update(ids=ids, weight=randn(V, D, std=D ** -0.5), scale=math.sqrt(D), pos=None, positions=None,
                 padding_idx=0 if case["pad"] else None)
        if case["pos"] != "none":
            s["pos"] = randn(case["L"], D, std=0.02)
        if case["pos"] == "given":
            start = torch.randint(0, case["L"] - T + 1, (B, 1), device=_DEV, generator=g)
            s["positions"] = start + torch.arange(T, device=_DEV)[None]
        if case["train"]:
            s["dout"] = randn(B, T, D)
            s["weight"].requires_grad_()
            if s["pos"] is not None:
                s["pos"].requires_grad_()
    elif op in ("scan", "step"):
        B, C = case["B"], case["C"]
        shape = (B, case["T"], C) if op == "scan" else (B, C)
        gate = randn(*shape, mean=2.0, dtype=torch.float32)   # a memory of about ten steps, some far longer
        s["gate"] = (gate if case["form"] == "sigmoid" else torch.sigmoid(gate)).to(dt)
        s["x"] = randn(*shape)
        s["h0"] = randn(B, C, dtype=torch.float32)
        s["lengths"] = None
        if op == "scan" and case["ragged"]:
            s["lengths"] = torch.randint(max(1, case["T"] // 2), case["T"] + 1, (B,), device=_DEV, generator=g,
                                         dtype=torch.int32)
            s["lengths"][0] = case["T"]
        if op == "scan" and case["train"]:
            s["dh"], s["dlast"] = randn(*shape), randn(B, C, dtype=torch.float32)
            for k in ("gate", "x", "h0"):
                s[k].requires_grad_()
    else:
        R, D = case["R"], case["D"]
        s["x"], s["branch"] = randn(R, D), randn(R, D, mean=0.1)
        s["gate"] = randn(R, D) if case["gate"] else None
        # parameters are kept in 32 bits, as in mixed-precision training
        s["scale"] = {"none": None, "one": randn(1, std=0.1, mean=0.5, dtype=torch.float32),
                      "channel": randn(D, std=0.1, mean=0.5, dtype=torch.float32)}[case["scale"]]
        s["weight"] = randn(D, std=0.1, mean=1.0, dtype=torch.float32)
        s["bias"] = randn(D, std=0.1, dtype=torch.float32) if case["norm"] == "layer" else None
        s["branch_weight"] = randn(D, std=0.1, mean=1.0, dtype=torch.float32) if case["branch_norm"] else None
        s["branch_bias"] = randn(D, std=0.1, dtype=torch.float32) if case["branch_norm"] and case["norm"] == "layer" else None
        if case["train"]:
            s["dy"], s["dn"] = randn(R, D), randn(R, D)
            for k in _RES_INPUTS:
                if s[k] is not None:
                    s[k].requires_grad_()
    return s


_RES_INPUTS = ("x", "branch", "gate", "scale", "weight", "bias", "branch_weight", "branch_bias")
_EPS = 1e-5


# ----------------------------------------------------------------------------- one pass
def run(s):
    op = s["case"]["op"]
    if own:
        return {"embed": _own_embed, "scan": _own_scan, "step": _own_step, "res": _own_res}[op](s)
    with torch.no_grad():
        return {"embed": _plain_embed, "scan": _plain_scan, "step": _plain_step, "res": _plain_res}[op](s)


def _own_embed(s):
    from mk_iii_technologies_tsrn_b200 import ops
    out = ops.embedding(s["ids"], s["weight"], s["scale"], pos_weight=s["pos"], positions=s["positions"],
                        padding_idx=s["padding_idx"])
    r = {"out": out}
    if s["case"]["train"]:
        wanted = [s["weight"]] + ([s["pos"]] if s["pos"] is not None else [])
        got = torch.autograd.grad(out, wanted, s["dout"])
        r["dweight"] = got[0]
        if s["pos"] is not None:
            r["dpos"] = got[1]
    return r


def _own_scan(s):
    from mk_iii_technologies_tsrn_b200 import ops
    h, last = ops.gated_scan(s["gate"], s["x"], s["h0"], form=s["case"]["form"], lengths=s["lengths"], return_state=True)
    r = {"h": h, "last": last}
    if s["case"]["train"]:
        r["dgate"], r["dx"], r["dh0"] = torch.autograd.grad((h, last), (s["gate"], s["x"], s["h0"]), (s["dh"], s["dlast"]))
    return r


def _own_step(s):
    from mk_iii_technologies_tsrn_b200 import ops
    return {"h": ops.gated_scan_step(s["gate"], s["x"], s["h0"], form=s["case"]["form"]), "state": s["h0"]}


def _own_res(s):
    from mk_iii_technologies_tsrn_b200 import ops
    c = s["case"]
    y, n = ops.residual_norm(s["x"], s["branch"], s["weight"], s["bias"], _EPS, norm=c["norm"], gate=s["gate"], scale=s["scale"],
                             branch_norm=c["branch_norm"], branch_weight=s["branch_weight"], branch_bias=s["branch_bias"])
    r = {"y": y, "n": n}
    if c["train"]:
        names = [k for k in _RES_INPUTS if s[k] is not None]
        got = torch.autograd.grad((y, n), [s[k] for k in names], (s["dy"], s["dn"]))
        r.update({"d" + k: v for k, v in zip(names, got)})
    return r


# ----------------------------------------------------------------------------- plain forms
def _plain_embed(s):
    c, dt = s["case"], _dtype(s["case"])
    ids, T = s["ids"], s["case"]["T"]
    out = s["weight"][ids].float() * s["scale"]
    if s["pos"] is not None:
        out = out + (s["pos"][:T] if s["positions"] is None else s["pos"][s["positions"]]).float()
    r = {"out": out.to(dt)}
    if c["train"]:
        d = s["dout"].float().reshape(-1, c["D"])
        dw = torch.zeros(c["V"], c["D"], device=_DEV).index_add_(0, ids.reshape(-1), d * s["scale"])
        if s["padding_idx"] is not None:
            dw[s["padding_idx"]] = 0
        r["dweight"] = dw.to(dt)
        if s["pos"] is not None:
            dp = torch.zeros(c["L"], c["D"], device=_DEV)
            if s["positions"] is None:
                dp[:T] = s["dout"].float().sum(0)
            else:
                dp.index_add_(0, s["positions"].reshape(-1), d)
            r["dpos"] = dp.to(dt)
    return r


def _recur(a, u):
    """h[:, t] = a[:, t] * h[:, t - 1] + u[:, t] from a zero state: pairs of steps are joined, the half
    as long recurrence solved, and the steps between filled in."""
    T = a.shape[1]
    if T == 1:
        return u
    n = T // 2 * 2
    h = torch.empty_like(u)
    h[:, 1:n:2] = _recur(a[:, 0:n:2] * a[:, 1:n:2], a[:, 1:n:2] * u[:, 0:n:2] + u[:, 1:n:2])
    h[:, 0] = u[:, 0]
    h[:, 2::2] = a[:, 2::2] * h[:, 1:T - 1:2] + u[:, 2::2]
    return h


def _plain_scan(s):
    c, dt = s["case"], _dtype(s["case"])
    z, x, h0 = s["gate"].float(), s["x"].float(), s["h0"]
    if c["form"] == "sigmoid":
        a, rest = torch.sigmoid(z), torch.sigmoid(-z)
        u = rest * x
    else:
        a, u = z, x
    live = None
    if s["lengths"] is not None:  # past its length a row keeps its state
        live = (torch.arange(c["T"], device=_DEV)[None] < s["lengths"][:, None])[..., None]
        a, u = torch.where(live, a, 1.0), torch.where(live, u, 0.0)
    first = u[:, :1] + a[:, :1] * h0[:, None]
    h = _recur(a, torch.cat((first, u[:, 1:]), 1))
    out = h if live is None else torch.where(live, h, 0.0)
    r = {"h": out.to(dt), "last": h[:, -1].contiguous()}
    if c["train"]:
        dh = s["dh"].float() if live is None else torch.where(live, s["dh"].float(), 0.0)
        dh = torch.cat((dh[:, :-1], dh[:, -1:] + s["dlast"][:, None]), 1)
        later = torch.cat((a[:, 1:], torch.zeros_like(a[:, :1])), 1)
        g = _recur(later.flip(1), dh.flip(1)).flip(1)
        before = torch.cat((h0[:, None], h[:, :-1]), 1)
        dx, dz = g, g * before
        if c["form"] == "sigmoid":
            dx, dz = g * rest, g * (before - x) * a * rest
        if live is not None:
            dx, dz = torch.where(live, dx, 0.0), torch.where(live, dz, 0.0)
        r.update(dgate=dz.to(dt), dx=dx.to(dt), dh0=a[:, 0] * g[:, 0])
    return r


def _plain_step(s):
    z, x = s["gate"].float(), s["x"].float()
    if s["case"]["form"] == "sigmoid":
        h = torch.sigmoid(z) * s["h0"] + torch.sigmoid(-z) * x
    else:
        h = z * s["h0"] + x
    s["h0"].copy_(h)
    return {"h": h.to(_dtype(s["case"])), "state": s["h0"]}


def _normal(v, norm):
    """(v without its mean and of unit size, 1 / size) of each row."""
    if norm == "layer":
        v = v - v.mean(-1, keepdim=True)
    r = 1.0 / torch.sqrt((v * v).mean(-1, keepdim=True) + _EPS)
    return v * r, r


def _normal_back(d, hat, r, norm):
    """The gradient of a row from that of its normalised form."""
    d = d - hat * (d * hat).mean(-1, keepdim=True) - (d.mean(-1, keepdim=True) if norm == "layer" else 0.0)
    return r * d


def _plain_res(s):
    c, dt = s["case"], _dtype(s["case"])
    norm = c["norm"]
    p = s["branch"].float()
    if c["branch_norm"]:
        bhat, br = _normal(p, norm)
        p = bhat * s["branch_weight"]
        if s["branch_bias"] is not None:
            p = p + s["branch_bias"]
    sg = torch.sigmoid(s["gate"].float()) if c["gate"] else None
    t = p if sg is None else sg * p
    y = s["x"].float() + (t if s["scale"] is None else s["scale"] * t)
    hat, rr = _normal(y, norm)
    n = hat * s["weight"]
    if s["bias"] is not None:
        n = n + s["bias"]
    r = {"y": y.to(dt), "n": n.to(dt)}
    if c["train"]:
        dn = s["dn"].float()
        r["dweight"] = (dn * hat).sum(0)
        if s["bias"] is not None:
            r["dbias"] = dn.sum(0)
        dy = s["dy"].float() + _normal_back(dn * s["weight"], hat, rr, norm)
        r["dx"] = dy.to(dt)
        if s["scale"] is not None:
            r["dscale"] = (dy * t).sum(0) if c["scale"] == "channel" else (dy * t).sum().reshape(1)
            dy = dy * s["scale"]
        if sg is not None:
            r["dgate"] = (dy * p * sg * (1.0 - sg)).to(dt)
            dy = dy * sg
        if c["branch_norm"]:
            r["dbranch_weight"] = (dy * bhat).sum(0)
            if s["branch_bias"] is not None:
                r["dbranch_bias"] = dy.sum(0)
            dy = _normal_back(dy * s["branch_weight"], bhat, br, norm)
        r["dbranch"] = dy.to(dt)
    return r


# ----------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"embed": _exact_embed, "scan": _exact_scan, "step": _exact_step, "res": _exact_res}[case["op"]](s)


def _exact_embed(s):
    c = s["case"]
    T, V, D = c["T"], c["V"], c["D"]
    with torch.no_grad():
        out = torch.index_select(s["weight"].double(), 0, s["ids"].reshape(-1)).mul_(s["scale"]).view(-1, T, D)
        where = None
        if s["pos"] is not None:
            where = s["positions"] if s["positions"] is not None else torch.arange(T, device=_DEV).expand(c["B"], T)
            out += torch.index_select(s["pos"].double(), 0, where.reshape(-1)).view(-1, T, D)
        r = {"out": out}
        if c["train"]:
            d = s["dout"].double().reshape(-1, D)
            ids, d0 = s["ids"].reshape(-1), d
            if s["padding_idx"] is not None:
                some = ids != s["padding_idx"]
                ids, d0 = ids[some], d[some]
            r["dweight"] = torch.zeros(V, D, device=_DEV, dtype=torch.float64).index_put_((ids,), d0 * s["scale"], accumulate=True)
            if where is not None:
                r["dpos"] = torch.zeros(c["L"], D, device=_DEV, dtype=torch.float64).index_put_((where.reshape(-1),), d, accumulate=True)
    return r


def _exact_scan(s):
    c = s["case"]
    T, sig = c["T"], c["form"] == "sigmoid"
    with torch.no_grad():
        z, x = s["gate"].double().transpose(0, 1).contiguous(), s["x"].double().transpose(0, 1).contiguous()
        a = 1.0 / (1.0 + torch.exp(-z)) if sig else z
        u = x / (1.0 + torch.exp(z)) if sig else x
        n = s["lengths"].tolist() if s["lengths"] is not None else [T] * c["B"]
        live = torch.tensor([[t < k for k in n] for t in range(T)], device=_DEV)[..., None]
        keep = not bool(live.all())
        h, hs = s["h0"].double(), torch.empty_like(x)
        for t in range(T):
            new = torch.addcmul(u[t], a[t], h)
            h = torch.where(live[t], new, h) if keep else new
            hs[t] = h
        out = torch.where(live, hs, 0.0) if keep else hs
        r = {"h": out.transpose(0, 1).contiguous(), "last": h}
        if c["train"]:
            dh = s["dh"].double().transpose(0, 1).contiguous()
            c_in, gs = s["dlast"].double(), torch.empty_like(x)  # the gradient of the state after step t
            for t in range(T - 1, -1, -1):
                g = dh[t] + c_in
                gs[t] = g
                c_in = torch.where(live[t], a[t] * g, c_in) if keep else a[t] * g
            before = torch.cat((s["h0"].double()[None], hs[:-1]))
            if sig:
                dz, dx = gs * (a * (1.0 - a) * before - a * u), gs * (1.0 / (1.0 + torch.exp(z)))
            else:
                dz, dx = gs * before, gs
            if keep:
                dz, dx = torch.where(live, dz, 0.0), torch.where(live, dx, 0.0)
            r.update(dgate=dz.transpose(0, 1).contiguous(), dx=dx.transpose(0, 1).contiguous(), dh0=c_in)
    return r


def _exact_step(s):
    z, x = s["gate"].double(), s["x"].double()
    a = 1.0 / (1.0 + torch.exp(-z)) if s["case"]["form"] == "sigmoid" else z
    h = a * s["h0"].double() + (x / (1.0 + torch.exp(z)) if s["case"]["form"] == "sigmoid" else x)
    return {"h": h, "state": h}


def _exact_res(s):
    c = s["case"]
    v = {k: s[k].detach().double().requires_grad_(c["train"]) if s[k] is not None else None for k in _RES_INPUTS}

    def norm(t, w, b):
        if c["norm"] == "layer":
            t = t - t.mean(-1, keepdim=True)
        t = t / (t.square().mean(-1, keepdim=True) + _EPS).sqrt() * w
        return t if b is None else t + b

    p = norm(v["branch"], v["branch_weight"], v["branch_bias"]) if c["branch_norm"] else v["branch"]
    if c["gate"]:
        p = p / (1.0 + torch.exp(-v["gate"]))
    if v["scale"] is not None:
        p = p * v["scale"]
    y = v["x"] + p
    n = norm(y, v["weight"], v["bias"])
    r = {"y": y.detach(), "n": n.detach()}
    if c["train"]:
        names = [k for k in _RES_INPUTS if v[k] is not None]
        got = torch.autograd.grad((y, n), [v[k] for k in names], (s["dy"].double(), s["dn"].double()))
        r.update({"d" + k: g for k, g in zip(names, got)})
    return r


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    e, op = _esize(case), case["op"]
    if op == "embed":
        N, D, V, L = case["B"] * case["T"], case["D"], case["V"], case["L"]
        met = V * (1.0 - math.exp(-N / V))                    # about the rows that are met (at most; ids are skewed)
        n_pos = 0 if case["pos"] == "none" else (case["T"] if case["pos"] == "row" else min(L, N))
        b = 8.0 * N * (2 if case["pos"] == "given" else 1) + e * D * (min(met, N) + n_pos + N)
        f = N * D * (1.0 + (n_pos > 0))
        if case["train"]:
            b += 8.0 * N + e * D * (N + V + (L if n_pos else 0))
            f += N * D * (1.0 + (n_pos > 0))
        return {"bytes": b, "flops": f}
    if op == "step":
        n = case["B"] * case["C"]
        return {"bytes": n * (3.0 * e + 8.0), "flops": 4.0 * n}
    if op == "scan":
        n, s = case["B"] * case["T"] * float(case["C"]), case["B"] * case["C"] * 4.0
        per = 3 + (5 if case["train"] else 0)                 # gate, x, h; then gate, x, dh, dgate, dx
        return {"bytes": n * e * per + s * (4 if case["train"] else 2), "flops": n * (4.0 + (10.0 if case["train"] else 0.0))}
    n, D = case["R"] * float(case["D"]), case["D"]
    k = 4 + (1 if case["gate"] else 0) + ((6 + (2 if case["gate"] else 0)) if case["train"] else 0)
    params = D * 4.0 * 4 * (2 if case["train"] else 1)
    return {"bytes": n * e * k + params, "flops": n * (12.0 + (30.0 if case["train"] else 0.0))}
