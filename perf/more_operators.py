"""Measured cases of the decoding operators: attention of one new token over a paged key-value
cache, the writing of a prompt into it, eviction from it by accumulated attention weight, and
sampling of the next token.

``run`` computes an operator in its plain form (elementary torch operations in 32 bits, in 64 for
the sampling's sums, rounded once at the end) or, with ``own`` set, through the framework's public
calls::

    ops.paged_attention(q, k_cache, v_cache, block_table, lengths, key=, value=, scale=, gate=, tau=, mass=)
    ops.paged_append(key, value, k_cache, v_cache, block_table, starts, counts)
    ops.cache_evict(k_cache, v_cache, block_table, lengths, mass, keep, recent, out=)
    ops.sample_tokens(logits, uniform, temperature=, top_k=, top_p=, min_p=, return_logprob=True)

A cache is [pages, page size, key heads, channels] with any strides of the first three dimensions;
row b of ``block_table`` lists the pages of sequence b, and slot j of it is in page j // page size.
Sizes are this repository's (8 heads of 64 channels, 2048 positions, byte vocabulary) and generic
ones.
"""
import math

import numpy as np
import torch

own = False

_DEV = "cuda"
_MOST_BYTES = 1.3e9       # no drawn case moves more than the largest listed one
_MOST_SUMS = 1 << 29      # nor forms more tropical sums than the plain form can hold


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _esize(case):
    return 2 if case["dtype"] == "bf16" else 4


# ----------------------------------------------------------------------------- cases
def _attn(name, B, H, Hkv, D, L, page, dtype, gated, mass, store=True, ragged=True, layout="slots"):
    """layout: "slots" (a page holds its slots one after another) or "heads" (its heads)."""
    return {"name": name, "op": "attn", "B": B, "H": H, "Hkv": Hkv, "D": D, "L": L, "page": page, "dtype": dtype,
            "gated": gated, "mass": mass, "store": store, "ragged": ragged, "layout": layout}


def _append(name, B, T, Hkv, D, L, page, dtype, ragged, layout="slots"):
    return {"name": name, "op": "append", "B": B, "T": T, "Hkv": Hkv, "D": D, "L": L, "page": page, "dtype": dtype,
            "ragged": ragged, "layout": layout}


def _evict(name, B, Hkv, D, L, keep, recent, page, dtype, ragged, layout="slots"):
    return {"name": name, "op": "evict", "B": B, "Hkv": Hkv, "D": D, "L": L, "keep": keep, "recent": recent, "page": page,
            "dtype": dtype, "ragged": ragged, "layout": layout}


def _sample(name, B, V, dtype, temperature, top_k=0, top_p=1.0, min_p=0.0, per_row=False, spread=3.0):
    """per_row: the choices are tensors, one of each request."""
    return {"name": name, "op": "sample", "B": B, "V": V, "dtype": dtype, "temperature": temperature, "top_k": top_k,
            "top_p": top_p, "min_p": min_p, "per_row": per_row, "spread": spread}


def listed():
    return [
        # a few users of the drop-in decoder (8 heads of 64, gate and temperatures), fp32 as its modules run
        _attn("attn_decode_few", 4, 8, 8, 64, 512, 16, "f32", True, False),
        # a batch of it at its full context in bf16, weights collected for eviction
        _attn("attn_decode_mass", 32, 8, 8, 64, 2048, 16, "bf16", True, True),
        # grouped query heads without a gate: a large serving batch
        _attn("attn_grouped_batch", 48, 32, 8, 128, 8192, 16, "bf16", False, False),
        # one long document
        _attn("attn_grouped_long", 1, 32, 8, 128, 131072, 64, "bf16", False, True, ragged=False),
        # odd group, channels and pages, heads apart in a page
        _attn("attn_odd", 5, 12, 4, 80, 3001, 24, "f32", False, True, layout="heads"),
        # a prompt of every sequence, padded
        _append("append_prompt", 8, 2048, 8, 128, 4096, 16, "bf16", True),
        # one token of every sequence
        _append("append_step", 64, 1, 8, 64, 512, 16, "f32", False),
        # a batch over its budget
        _evict("evict_batch", 32, 8, 64, 1280, 1024, 256, 16, "bf16", True),
        # long caches brought to a quarter
        _evict("evict_long", 2, 8, 128, 32768, 8192, 1024, 64, "bf16", False),
        # a byte vocabulary without filters
        _sample("sample_bytes", 16, 256, "f32", 0.8),
        # a subword vocabulary: the nucleus and a floor relative to the best
        _sample("sample_nucleus", 32, 49999, "f32", 0.9, top_p=0.95, min_p=0.02),
        # a large vocabulary, every request with its own choices
        _sample("sample_requests", 64, 131072, "bf16", 0.7, top_k=50, top_p=0.9, per_row=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _one(rng):
    dtype, op = rng.choice(["f32", "bf16"]), rng.choice(["attn", "attn", "attn", "append", "evict", "evict", "sample", "sample"])
    D = rng.choice([64, 64, 128, 128, 8 * rng.randint(2, 32)])
    page, layout = rng.choice([16, 16, 32, 64, rng.randint(5, 100)]), rng.choice(["slots", "slots", "heads"])
    Hkv, B = rng.choice([1, 2, 4, 8, 8, 12, 16]), _log(rng, 1, 128)
    if op == "attn":
        G = rng.choice([1, 1, 2, 3, 4, 4, 5, 8, 16])
        return _attn("", B, Hkv * G, Hkv, D, _log(rng, 1, 65536), page, dtype, rng.random() < 0.4, rng.random() < 0.4,
                     store=rng.random() < 0.7, ragged=rng.random() < 0.7, layout=layout)
    if op == "append":
        T = _log(rng, 1, 4096)
        return _append("", B, T, Hkv, D, T + rng.randint(0, 1024), page, dtype, rng.random() < 0.5, layout)
    if op == "evict":
        L = _log(rng, 32, 65536)
        keep = max(1, int(L * rng.uniform(0.1, 0.9)))
        return _evict("", B, Hkv, D, L, keep, int(keep * rng.uniform(0.0, 0.5)), page, dtype, rng.random() < 0.5, layout)
    return _sample("", _log(rng, 1, 256), _log(rng, 100, 200000), dtype, rng.uniform(0.3, 1.5), rng.choice([0, 0, 1, 20, 50, 400]),
                   rng.choice([1.0, 0.5, 0.9, 0.95]), rng.choice([0.0, 0.0, 0.05]), rng.random() < 0.5, rng.choice([1.0, 3.0, 3.0]))


def _fits(c):
    if work(c)["bytes"] > _MOST_BYTES:
        return False
    if c["op"] == "attn":
        return c["B"] * c["H"] * c["L"] * (c["D"] if c["gated"] else 4) <= _MOST_SUMS
    if c["op"] == "evict":
        return c["B"] * c["Hkv"] * c["L"] * c["D"] <= _MOST_SUMS
    return c["op"] != "sample" or c["B"] * c["V"] <= 64 * 131072


def draw(rng):
    c = _one(rng)
    while not _fits(c):
        c = _one(rng)
    return {k: v for k, v in c.items() if k != "name"}


# ----------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=_DEV).manual_seed(int(seed) * 2654435761 % (1 << 62) + 29)


def _slots(case):
    """Slots of a sequence: its pages are full ones."""
    return -(-case["L"] // case["page"]) * case["page"]


def _lengths(case, g):
    B, L = case["B"], case["L"]
    n = torch.randint(max(1, L // 2), L + 1, (B,), device=_DEV, generator=g, dtype=torch.int32) if case["ragged"] else \
        torch.full((B,), L, device=_DEV, dtype=torch.int32)
    n[0] = L
    return n


def prepare(case, seed):
    g, dt, op, B = _gen(seed), _dtype(case), case["op"], case["B"]

    def randn(*shape, std=1.0, mean=0.0, dtype=dt):
        return torch.empty(shape, device=_DEV, dtype=torch.float32).normal_(mean, std, generator=g).to(dtype)

    s = {"case": dict(case)}
    if op == "sample":
        s["logits"] = randn(B, case["V"], std=case["spread"])
        s["uniform"] = torch.rand(B, device=_DEV, generator=g)
        for k in ("temperature", "top_p", "min_p", "top_k"):
            s[k] = case[k]
            if case["per_row"]:
                vary = torch.rand(B, device=_DEV, generator=g)
                if k == "top_k":
                    s[k] = (case[k] * (0.5 + vary)).int()
                elif k == "top_p":
                    s[k] = case[k] * (1.0 - 0.1 * vary) if case[k] < 1.0 else torch.ones(B, device=_DEV)
                else:
                    s[k] = case[k] * (0.75 + 0.5 * vary)
        return s
    Hkv, D, page = case["Hkv"], case["D"], case["page"]
    per = _slots(case) // page
    pages = B * per + 3                                    # pages in use lie anywhere among them
    s["table"] = torch.randperm(pages, device=_DEV, generator=g)[:B * per].view(B, per).int()
    shape = (pages, page, Hkv, D) if case["layout"] == "slots" else (pages, Hkv, page, D)
    s["k"], s["v"] = randn(*shape), randn(*shape)
    if case["layout"] == "heads":
        s["k"], s["v"] = s["k"].transpose(1, 2), s["v"].transpose(1, 2)
    if op == "append":
        T = case["T"]
        s["key"], s["value"] = randn(B, T, Hkv, D), randn(B, T, Hkv, D)
        s["starts"] = torch.randint(0, case["L"] - T + 1, (B,), device=_DEV, generator=g, dtype=torch.int32)
        s["counts"] = None
        if case["ragged"]:
            s["counts"] = torch.randint(max(1, T // 2), T + 1, (B,), device=_DEV, generator=g, dtype=torch.int32)
        return s
    s["lengths"] = _lengths(case, g)
    if op == "evict":
        # weights that fall off over several orders of magnitude, as accumulated attention does
        s["mass"] = torch.exp(randn(B, Hkv, _slots(case), std=2.0, mean=-3.0, dtype=torch.float32))
        s["out"] = torch.zeros_like(s["mass"])
        return s
    H = case["H"]
    s["q"] = randn(B, H, D, std=1.5)
    s["scale"] = D ** -0.5
    s["key"] = s["value"] = s["gate"] = s["tau"] = s["mass"] = None
    if case["store"]:
        s["key"], s["value"] = randn(B, Hkv, D), randn(B, Hkv, D)
    if case["gated"]:
        s["gate"] = torch.sigmoid(randn(B, H, mean=-1.0, dtype=torch.float32))
        s["tau"] = torch.exp(randn(H, std=0.3, dtype=torch.float32))
    if case["mass"]:
        s["mass"] = torch.rand(B, Hkv, _slots(case), device=_DEV, generator=g)
    return s


# ----------------------------------------------------------------------------- one pass
def run(s):
    op = s["case"]["op"]
    with torch.no_grad():
        if own:
            return {"attn": _own_attn, "append": _own_append, "evict": _own_evict, "sample": _own_sample}[op](s)
        return {"attn": _plain_attn, "append": _plain_append, "evict": _plain_evict, "sample": _plain_sample}[op](s)


def _attn_outputs(s, o):
    r = {"o": o}
    if s["key"] is not None:
        r["k"], r["v"] = s["k"], s["v"]
    if s["mass"] is not None:
        r["mass"] = s["mass"]
    return r


def _own_attn(s):
    from mk_iii_technologies_tsrn_b200 import ops
    return _attn_outputs(s, ops.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], key=s["key"], value=s["value"],
                                                scale=s["scale"], gate=s["gate"], tau=s["tau"], mass=s["mass"]))


def _own_append(s):
    from mk_iii_technologies_tsrn_b200 import ops
    ops.paged_append(s["key"], s["value"], s["k"], s["v"], s["table"], s["starts"], s["counts"])
    return {"k": s["k"], "v": s["v"]}


def _own_evict(s):
    from mk_iii_technologies_tsrn_b200 import ops
    c = s["case"]
    kept = ops.cache_evict(s["k"], s["v"], s["table"], s["lengths"], s["mass"], c["keep"], c["recent"], out=s["out"])
    return {"kept": kept, "k": s["k"], "v": s["v"], "mass": s["out"]}


def _own_sample(s):
    from mk_iii_technologies_tsrn_b200 import ops
    token, logprob = ops.sample_tokens(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"],
                                       top_p=s["top_p"], min_p=s["min_p"], return_logprob=True)
    return {"token": token, "logprob": logprob}


# ----------------------------------------------------------------------------- plain forms
def _place(table, page, slot, b=None):
    """(page, slot in it) of slots [B, n] of their sequences."""
    b = torch.arange(table.shape[0], device=_DEV)[:, None] if b is None else b
    return table[b, slot // page].long(), slot % page


def _plain_attn(s):
    c, table, n = s["case"], s["table"], s["lengths"].long()
    B, H, Hkv, D, page = (c[k] for k in ("B", "H", "Hkv", "D", "page"))
    if s["key"] is not None:
        p, r = _place(table, page, n[:, None] - 1)
        s["k"][p[:, 0], r[:, 0]] = s["key"]
        s["v"][p[:, 0], r[:, 0]] = s["value"]
    S = table.shape[1] * page
    k = s["k"][table.long()].reshape(B, S, Hkv, D).transpose(1, 2).float()     # [B, Hkv, S, D]
    v = s["v"][table.long()].reshape(B, S, Hkv, D).transpose(1, 2).float()
    q = s["q"].float().view(B, Hkv, H // Hkv, D)
    score = q @ k.transpose(2, 3)
    if s["gate"] is not None:
        gate = s["gate"].view(B, Hkv, H // Hkv, 1)
        trop = (q[:, :, :, None] + k[:, :, None]).amax(-1)
        score = gate * trop + (1.0 - gate) * score
    score = score * s["scale"]
    if s["tau"] is not None:
        score = score / s["tau"].view(1, Hkv, H // Hkv, 1)
    live = (torch.arange(S, device=_DEV)[None] < n[:, None])[:, None, None]
    score = torch.where(live, score, float("-inf"))
    w = torch.exp(score - score.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    o = (w @ v).reshape(B, H, D).to(_dtype(c))
    if s["mass"] is not None:
        total = w.sum(2)                                                       # [B, Hkv, S]
        old = s["mass"]
        if s["key"] is not None:                                               # the new slot begins
            old = torch.where(torch.arange(S, device=_DEV)[None] == n[:, None] - 1, 0.0, old.transpose(0, 1)).transpose(0, 1)
        s["mass"].copy_(old + total)
    return _attn_outputs(s, o)


def _plain_append(s):
    c = s["case"]
    T = c["T"]
    at = torch.arange(T, device=_DEV)[None]
    live = at < (s["counts"][:, None] if s["counts"] is not None else T)
    b, t = torch.nonzero(live.expand(c["B"], T), as_tuple=True)
    p, r = _place(s["table"], c["page"], (s["starts"].long()[:, None] + at)[b, t], b)
    s["k"][p, r] = s["key"][b, t]
    s["v"][p, r] = s["value"][b, t]
    return {"k": s["k"], "v": s["v"]}


def _plain_evict(s):
    c, n = s["case"], s["lengths"].long()[:, None, None]
    B, Hkv, keep = c["B"], c["Hkv"], c["keep"]
    S = s["mass"].shape[2]
    at = torch.arange(S, device=_DEV)
    order = torch.where(at >= n - c["recent"], float("inf"), s["mass"])
    order = torch.where(at < n, order, float("-inf"))
    kept = torch.sort(order, dim=-1, descending=True, stable=True)[1][..., :keep]
    kept = torch.sort(torch.where(kept < n, kept, S), dim=-1)[0]               # what is not there comes last
    b, h, i = torch.nonzero(kept < S, as_tuple=True)
    src = kept[b, h, i]
    p, r = _place(s["table"], c["page"], src, b)
    q, t = _place(s["table"], c["page"], i, b)
    k, v = s["k"][p, r, h], s["v"][p, r, h]
    s["k"][q, t, h] = k
    s["v"][q, t, h] = v
    s["out"][b, h, i] = s["mass"][b, h, src]
    return {"kept": torch.where(kept < S, kept, -1).int(), "k": s["k"], "v": s["v"], "mass": s["out"]}


def _column(x, like):
    """A number, or one of each row, as a column in 64 bits."""
    x = x.double() if torch.is_tensor(x) else torch.tensor(x, device=_DEV, dtype=torch.float64)
    return x.expand(like.shape[0])[:, None]


def _plain_sample(s):
    # in 64 bits: a rounded sum next to the random number's place would be another token
    x = s["logits"].double()
    V = x.shape[1]
    top_k, top_p, min_p = (_column(s[k], x) for k in ("top_k", "top_p", "min_p"))
    xs, order = torch.sort(x, dim=-1, descending=True, stable=True)
    w = torch.exp((xs - xs[:, :1]) / _column(s["temperature"], x))
    rank = torch.arange(V, device=_DEV)[None]
    keep = (top_k <= 0) | (rank < top_k)
    sums = torch.cumsum(torch.where(keep, w, 0.0), -1)
    keep &= (top_p >= 1.0) | (sums - w < top_p * sums[:, -1:])
    keep &= w >= min_p
    keep |= rank == 0
    w = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))
    sums = torch.cumsum(w, -1)
    token = (sums <= s["uniform"].double()[:, None] * sums[:, -1:]).sum(-1)
    token = torch.minimum(token, torch.where(w > 0, rank, -1).amax(-1))
    logprob = torch.log(w.gather(1, token[:, None]) / sums[:, -1:])[:, 0]
    return {"token": token, "logprob": logprob.float()}


# ----------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"attn": _exact_attn, "append": _exact_append, "evict": _exact_evict, "sample": _exact_sample}[case["op"]](s)


def _rows(cache, table, b, n):
    """Slots 0 .. n - 1 of sequence b, one page after another: [n, heads, channels]."""
    return cache[table[b, :-(-n // cache.shape[1])].long()].flatten(0, 1)[:n]


def _exact_attn(s):
    c = s["case"]
    H, Hkv, page = c["H"], c["Hkv"], c["page"]
    G = H // Hkv
    out = torch.zeros(c["B"], H, c["D"], device=_DEV, dtype=torch.float64)
    mass = s["mass"].double() if s["mass"] is not None else None
    for b, n in enumerate(s["lengths"].tolist()):
        if s["key"] is not None:
            at = int(s["table"][b, (n - 1) // page])
            s["k"][at, (n - 1) % page] = s["key"][b]
            s["v"][at, (n - 1) % page] = s["value"][b]
            if mass is not None:
                mass[b, :, n - 1] = 0.0
        k, v = _rows(s["k"], s["table"], b, n), _rows(s["v"], s["table"], b, n)
        for h in range(H):
            kh, vh, q = k[:, h // G].double(), v[:, h // G].double(), s["q"][b, h].double()
            score = (kh * q).sum(1)
            if s["gate"] is not None:
                g = s["gate"][b, h].double()
                score = score + g * ((kh + q).max(1).values - score)
            score = score * s["scale"]
            if s["tau"] is not None:
                score = score / s["tau"][h].double()
            w = torch.exp(score - torch.logsumexp(score, 0))
            out[b, h] = (w[:, None] * vh).sum(0)
            if mass is not None:
                mass[b, h // G, :n] += w
    r = {"o": out}
    if s["key"] is not None:
        r["k"], r["v"] = s["k"].double(), s["v"].double()
    if mass is not None:
        r["mass"] = mass
    return r


def _exact_append(s):
    c, page = s["case"], s["case"]["page"]
    table, starts = s["table"].tolist(), s["starts"].tolist()
    counts = s["counts"].tolist() if s["counts"] is not None else [c["T"]] * c["B"]
    for b in range(c["B"]):
        t = 0
        while t < counts[b]:                               # from page to page
            slot = starts[b] + t
            m = min(counts[b] - t, page - slot % page)
            for cache, new in ((s["k"], s["key"]), (s["v"], s["value"])):
                cache[table[b][slot // page], slot % page:slot % page + m] = new[b, t:t + m]
            t += m
    return {"k": s["k"].double(), "v": s["v"].double()}


def _exact_evict(s):
    c, page, keep = s["case"], s["case"]["page"], s["case"]["keep"]
    kept = np.full((c["B"], c["Hkv"], keep), -1, dtype=np.int32)
    mass, out = s["mass"].cpu().numpy(), s["out"].double()
    for b, n in enumerate(s["lengths"].tolist()):
        k, v = _rows(s["k"], s["table"], b, n), _rows(s["v"], s["table"], b, n)
        old = max(0, n - c["recent"])
        for h in range(c["Hkv"]):
            if n <= keep:
                take = np.arange(n)
            else:                                          # the heaviest of the old ones, the earlier of equals
                best = np.lexsort((np.arange(old), -mass[b, h, :old]))[:keep - (n - old)]
                take = np.concatenate((np.sort(best), np.arange(old, n)))
            kept[b, h, :len(take)] = take
            src = torch.as_tensor(take, device=_DEV)
            out[b, h, :len(take)] = s["mass"][b, h, src].double()
            slot = torch.arange(len(take), device=_DEV)
            where = s["table"][b].long()[slot // page], slot % page, h
            s["k"].index_put_(tuple(torch.as_tensor(i, device=_DEV) for i in where), k[src, h])
            s["v"].index_put_(tuple(torch.as_tensor(i, device=_DEV) for i in where), v[src, h])
    return {"kept": torch.as_tensor(kept, device=_DEV), "k": s["k"].double(), "v": s["v"].double(), "mass": out}


def _exact_sample(s):
    c = s["case"]
    x, u = s["logits"].double().cpu().numpy(), s["uniform"].double().cpu().numpy()
    pick = {k: np.broadcast_to(s[k].double().cpu().numpy() if torch.is_tensor(s[k]) else np.float64(s[k]), (c["B"],))
            for k in ("temperature", "top_k", "top_p", "min_p")}
    out, logprob = np.zeros(c["B"], dtype=np.int64), np.zeros(c["B"])
    for b in range(c["B"]):
        order = np.argsort(-x[b], kind="stable")
        w = np.exp((x[b][order] - x[b][order[0]]) / pick["temperature"][b])
        m = len(w) if pick["top_k"][b] <= 0 else min(len(w), int(pick["top_k"][b]))
        if pick["top_p"][b] < 1.0:                         # as many as reach the share
            m = min(m, 1 + int(np.searchsorted(np.cumsum(w[:m]), pick["top_p"][b] * math.fsum(w[:m]))))
        m = max(1, min(m, int((w >= pick["min_p"][b]).sum())))
        kept = np.sort(order[:m])
        p = np.exp((x[b][kept] - x[b].max()) / pick["temperature"][b])
        sums = np.cumsum(p)
        i = min(m - 1, int(np.searchsorted(sums, u[b] * sums[-1], side="right")))
        out[b] = kept[i]
        logprob[b] = (x[b][kept[i]] - x[b].max()) / pick["temperature"][b] - math.log(math.fsum(p))
    return {"token": torch.as_tensor(out, device=_DEV), "logprob": torch.as_tensor(logprob, device=_DEV)}


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    e, op, B = _esize(case), case["op"], case["B"]
    if op == "sample":
        n = B * float(case["V"])
        return {"bytes": e * n + 16.0 * B, "flops": 4.0 * n}
    Hkv, D, L = case["Hkv"], case["D"], case["L"]
    if op == "append":
        n = B * float(case["T"]) * (0.75 if case["ragged"] else 1.0)
        return {"bytes": 4.0 * e * n * Hkv * D, "flops": 0.0}
    n = L + (B - 1) * L * (0.75 if case["ragged"] else 1.0)      # slots in use
    if op == "evict":
        m = min(n, float(B * case["keep"]))
        return {"bytes": Hkv * (m * (4.0 * e * D + 8.0) + 4.0 * n), "flops": 4.0 * n * Hkv}
    b = 2.0 * e * n * Hkv * D + 2.0 * e * B * case["H"] * D + 4.0 * n / case["page"]
    if case["store"]:
        b += 2.0 * e * B * Hkv * D
    if case["mass"]:
        b += 8.0 * n * Hkv
    return {"bytes": b, "flops": n * case["H"] * D * (6.0 if case["gated"] else 4.0)}
