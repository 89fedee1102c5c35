"""Cases of the paged-attention operators: rotary positions, appending to a paged key/value
cache, and attention of a batch that shares a long prefix.

`run` makes one pass through one operator, either in its plain form (elementary torch
operations in 32 bits, rounded once at the end) or, where the module's `own` is true, through
the calls of tilegen_b200.paged.  A sequence's pages are a row of a CSR table
(page_indptr, page_indices); the pages are drawn without order from the cache.
"""

import math

import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}


# ------------------------------------------------------------------------------ the cases
def _rope(name, tokens, heads, dim, rot, layout, dtype, backward=False, factor=1.0, span=4096):
    """tokens x heads rows of dim, of which the first rot rotate; positions below span."""
    return {"op": "rope", "name": name, "tokens": tokens, "heads": heads, "dim": dim, "rot": rot, "layout": layout,
            "dtype": dtype, "backward": backward, "factor": factor, "span": span}


def _append(name, batch, n_lo, n_hi, len_hi, heads, kv_heads, dim, rot, layout, page, dtype, base=0):
    """n_lo..n_hi new tokens for each of batch sequences, up to len_hi long after them."""
    return {"op": "append", "name": name, "batch": batch, "n_lo": n_lo, "n_hi": n_hi, "len_hi": len_hi, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "rot": rot, "layout": layout, "page": page, "dtype": dtype, "base": base}


def _attend(name, batch, n_lo, n_hi, own_lo, own_hi, prefix, heads, kv_heads, dim, page, dtype):
    """n_lo..n_hi query tokens for each of batch sequences whose own parts are own_lo..own_hi
    long (the query tokens among them), behind a shared prefix."""
    return {"op": "attend", "name": name, "batch": batch, "n_lo": n_lo, "n_hi": n_hi, "own_lo": own_lo, "own_hi": own_hi,
            "prefix": prefix, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype}


def listed():
    return [
        # the queries of one decoding step of a small batch, deep in a long, scaled context
        _rope("rope_decode", 5, 32, 128, 128, "half", "bf16", factor=8.0, span=120000),
        # queries of a training step: an odd number of packed tokens, neighbours rotate
        _rope("rope_train", 16383, 32, 128, 128, "interleaved", "bf16"),
        # the gradient of half-rotated heads in 32 bits
        _rope("rope_grad", 8192, 24, 96, 48, "half", "f32", backward=True),
        # one new token for each of a few sequences: all latency
        _append("append_decode", 6, 1, 1, 900, 32, 8, 128, 128, "half", 16, "bf16", base=700),
        # one new token for each sequence of a full server, neighbours rotate
        _append("append_batch", 512, 1, 1, 700, 32, 8, 128, 64, "interleaved", 32, "f16"),
        # whole prompts of many lengths are written
        _append("append_prompts", 24, 40, 1900, 1900, 32, 8, 128, 128, "half", 16, "bf16"),
        # the smallest serving step: few sequences, a short prefix
        _attend("attend_small", 4, 1, 1, 9, 90, 700, 16, 4, 64, 16, "bf16"),
        # two sequences far into one long document: a long axis and few rows
        _attend("attend_long", 2, 1, 1, 300, 1500, 131071, 32, 8, 128, 64, "f16"),
        # a serving batch: as many bytes in the sequences' own pages as in the prefix and more
        _attend("attend_batch", 64, 1, 1, 64, 1021, 8192, 32, 8, 128, 16, "bf16"),
        # a large batch on a long system prompt: the prefix is a matrix product
        _attend("attend_wide", 256, 1, 1, 100, 260, 32768, 32, 8, 128, 16, "bf16"),
        # a few tokens for each sequence, as drafts are checked, heads of 64
        _attend("attend_drafts", 48, 2, 7, 40, 600, 5003, 32, 4, 64, 32, "f16"),
        # questions of many tokens on one document: the compute-bound end
        _attend("attend_questions", 24, 60, 250, 60, 400, 16384, 32, 8, 128, 16, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "append", "attend", "attend"])
    dtype = rng.choice(["bf16", "f16"])
    layout = rng.choice(["half", "interleaved"])
    if op == "rope":
        dim = rng.choice([64, 80, 96, 128, 256])
        heads = rng.choice([1, 5, 8, 16, 24, 32])
        dtype = rng.choice(["bf16", "f16", "f32"])
        tokens = min(_log(rng, 1, 16384), 16383 * 32 * 128 * 2 // (heads * dim * _SIZE[dtype]))
        c = _rope("", tokens, heads, dim, rng.choice([dim, dim // 2]), layout, dtype, rng.random() < 0.5,
                  rng.choice([1.0, 4.0, 8.0]), _log(rng, 2048, 131072))
    elif op == "append":
        dim = rng.choice([64, 96, 128])
        kv_heads = rng.choice([1, 4, 8])
        heads = kv_heads * rng.choice([1, 4, 5, 8])
        batch = _log(rng, 1, 512)
        n_hi = rng.choice([1, 1, 3, max(1, min(1900, 24000 // batch))])
        c = _append("", batch, max(1, n_hi // 40), n_hi, n_hi + rng.randrange(700), heads, kv_heads, dim,
                    rng.choice([dim, dim // 2]), layout, rng.choice([8, 16, 24, 32, 64]), dtype, rng.choice([0, 700, 8191]))
    else:
        dim = rng.choice([64, 128])
        kv_heads = rng.choice([2, 4, 8])
        heads = kv_heads * rng.choice([1, 4, 5, 8])
        batch = _log(rng, 1, 256)
        n_hi = rng.choice([1, 1, 6, max(1, min(250, 3000 // batch))])
        own_hi = n_hi + _log(rng, 16, 1000)
        top = 3000 * 32 * 16384 // (batch * n_hi * heads)
        c = _attend("", batch, max(1, n_hi // 4), n_hi, max(n_hi, own_hi // 8), own_hi, _log(rng, 200, max(400, min(131072, top))),
                    heads, kv_heads, dim, rng.choice([8, 16, 24, 32, 64]), dtype)
    del c["name"]
    return c


def _spread(lo, hi, n):
    """n whole numbers from hi down to lo."""
    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _shape(case):
    """(new tokens, own lengths) of a ragged case's sequences."""
    n = _spread(case["n_lo"], case["n_hi"], case["batch"])
    if case["op"] == "append":
        lens = [x + (case["len_hi"] - x) * i // max(1, case["batch"]) for i, x in enumerate(n)]
    else:
        lens = [max(a, b) for a, b in zip(n, reversed(_spread(case["own_lo"], case["own_hi"], case["batch"])))]
    return n, lens


def work(case):
    size = _SIZE[case["dtype"]]
    if case["op"] == "rope":
        cells = case["tokens"] * case["heads"]
        return {"bytes": 2 * cells * case["dim"] * size + 8 * case["tokens"], "flops": 3 * cells * case["rot"]}
    n, lens = _shape(case)
    tokens = sum(n)
    if case["op"] == "append":
        cells = case["heads"] + 2 * case["kv_heads"]
        return {"bytes": 2 * tokens * cells * case["dim"] * size + 8 * len(n),
                "flops": 3 * tokens * (case["heads"] + case["kv_heads"]) * case["rot"]}
    keys = case["prefix"] + sum(lens)
    seen = sum(a * (case["prefix"] + l) - a * (a - 1) // 2 for a, l in zip(n, lens))
    return {"bytes": 2 * keys * case["kv_heads"] * case["dim"] * size + 2 * tokens * case["heads"] * case["dim"] * size,
            "flops": 4 * seen * case["heads"] * case["dim"]}


# ------------------------------------------------------------------------------ the inputs
def _frequencies(rot, factor, device, base=500000.0, original=8192):
    """Angle per position of each rotating pair, in 64 bits.  For a context `factor` times the
    original one, pairs of long wavelength turn `factor` times slower, short ones as before, and
    those between are blended."""
    f = base ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    turns = f * original / (2 * math.pi)
    keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
    return f * (keep + (1 - keep) / factor)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = _DTYPE[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32).to(dt)

    s = dict(case)
    if case["op"] == "rope":
        s["x"] = normal(case["tokens"], case["heads"], case["dim"])
        if case["tokens"] > 1000:  # packed sequences
            s["positions"] = torch.arange(case["tokens"], device=dev) % case["span"]
        else:
            s["positions"] = torch.randint(0, case["span"], (case["tokens"],), generator=g, device=dev)
        s["freq"] = _frequencies(case["rot"], case["factor"], dev)
        s["scale"] = 0.1 * math.log(case["factor"]) + 1.0
        return s
    n, lens = _shape(case)
    batch, page, tokens = case["batch"], case["page"], sum(n)
    pages = [-(-x // page) for x in lens]
    prefix_pages = -(-case.get("prefix", 0) // page)
    order = torch.randperm(sum(pages) + prefix_pages, generator=g, device=dev)
    s["prefix_pages"], s["page_indices"] = order[:prefix_pages].contiguous(), order[prefix_pages:].contiguous()

    def starts(v):
        return torch.tensor([0] + v, device=dev, dtype=torch.int64).cumsum(0)

    s["page_indptr"], s["q_indptr"] = starts(pages), starts(n)
    s["seq_len"] = torch.tensor(lens, device=dev, dtype=torch.int64)
    s["max_pages"], s["max_len"], s["max_q"], s["tokens"] = max(pages), max(lens), max(n), tokens
    s["ragged"] = case["n_hi"] > 1
    s["q"] = normal(tokens, case["heads"], case["dim"])
    s["k_cache"] = normal(order.numel(), page, case["kv_heads"], case["dim"])
    s["v_cache"] = normal(order.numel(), page, case["kv_heads"], case["dim"])
    if case["op"] == "append":
        s["k"], s["v"] = normal(tokens, case["kv_heads"], case["dim"]), normal(tokens, case["kv_heads"], case["dim"])
        s["freq"], s["scale"] = _frequencies(case["rot"], 1.0, dev), 1.0
    return s


# ------------------------------------------------------------------------------ plain forms
def _rotate(x, positions, freq, scale, layout, sign=1.0):
    """x [tokens, heads, dim] in 32 bits.  The angle is taken in 64 bits: at position 1e5 a
    32-bit angle has lost three digits."""
    angle = positions.double()[:, None] * freq
    c = (angle.cos() * scale).float()[:, None]
    d = (angle.sin() * (sign * scale)).float()[:, None]
    rot = 2 * freq.numel()
    r, rest = x[..., :rot], x[..., rot:]
    if layout == "half":
        a, b = r[..., : rot // 2], r[..., rot // 2 :]
        y = torch.cat((a * c - b * d, b * c + a * d), -1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        y = torch.stack((a * c - b * d, b * c + a * d), -1).flatten(-2)
    return torch.cat((y, rest), -1)


def _owners(s):
    """(sequence, place among its new tokens, place in its own part) of each new token."""
    t = torch.arange(s["tokens"], device=s["q"].device)
    b = torch.searchsorted(s["q_indptr"], t, right=True) - 1
    i = t - s["q_indptr"][b]
    return b, i, s["seq_len"][b] - (s["q_indptr"][b + 1] - s["q_indptr"][b]) + i


def _plain_append(s):
    b, _, at = _owners(s)
    k = _rotate(s["k"].float(), at + s["base"], s["freq"], s["scale"], s["layout"]).to(s["k"].dtype)
    q = _rotate(s["q"].float(), at + s["base"], s["freq"], s["scale"], s["layout"]).to(s["q"].dtype)
    page = s["page_indices"][s["page_indptr"][b] + at // s["page"]]
    s["k_cache"][page, at % s["page"]] = k
    s["v_cache"][page, at % s["page"]] = s["v"]
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attend(s):
    kvh, dim, page, tokens = s["kv_heads"], s["dim"], s["page"], s["tokens"]
    group, batch, width, long = s["heads"] // kvh, s["batch"], s["max_q"], s["max_len"]
    q = s["q"].float() * dim ** -0.5
    b, i, at = _owners(s)

    # the prefix: one product for all rows, [kv head, token x group, key]
    def prefix(cache):
        return cache[s["prefix_pages"]].flatten(0, 1)[: s["prefix"]].float().transpose(0, 1)

    rows = q.view(tokens, kvh, group, dim).transpose(0, 1).reshape(kvh, tokens * group, dim)
    sp = rows @ prefix(s["k_cache"]).transpose(1, 2)
    mp = sp.amax(-1)
    sp = sp.sub_(mp[..., None]).exp_()
    lp = sp.sum(-1)
    ap = sp @ prefix(s["v_cache"])

    # the own parts: padded to the longest
    j = torch.arange(long, device=q.device)
    at_page = (s["page_indptr"][:-1, None] + j // page).clamp(max=s["page_indices"].numel() - 1)
    held = (j < s["seq_len"][:, None])[..., None, None]

    def owned(cache):
        x = cache[s["page_indices"][at_page], j % page].float()
        return torch.where(held, x, 0.0).transpose(1, 2)  # [sequence, kv head, key, dim]

    wide = q.new_zeros(batch, width, s["heads"], dim)
    wide[b, i] = q
    wide = wide.view(batch, width, kvh, group, dim).permute(0, 2, 1, 3, 4).reshape(batch, kvh, width * group, dim)
    so = (wide @ owned(s["k_cache"]).transpose(2, 3)).view(batch, kvh, width, group, long)
    n = s["q_indptr"].diff()
    last = s["seq_len"][:, None] - n[:, None] + torch.arange(width, device=q.device)
    so = torch.where((j <= last[..., None])[:, None, :, None], so, -math.inf)
    mo = so.amax(-1)
    so = so.sub_(mo.clamp(min=-1e30)[..., None]).exp_()
    lo = so.sum(-1)
    ao = (so.view(batch, kvh, width * group, long) @ owned(s["v_cache"])).view(batch, kvh, width, group, dim)

    # joined by the larger maximum, [token, kv head, group]
    mp, lp = (x.view(kvh, tokens, group).transpose(0, 1) for x in (mp, lp))
    ap = ap.view(kvh, tokens, group, dim).transpose(0, 1)
    mo, lo, ao = (x.transpose(1, 2)[b, i] for x in (mo, lo, ao))
    m = torch.maximum(mp, mo)
    wp, wo = (mp - m).exp(), (mo - m).exp()
    out = (ap * wp[..., None] + ao * wo[..., None]) / (lp * wp + lo * wo)[..., None]
    return out.reshape(tokens, s["heads"], dim).to(s["q"].dtype)


# ------------------------------------------------------------------------------ one pass
def _own_run(s):
    from tilegen_b200 import paged

    if s["op"] != "attend":
        rope = paged.Rope(s["freq"], s["layout"], s["scale"])
    if s["op"] == "rope":
        return (paged.rope_backward if s["backward"] else paged.rope)(s["x"], rope, s["positions"])
    cache = paged.PagedKV(s["k_cache"], s["v_cache"])
    table = paged.PageTable(s["page_indptr"], s["page_indices"])
    ragged = {"q_indptr": s["q_indptr"], "max_q_len": s["max_q"]} if s["ragged"] else {}
    if s["op"] == "append":
        q = paged.kv_append(cache, table, s["seq_len"], s["k"], s["v"], rope=rope, q=s["q"], position_base=s["base"],
                            q_indptr=ragged.get("q_indptr"))
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    return paged.prefix_attention(s["q"], cache, table, s["seq_len"], prefix_pages=s["prefix_pages"],
                                  prefix_len=s["prefix"], max_seq_len=s["max_len"], **ragged)


def run(state):
    if own:
        return _own_run(state)
    if state["op"] == "rope":
        return _rotate(state["x"].float(), state["positions"], state["freq"], state["scale"], state["layout"],
                       -1.0 if state["backward"] else 1.0).to(state["x"].dtype)
    return _plain_append(state) if state["op"] == "append" else _plain_attend(state)


# ------------------------------------------------------------------------------ in 64 bits
def _turned(x, positions, freq, scale, layout, back=False):
    """Each pair as a complex number times scale * exp(+-i angle)."""
    rot = 2 * freq.numel()
    y = x.double().clone()
    turn = torch.polar(torch.full_like(freq, scale).expand(positions.numel(), -1),
                       positions.double()[:, None] * (-freq if back else freq))[:, None]
    first, second = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    z = torch.complex(y[..., first].clone(), y[..., second].clone()) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _turned(s["x"], s["positions"], s["freq"], s["scale"], case["layout"], case["backward"])
    n, lens = _shape(case)
    ip, ix, page = s["page_indptr"].tolist(), s["page_indices"], case["page"]
    if case["op"] == "append":
        kc, vc, out, t = s["k_cache"].double(), s["v_cache"].double(), [], 0
        for b in range(case["batch"]):
            at = torch.arange(lens[b] - n[b], lens[b], device=kc.device)
            place = (ix[ip[b]:ip[b + 1]][at // page], at % page)
            out.append(_turned(s["q"][t:t + n[b]], at + case["base"], s["freq"], s["scale"], case["layout"]))
            kc[place] = _turned(s["k"][t:t + n[b]], at + case["base"], s["freq"], s["scale"], case["layout"])
            vc[place] = s["v"][t:t + n[b]].double()
            t += n[b]
        return {"q": torch.cat(out), "k_cache": kc, "v_cache": vc}
    if work(case)["flops"] > 2e13:
        return None
    heads, kvh, dim = case["heads"], case["kv_heads"], case["dim"]
    shared = [c[s["prefix_pages"]].flatten(0, 1)[: case["prefix"]].double() for c in (s["k_cache"], s["v_cache"])]
    out, t = [], 0
    for b in range(case["batch"]):
        k, v = (torch.cat((p, c[ix[ip[b]:ip[b + 1]]].flatten(0, 1)[: lens[b]].double()))
                for p, c in zip(shared, (s["k_cache"], s["v_cache"])))
        q = s["q"][t:t + n[b]].double().view(n[b], kvh, heads // kvh, dim)
        score = torch.einsum("nhgd,khd->nhgk", q, k) / math.sqrt(dim)
        key = torch.arange(k.shape[0], device=q.device)
        hidden = key[None] > (k.shape[0] - n[b] + torch.arange(n[b], device=q.device))[:, None]
        score = score.masked_fill(hidden[:, None, None], -math.inf)
        out.append(torch.einsum("nhgk,khd->nhgd", score.softmax(-1), v).reshape(n[b], heads, dim))
        t += n[b]
    return torch.cat(out)
