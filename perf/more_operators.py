"""Cases of the operators around a bounded paged cache: norms of queries and keys with the
rotation in the same pass (forward, gradient, and on the way into the cache), the attention
weight that each cached key has gathered, and eviction of the keys that gathered least.

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
_EPS = 1e-6


# ------------------------------------------------------------------------------ the cases
def _norm(name, tokens, heads, kv_heads, dim, rot, layout, dtype, backward=False, offset=0.0, span=4096):
    """tokens rows of heads + kv_heads heads of dim, normed, of which the first rot rotate."""
    return {"op": "norm", "name": name, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rot": rot,
            "layout": layout, "dtype": dtype, "backward": backward, "offset": offset, "span": span}


def _append(name, batch, n_lo, n_hi, len_hi, heads, kv_heads, dim, rot, layout, page, dtype, offset=0.0):
    """n_lo..n_hi new tokens for each of batch sequences, up to len_hi long after them."""
    return {"op": "append", "name": name, "batch": batch, "n_lo": n_lo, "n_hi": n_hi, "len_hi": len_hi, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "rot": rot, "layout": layout, "page": page, "dtype": dtype, "offset": offset}


def _mass(name, batch, n_lo, n_hi, len_lo, len_hi, heads, kv_heads, dim, page, dtype, decay=1.0):
    """n_lo..n_hi query tokens for each of batch sequences that are len_lo..len_hi long with them."""
    return {"op": "mass", "name": name, "batch": batch, "n_lo": n_lo, "n_hi": n_hi, "len_lo": len_lo, "len_hi": len_hi,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "decay": decay}


def _evict(name, batch, len_lo, len_hi, budget, first, recent, kv_heads, dim, page, dtype):
    """Sequences of len_lo..len_hi keys are cut to budget: the first, the recent, the heaviest."""
    return {"op": "evict", "name": name, "batch": batch, "len_lo": len_lo, "len_hi": len_hi, "budget": budget,
            "first": first, "recent": recent, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype}


def listed():
    return [
        # queries and keys of one decoding step of a small batch
        _norm("norm_decode", 7, 32, 8, 128, 128, "half", "bf16"),
        # a training step: an odd number of packed tokens, views of one joint projection
        _norm("norm_train", 16381, 32, 8, 128, 128, "half", "bf16"),
        # its gradient, with those of both weights
        _norm("norm_grad", 16381, 32, 8, 128, 128, "half", "bf16", backward=True),
        # the gradient in 32 bits: neighbours rotate, half of each head does not
        _norm("norm_grad_f32", 5003, 12, 4, 96, 48, "interleaved", "f32", backward=True, offset=1.0),
        # one new token for each sequence of a server
        _append("append_step", 300, 1, 1, 900, 32, 8, 128, 128, "half", 16, "f16"),
        # whole prompts of many lengths are written
        _append("append_prompts", 24, 40, 1900, 1900, 32, 8, 128, 128, "half", 16, "bf16"),
        # the smallest step: a few short sequences
        _mass("mass_small", 3, 1, 1, 50, 300, 16, 4, 64, 16, "bf16"),
        # one token for each sequence of a server: the keys are read once more
        _mass("mass_step", 64, 1, 1, 200, 4000, 32, 8, 128, 16, "bf16", decay=0.98),
        # the last tokens of long prompts weigh them before they are cut
        _mass("mass_window", 12, 32, 32, 700, 16001, 32, 8, 128, 32, "f16", decay=0.0),
        # every token of whole prompts: the compute-bound end
        _mass("mass_prompts", 10, 300, 3500, 300, 3500, 32, 8, 128, 16, "bf16", decay=0.0),
        # sequences a few tokens over their budget, between two decoding steps
        _evict("evict_step", 64, 1000, 1040, 1024, 4, 64, 8, 128, 16, "bf16"),
        # one very long context is cut to an eighth
        _evict("evict_long", 2, 110000, 120001, 15000, 4, 128, 8, 128, 64, "f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "append", "mass", "mass", "evict", "evict"])
    dtype = rng.choice(["bf16", "f16"])
    layout = rng.choice(["half", "interleaved"])
    offset = rng.choice([0.0, 0.0, 1.0])
    if op == "norm":
        dim = rng.choice([64, 80, 96, 128, 256])
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 3, 4, 5])
        dtype = rng.choice(["bf16", "f16", "f32"])
        tokens = min(_log(rng, 1, 16384), 16381 * 40 * 128 * 2 // ((heads + kv_heads) * dim * _SIZE[dtype]))
        c = _norm("", tokens, heads, kv_heads, dim, rng.choice([dim, dim // 2]), layout, dtype, rng.random() < 0.5, offset,
                  _log(rng, 2048, 131072))
    elif op == "append":
        dim = rng.choice([64, 96, 128])
        kv_heads = rng.choice([1, 4, 8])
        heads = kv_heads * rng.choice([1, 4, 5])
        batch = _log(rng, 1, 512)
        n_hi = rng.choice([1, 1, 3, max(1, min(1900, 20000 // batch))])
        c = _append("", batch, max(1, n_hi // 40), n_hi, n_hi + rng.randrange(700), heads, kv_heads, dim,
                    rng.choice([dim, dim // 2]), layout, rng.choice([8, 16, 24, 32, 64]), dtype, offset)
    elif op == "mass":
        dim = rng.choice([64, 128])
        kv_heads = rng.choice([2, 4, 8])
        heads = kv_heads * rng.choice([1, 4, 5, 8])
        batch = _log(rng, 1, 128)
        n_hi = rng.choice([1, 1, 8, 32, max(1, min(2000, 3000 // batch))])
        top = min(120000 // batch, 10 ** 9 // (batch * n_hi * heads))
        len_hi = max(n_hi, _log(rng, 30, max(31, min(60000, top))))
        c = _mass("", batch, max(1, n_hi // 4), n_hi, max(n_hi, len_hi // 8), len_hi, heads, kv_heads, dim,
                  rng.choice([8, 16, 24, 32, 64]), dtype, rng.choice([0.0, 0.9, 1.0]))
    else:
        dim = rng.choice([64, 96, 128])
        kv_heads = rng.choice([1, 4, 8])
        batch = _log(rng, 1, 128)
        len_hi = _log(rng, 40, max(41, min(100000, 200000 // batch)))
        budget = max(16, int(len_hi * rng.uniform(0.1, 0.95)))
        recent = rng.randrange(0, max(1, budget // 4))
        c = _evict("", batch, max(1, int(len_hi * rng.uniform(0.3, 1.0))), len_hi, budget, rng.choice([0, 1, 4]), recent,
                   kv_heads, dim, rng.choice([8, 16, 24, 32, 64]), dtype)
    del c["name"]
    return c


def _spread(lo, hi, n):
    """n whole numbers from hi down to lo."""
    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _shape(case):
    """(new tokens, lengths) of a ragged case's sequences."""
    if case["op"] == "evict":
        return [0] * case["batch"], _spread(case["len_lo"], case["len_hi"], case["batch"])
    n = _spread(case["n_lo"], case["n_hi"], case["batch"])
    if case["op"] == "append":
        return n, [x + (case["len_hi"] - x) * i // max(1, case["batch"]) for i, x in enumerate(n)]
    return n, [max(a, b) for a, b in zip(n, _spread(case["len_lo"], case["len_hi"], case["batch"]))]


def work(case):
    size = _SIZE[case["dtype"]]
    if case["op"] == "norm":
        cells = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": (3 if case["backward"] else 2) * cells * size + 8 * case["tokens"],
                "flops": (12 if case["backward"] else 7) * cells}
    n, lens = _shape(case)
    tokens, kvh, dim = sum(n), case["kv_heads"], case["dim"]
    if case["op"] == "append":
        return {"bytes": 2 * tokens * (case["heads"] + 2 * kvh) * dim * size + 8 * len(n),
                "flops": 7 * tokens * (case["heads"] + kvh) * dim}
    if case["op"] == "mass":
        seen = sum(a * l - a * (a - 1) // 2 for a, l in zip(n, lens))
        old = 4 * (sum(lens) - tokens) * kvh if case["decay"] else 0
        return {"bytes": sum(lens) * kvh * (dim * size + 4) + old + tokens * case["heads"] * (dim * size + 4),
                "flops": 2 * seen * case["heads"] * dim}
    total = 0
    for l in lens:
        budget = min(case["budget"], l)
        gone = l - budget
        if gone:  # the heaviest lie anywhere: so many of them behind their new places
            recent = min(case["recent"], budget)
            heavy = budget - recent - min(case["first"], budget - recent)
            moved = heavy * gone // max(1, heavy + gone) + recent
            total += kvh * (4 * (heavy + gone) + moved * 2 * (2 * dim * size + 4) + 4 * budget)
    return {"bytes": max(total, 1), "flops": sum(lens) * kvh}


# ------------------------------------------------------------------------------ the inputs
def _frequencies(rot, device, base=500000.0):
    return base ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = _DTYPE[case["dtype"]]
    kvh, dim = case["kv_heads"], case["dim"]

    def normal(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32).to(dtype)

    def weight():
        return (1.0 - case["offset"] + 0.3 * normal(dim, dtype=torch.float32)).to(dt)

    s = dict(case)
    if case["op"] in ("norm", "append"):
        s["freq"] = _frequencies(case["rot"], dev)
        s["q_weight"], s["k_weight"] = weight(), weight()
    if case["op"] == "norm":
        heads, tokens = case["heads"], case["tokens"]
        # a joint projection's output, whose heads differ in size
        qkv = (normal(tokens, heads + 2 * kvh, dim, dtype=torch.float32)
               * torch.exp(normal(heads + 2 * kvh, 1, dtype=torch.float32))).to(dt)
        s["q"], s["k"] = qkv[:, :heads], qkv[:, heads:heads + kvh]
        if tokens > 1000:  # packed sequences
            s["positions"] = torch.arange(tokens, device=dev) % case["span"]
        else:
            s["positions"] = torch.randint(0, case["span"], (tokens,), generator=g, device=dev)
        if case["backward"]:
            s["dq"], s["dk"] = normal(tokens, heads, dim), normal(tokens, kvh, dim)
        return s
    n, lens = _shape(case)
    batch, page, tokens = case["batch"], case["page"], sum(n)
    pages = [-(-x // page) for x in lens]
    s["page_indices"] = torch.randperm(sum(pages), generator=g, device=dev)

    def starts(v):
        return torch.tensor([0] + v, device=dev, dtype=torch.int64).cumsum(0)

    s["page_indptr"], s["q_indptr"] = starts(pages), starts(n)
    s["seq_len"] = torch.tensor(lens, device=dev, dtype=torch.int64)
    s["max_pages"], s["max_len"], s["max_q"], s["tokens"] = max(pages), max(lens), max(n), tokens
    s["ragged"] = max(n) > 1
    s["k_cache"] = normal(sum(pages), page, kvh, dim)
    if case["op"] != "mass":
        s["v_cache"] = normal(sum(pages), page, kvh, dim)
    if case["op"] == "append":
        s["q"] = normal(tokens, case["heads"], dim)
        s["k"], s["v"] = normal(tokens, kvh, dim), normal(tokens, kvh, dim)
        return s
    # the weight gathered so far, a few keys with most of it; stored head by head
    some = 4 * case.get("heads", kvh) / kvh / s["max_len"]
    s["mass"] = some * torch.exp(2 * normal(sum(pages), kvh, page, dtype=torch.float32)).transpose(1, 2)
    if case["op"] == "evict":
        s["mass_out"] = torch.zeros(sum(pages), kvh, page, device=dev).transpose(1, 2)
        return s
    s["q"] = normal(tokens, case["heads"], dim)
    # what attention left of its softmax: the logarithm of each row's sum
    s["lse"] = torch.empty(tokens, case["heads"], device=dev)
    t = p = 0
    for a, l, c in zip(n, lens, pages):
        k = s["k_cache"][s["page_indices"][p:p + c]].flatten(0, 1)[:l].float()
        j = torch.arange(l, device=dev)
        hidden = j > (l - a + torch.arange(a, device=dev))[:, None]
        for h in range(kvh):
            group = case["heads"] // kvh
            score = (s["q"][t:t + a, h * group:(h + 1) * group].float() * dim ** -0.5) @ k[:, h].T
            s["lse"][t:t + a, h * group:(h + 1) * group] = score.masked_fill_(hidden[:, None], -math.inf).logsumexp(-1)
        t, p = t + a, p + c
    return s


# ------------------------------------------------------------------------------ plain forms
def _rotate(x, positions, freq, layout, sign=1.0):
    """x [tokens, heads, dim] in 32 bits.  The angle is taken in 64 bits."""
    angle = positions.double()[:, None] * freq
    c, d = angle.cos().float()[:, None], (angle.sin() * sign).float()[:, None]
    rot = 2 * freq.numel()
    r, rest = x[..., :rot], x[..., rot:]
    if layout == "half":
        a, b = r[..., : rot // 2], r[..., rot // 2 :]
        y = torch.cat((a * c - b * d, b * c + a * d), -1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        y = torch.stack((a * c - b * d, b * c + a * d), -1).flatten(-2)
    return torch.cat((y, rest), -1)


def _normed(s, x, weight, positions):
    x = x.float()
    y = x * ((x * x).mean(-1, keepdim=True) + _EPS).rsqrt() * (s["offset"] + weight.float())
    return _rotate(y, positions, s["freq"], s["layout"]).to(weight.dtype)


def _normed_grad(s, dy, x, weight):
    x = x.float()
    r = ((x * x).mean(-1, keepdim=True) + _EPS).rsqrt()
    g = _rotate(dy.float(), s["positions"], s["freq"], s["layout"], -1.0)
    xh, u = x * r, g * (s["offset"] + weight.float())
    dx = r * (u - xh * (u * xh).mean(-1, keepdim=True))
    return dx.to(weight.dtype), (g * xh).sum((0, 1)).to(weight.dtype)


def _owners(s):
    """(sequence, place among its new tokens, place in its sequence) of each new token."""
    t = torch.arange(s["tokens"], device=s["q"].device)
    b = torch.searchsorted(s["q_indptr"], t, right=True) - 1
    i = t - s["q_indptr"][b]
    return b, i, s["seq_len"][b] - (s["q_indptr"][b + 1] - s["q_indptr"][b]) + i


def _plain_append(s):
    b, _, at = _owners(s)
    page = s["page_indices"][s["page_indptr"][b] + at // s["page"]]
    s["k_cache"][page, at % s["page"]] = _normed(s, s["k"], s["k_weight"], at)
    s["v_cache"][page, at % s["page"]] = s["v"]
    return {"q": _normed(s, s["q"], s["q_weight"], at), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _places(s):
    """(places 0 .. longest, page of each, slot of each, whether it is held), by sequence."""
    j = torch.arange(s["max_len"], device=s["seq_len"].device)
    at = (s["page_indptr"][:-1, None] + j // s["page"]).clamp(max=s["page_indices"].numel() - 1)
    return j, s["page_indices"][at], (j % s["page"]).expand(at.shape), j < s["seq_len"][:, None]


def _plain_mass(s):
    kvh, dim, heads, batch, width, long = s["kv_heads"], s["dim"], s["heads"], s["batch"], s["max_q"], s["max_len"]
    group = heads // kvh
    j, page, slot, held = _places(s)
    b, i, _ = _owners(s)
    wide = s["q"].new_zeros(batch, width, heads, dim, dtype=torch.float32)
    wide[b, i] = s["q"].float() * dim ** -0.5
    lse = torch.full((batch, width, heads), math.inf, device=wide.device)  # no token: no weight
    lse[b, i] = s["lse"]
    n = s["q_indptr"].diff()
    last = s["seq_len"][:, None] - n[:, None] + torch.arange(width, device=wide.device)
    hidden = j > last[..., None]
    mass = s["mass"][page, slot]  # [sequence, place, kv head]
    mass = torch.where((j < (s["seq_len"] - n)[:, None])[..., None], s["decay"] * mass, 0.0)
    for h in range(kvh):
        k = s["k_cache"][page, slot, h].float()
        rows = wide[:, :, h * group:(h + 1) * group].reshape(batch, width * group, dim)
        p = rows @ k.transpose(1, 2)
        p = p.sub_(lse[:, :, h * group:(h + 1) * group].reshape(batch, -1, 1)).exp_()
        p = p.view(batch, width, group, long).masked_fill_(hidden[:, :, None], 0.0)
        mass[..., h] += p.sum((1, 2))
    at = held.nonzero(as_tuple=True)
    s["mass"][page[at], slot[at]] = mass[at]
    return s["mass"]


def _plain_evict(s):
    kvh = s["kv_heads"]
    j, page, slot, held = _places(s)
    length = s["seq_len"][:, None, None]
    kept_len = length.clamp(max=s["budget"])
    gone = length - kept_len
    recent = torch.minimum(kept_len, torch.full_like(kept_len, s["recent"]))
    first = torch.minimum(kept_len - recent, torch.full_like(kept_len, s["first"]))
    heavy = kept_len - recent - first
    between = (j >= first) & (j < length - recent)
    mass = s["mass"][page, slot].transpose(1, 2)  # [sequence, kv head, place]
    order = torch.where(between, mass, -math.inf).argsort(dim=-1, descending=True, stable=True)
    chosen = torch.zeros_like(mass, dtype=torch.bool).scatter_(2, order, (j < heavy).expand(mass.shape))
    front = j < first + heavy
    hole, moved = between & front & ~chosen, chosen & ~front
    # the moved ones, in order, and the holes that they fill, in order
    sources = moved.int().argsort(dim=-1, descending=True, stable=True)
    fill = sources.gather(2, (hole.cumsum(-1) - 1).clamp(min=0))
    kept = torch.where(hole, fill, j.expand(mass.shape))
    kept = torch.where(front, kept, (j + gone).expand(mass.shape))
    kept = torch.where(j < kept_len, kept, -1)
    b, h, to = (kept >= 0).nonzero(as_tuple=True)
    old = kept[b, h, to]
    src, dst = (page[b, old], slot[b, old], h), (page[b, to], slot[b, to], h)
    for x, y in ((s["k_cache"], s["k_cache"]), (s["v_cache"], s["v_cache"]), (s["mass"], s["mass_out"])):
        y[dst] = x[src]
    return {"seq_len": kept_len.flatten(), "kept": kept[..., : s["budget"]].int(), "k_cache": s["k_cache"],
            "v_cache": s["v_cache"], "mass": s["mass_out"]}


# ------------------------------------------------------------------------------ one pass
def _own_run(s):
    from tilegen_b200 import paged

    if s["op"] in ("norm", "append"):
        rope = paged.Rope(s["freq"], s["layout"])
        norms = [paged.HeadNorm(s[w], _EPS, s["offset"]) for w in ("q_weight", "k_weight")]
    if s["op"] == "norm":
        if s["backward"]:
            return paged.norm_rope_backward(s["dq"], s["dk"], s["q"], s["k"], *norms, rope, s["positions"])
        return paged.norm_rope(s["q"], s["k"], *norms, rope, s["positions"])
    table = paged.PageTable(s["page_indptr"], s["page_indices"])
    if s["op"] == "mass":
        ragged = {"q_indptr": s["q_indptr"], "max_q_len": s["max_q"]} if s["ragged"] else {}
        cache = paged.PagedKV(s["k_cache"], s["k_cache"])  # values are not read
        return paged.attention_mass(s["mass"], s["q"], cache, table, s["seq_len"], s["lse"], max_seq_len=s["max_len"],
                                    decay=s["decay"], **ragged)
    cache = paged.PagedKV(s["k_cache"], s["v_cache"])
    if s["op"] == "append":
        q = paged.kv_append(cache, table, s["seq_len"], s["k"], s["v"], rope=rope, q=s["q"], q_norm=norms[0], k_norm=norms[1],
                            q_indptr=s["q_indptr"] if s["ragged"] else None)
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    seq_len, kept = paged.kv_evict(cache, table, s["seq_len"], s["mass"], s["budget"], first=s["first"], recent=s["recent"],
                                   max_seq_len=s["max_len"], mass_out=s["mass_out"], kept=True)
    return {"seq_len": seq_len, "kept": kept, "k_cache": s["k_cache"], "v_cache": s["v_cache"], "mass": s["mass_out"]}


def run(state):
    s = state
    if own:
        return _own_run(s)
    if s["op"] == "append":
        return _plain_append(s)
    if s["op"] == "mass":
        return _plain_mass(s)
    if s["op"] == "evict":
        return _plain_evict(s)
    if not s["backward"]:
        return tuple(_normed(s, s[x], s[x + "_weight"], s["positions"]) for x in "qk")
    (dq, dqw), (dk, dkw) = (_normed_grad(s, s["d" + x], s[x], s[x + "_weight"]) for x in "qk")
    return dq, dk, dqw, dkw


# ------------------------------------------------------------------------------ in 64 bits
def _turned(s, x, weight, positions):
    """x over the root of its mean square, each pair as a complex number times exp(i angle)."""
    rot = 2 * s["freq"].numel()
    x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + _EPS) * (weight + s["offset"])
    first, second = ((slice(0, rot // 2), slice(rot // 2, rot)) if s["layout"] == "half"
                     else (slice(0, rot, 2), slice(1, rot, 2)))
    angle = positions.double()[:, None] * s["freq"]
    z = torch.complex(x[..., first], x[..., second]) * torch.polar(torch.ones_like(angle), angle)[:, None]
    pairs = (z.real, z.imag)
    turned = torch.cat(pairs, -1) if s["layout"] == "half" else torch.stack(pairs, -1).flatten(-2)
    return torch.cat((turned, x[..., rot:]), -1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        if not case["backward"]:
            return tuple(_turned(s, s[x].double(), s[x + "_weight"].double(), s["positions"]) for x in "qk")
        grads = []
        for x in "qk":
            leaf = s[x].double().requires_grad_()
            w = s[x + "_weight"].double().requires_grad_()
            grads.append(torch.autograd.grad(_turned(s, leaf, w, s["positions"]), (leaf, w), s["d" + x].double()))
        return grads[0][0], grads[1][0], grads[0][1], grads[1][1]
    n, lens = _shape(case)
    ip, ix, page, kvh = s["page_indptr"].tolist(), s["page_indices"], case["page"], case["kv_heads"]
    places = [torch.arange(l, device=ix.device) for l in lens]
    where = [(ix[ip[b]:ip[b + 1]][j // page], j % page) for b, j in enumerate(places)]
    if case["op"] == "append":
        kc, vc, out, t = s["k_cache"].double(), s["v_cache"].double(), [], 0
        for b in range(case["batch"]):
            new = slice(lens[b] - n[b], lens[b])
            to = tuple(w[new] for w in where[b])
            out.append(_turned(s, s["q"][t:t + n[b]].double(), s["q_weight"].double(), places[b][new]))
            kc[to] = _turned(s, s["k"][t:t + n[b]].double(), s["k_weight"].double(), places[b][new])
            vc[to] = s["v"][t:t + n[b]].double()
            t += n[b]
        return {"q": torch.cat(out), "k_cache": kc, "v_cache": vc}
    if case["op"] == "mass":
        if work(case)["flops"] > 1e13:
            return None
        mass, t = s["mass"].double(), 0
        group = case["heads"] // kvh
        for b in range(case["batch"]):
            k = s["k_cache"][where[b]].double()
            for h in range(kvh):
                q = s["q"][t:t + n[b], h * group:(h + 1) * group].double()
                p = torch.exp(torch.einsum("ngd,kd->ngk", q, k[:, h]) / math.sqrt(case["dim"])
                              - s["lse"][t:t + n[b], h * group:(h + 1) * group].double()[..., None])
                sees = places[b][None] <= (lens[b] - n[b] + torch.arange(n[b], device=k.device))[:, None]
                gathered = (p * sees[:, None]).sum((0, 1))
                old = mass[where[b] + (torch.full_like(places[b], h),)]
                old[lens[b] - n[b]:] = 0.0
                mass[where[b] + (torch.full_like(places[b], h),)] = case["decay"] * old + gathered
            t += n[b]
        return mass
    kc, vc, out = s["k_cache"].double(), s["v_cache"].double(), s["mass_out"].double()
    kept = torch.full((case["batch"], kvh, min(case["budget"], max(lens))), -1, device=ix.device, dtype=torch.int32)
    new_len = []
    for b, l in enumerate(lens):
        size = min(l, case["budget"])
        recent = min(case["recent"], size)
        first = min(case["first"], size - recent)
        heavy, new = size - recent - first, size - recent
        new_len.append(size)
        for h in range(kvh):
            m = s["mass"][where[b]][:, h]
            value, at = torch.sort(m[first:l - recent], descending=True, stable=True)
            chosen = (at[:heavy] + first).sort().values
            stay, move = chosen[chosen < new], chosen[chosen >= new]
            source = places[b][:size].clone()
            free = torch.ones(size, dtype=torch.bool, device=m.device)
            free[:first], free[new:], free[stay] = False, False, False
            source[free] = move
            source[new:] = places[b][l - recent:]
            kept[b, h, :size] = source.int()
            page_of, slot_of = where[b]
            for x, y in ((s["k_cache"], kc), (s["v_cache"], vc), (s["mass"], out)):
                y[page_of[:size], slot_of[:size], h] = x[page_of[source], slot_of[source], h].double()
    return {"seq_len": torch.tensor(new_len, device=ix.device), "kept": kept, "k_cache": kc, "v_cache": vc, "mass": out}
