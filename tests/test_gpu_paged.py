"""Rotary positions, cache append and shared-prefix attention on the GPU against plain
implementations in 64 bits.

Bounds, all derived before the first run.  u is half an ulp of the 16-bit type relative to the
value (2^-8 bfloat16, 2^-11 float16, 2^-24 float32; float16 below 2^-14 has an absolute 2^-25).

* A rotation is one rounding of a 32-bit result: u |y| + 2^-20 scale (|a| + |b|) (sine, cosine
  and the reduced angle are good to 2^-22, three 32-bit operations follow).
* Attention rounds P once and the output once: u |out| + u sum_k p_k |v_k|, and the scores carry
  32-bit errors of the products' sums, e = 2^-18 (1 + max_k scale sum_d |q_d k_d|), each p_k a
  relative error of at most 2 e: (u + 4 e) sum_k p_k |v_k| + u |out|.
* log-sum-exp: 4 e absolute.
"""

from __future__ import annotations

import math

import pytest
import torch

from tilegen_b200 import lib
from tilegen_b200 import paged as P

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


# ------------------------------------------------------------------ rotary positions
def rotate64(x, pos, r, sign=1):
    """(rotated, bound's |a| + |b|) in 64 bits."""
    x = x.double()
    n = r.freq.numel()
    t = (pos.double()[:, None] * r.freq)[:, None]
    c, s = t.cos() * r.scale, t.sin() * r.scale * sign
    y, mag = x.clone(), torch.zeros_like(x)
    ia, ib = ((slice(0, n), slice(n, 2 * n)) if r.layout == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2)))
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia] = mag[..., ib] = (a.abs() + b.abs()) * r.scale
    return y, mag


def check_rotated(y, ref, mag, dtype):
    tol = U[dtype] * ref.abs() + 2.0 ** -20 * mag + (2.0 ** -25 if dtype == F16 else 0.0)
    bad = (y.double() - ref).abs() > tol
    assert not bool(bad.any()), "%d of %d, worst %g" % (int(bad.sum()), bad.numel(), float((y.double() - ref).abs().max()))


ROPE_SHAPES = [  # tokens, heads, dim, rotating
    (1, 1, 2, 2), (1, 32, 128, 128), (5, 3, 80, 40), (7, 5, 96, 48), (33, 2, 20, 12), (130, 8, 64, 64), (3, 1, 36, 0),
    (1201, 4, 128, 32), (2, 3, 600, 600), (9, 40, 256, 256), (64, 1, 7, 4),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,dim,rot", ROPE_SHAPES)
def test_rope(tokens, heads, dim, rot, layout, dtype):
    g = gen(tokens * 1000 + dim)
    x = normal(g, tokens, heads, dim, dtype=dtype)
    pos = torch.randint(0, 1 << 20, (tokens,), generator=g, device="cuda")
    r = P.Rope(P.rope_frequencies(rot, scaling="banded", factor=4.0), layout, 1.25)
    y = P.rope(x, r, pos)
    check_rotated(y, *rotate64(x, pos, r), dtype)
    z = P.rope_backward(x, r, pos)
    check_rotated(z, *rotate64(x, pos, r, -1), dtype)
    assert torch.equal(y[..., rot:], x[..., rot:]) and torch.equal(z[..., rot:], x[..., rot:])
    w = x.clone()
    assert P.rope(w, r, pos, out=w) is w and torch.equal(w, y)  # in place


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_strides_and_far_positions(layout):
    g = gen(3)
    qkv = normal(g, 50, 3, 6, 64, dtype=BF16)  # heads of a joint projection
    x = qkv[:, 1]
    pos = torch.tensor([0, 1, -5, (1 << 31) + 7, 1 << 40] * 10, device="cuda")
    r = P.Rope(P.rope_frequencies(64), layout)
    check_rotated(P.rope(x, r, pos), *rotate64(x, pos, r), BF16)
    heads_first = normal(g, 6, 50, 64, dtype=BF16).transpose(0, 1)
    out = torch.empty(50, 6, 65, dtype=BF16, device="cuda")[..., :64]  # rows off the 16-byte grid
    assert P.rope(heads_first, r, pos, out=out) is out
    check_rotated(out, *rotate64(heads_first, pos, r), BF16)
    shifted = torch.empty(50 * 6 * 64 + 1, dtype=BF16, device="cuda")[1:].view(50, 6, 64).copy_(x)
    check_rotated(P.rope(shifted, r, pos), *rotate64(x, pos, r), BF16)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_gradient_against_autograd_and_differences(layout):
    g = gen(11)
    x, dy = normal(g, 6, 3, 24), normal(g, 6, 3, 24)
    pos = torch.randint(0, 5000, (6,), generator=g, device="cuda")
    r = P.Rope(P.rope_frequencies(16), layout, 0.75)
    dx = P.rope_backward(dy, r, pos)
    leaf = x.double().requires_grad_()
    t = (pos.double()[:, None] * r.freq)[:, None]
    c, s = t.cos() * r.scale, t.sin() * r.scale
    a, b = (leaf[..., :8], leaf[..., 8:16]) if layout == "half" else (leaf[..., 0:16:2], leaf[..., 1:16:2])
    u, w = a * c - b * s, b * c + a * s
    y = torch.cat((torch.cat((u, w), -1) if layout == "half" else torch.stack((u, w), -1).flatten(-2), leaf[..., 16:]), -1)
    y.backward(dy.double())
    check_rotated(dx, leaf.grad, torch.full_like(leaf.grad, 8.0), F32)
    # the map is linear: a difference quotient is exact up to 32-bit rounding of its two ends
    step = normal(g, 6, 3, 24)
    num = ((P.rope(x + step, r, pos).double() - P.rope(x - step, r, pos).double()) / 2 * dy.double()).sum()
    assert abs(float(num - (dx.double() * step.double()).sum())) < 6 * 3 * 24 * 8 * 16 * 2.0 ** -22


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rope_takes_part_in_autograd(layout, dtype):
    """The gradient that reaches x is rope_backward's, of a whole tensor, of a joint projection's
    view and of an expanded number; without a gradient asked for, the result has none."""
    g = gen(13)
    r = P.Rope(P.rope_frequencies(40), layout, 1.5)
    pos = torch.randint(0, 9000, (33,), generator=g, device="cuda")
    qkv = normal(g, 33, 6, 64, dtype=dtype).requires_grad_()
    x, dy = qkv[:, 1:5], normal(g, 33, 4, 64, dtype=dtype)
    y = P.rope(x, r, pos)
    assert torch.equal(y, P.rope(x.detach(), r, pos))
    (grad,) = torch.autograd.grad(y, qkv, dy, retain_graph=True)
    assert torch.equal(grad[:, 1:5], P.rope_backward(dy, r, pos)) and not bool(grad[:, 0].any() | grad[:, 5].any())
    (grad,) = torch.autograd.grad(y.sum(), qkv)
    assert torch.equal(grad[:, 1:5], P.rope_backward(torch.ones_like(dy), r, pos))
    # of the gradient in turn, and on another stream
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    y = P.rope(x, r, pos, stream=st)
    torch.cuda.current_stream().wait_stream(st)
    up = dy.clone().requires_grad_()
    (grad,) = torch.autograd.grad(y, x, up, create_graph=True)
    (back,) = torch.autograd.grad(grad, up, x.detach())
    assert torch.equal(back, y.detach())
    with torch.no_grad():
        assert not P.rope(x, r, pos).requires_grad
    assert not P.rope(x, r, pos, out=torch.empty_like(dy)).requires_grad


def test_rope_empty_and_refusals():
    r = P.Rope(P.rope_frequencies(8))
    pos = torch.zeros(4, dtype=torch.int64, device="cuda")
    assert P.rope(torch.zeros(0, 3, 8, device="cuda"), r, pos[:0]).shape == (0, 3, 8)
    assert P.rope(torch.zeros(4, 0, 8, device="cuda"), r, pos).shape == (4, 0, 8)
    x = torch.zeros(4, 3, 8, device="cuda")
    for bad in (lambda: P.rope(x.double(), r, pos), lambda: P.rope(x, r, pos[:3]), lambda: P.rope(x, r, pos.int()),
                lambda: P.rope(x.transpose(1, 2), r, pos), lambda: P.rope(x, P.Rope(r.freq.float()), pos),
                lambda: P.rope(x, P.Rope(r.freq, "quarter"), pos), lambda: P.rope(x, r, pos, out=x[:, :2]),
                lambda: P.rope(x, P.Rope(r.freq.cpu()), pos)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(lib.TgError) as e:
        P.rope(x[..., :6], r, pos)  # rotates more than the head
    assert e.value.status == lib.TG_EINVAL


# ------------------------------------------------------------------ a cache and its sequences
class Batch:
    """Sequences with `news` query tokens and own lengths `lens` behind `prefix` shared tokens,
    on pages in random order; every slot that no sequence holds is NaN."""

    def __init__(self, news, lens, prefix, heads, kv_heads, dim, page, dtype, seed=0, heads_first=False, spare=3):
        g = gen(seed)
        self.news, self.lens, self.prefix, self.page, self.dim, self.dtype = news, lens, prefix, page, dim, dtype
        self.heads, self.kv_heads = heads, kv_heads
        own = [-(-n // page) for n in lens]
        npre = -(-prefix // page)
        total = sum(own) + npre + spare
        order = torch.randperm(total, generator=g, device="cuda")
        self.prefix_pages = order[:npre].contiguous()
        flat = order[npre:npre + sum(own)].tolist()
        rows, at = [], 0
        for n in own:
            rows.append(flat[at:at + n])
            at += n
        self.table = P.PageTable.from_lists(rows)
        shape = (total, kv_heads, page, dim) if heads_first else (total, page, kv_heads, dim)
        k, v = (torch.full(shape, math.nan, device="cuda", dtype=dtype) for _ in range(2))
        if heads_first:
            k, v = k.transpose(1, 2), v.transpose(1, 2)
        self.cache = P.PagedKV(k, v)
        self.own = []
        for pages, n in [(self.prefix_pages.tolist(), prefix)] + list(zip(rows, lens)):
            kk, vv = normal(g, n, kv_heads, dim, dtype=dtype), normal(g, n, kv_heads, dim, dtype=dtype)
            self.own.append([kk, vv])
            self.write(pages, kk, vv)
        self.rows = rows
        self.shared = self.own.pop(0)
        self.seq_len = torch.tensor(lens, dtype=torch.int64, device="cuda")
        self.q = normal(g, sum(news), heads, dim, dtype=dtype)
        self.q_indptr = torch.tensor([0] + news, dtype=torch.int64, device="cuda").cumsum(0)

    def write(self, pages, k, v):
        for i, pg in enumerate(pages):
            part = slice(i * self.page, (i + 1) * self.page)
            n = k[part].shape[0]
            self.cache.k[pg, :n], self.cache.v[pg, :n] = k[part], v[part]

    def args(self, **kw):
        a = dict(prefix_pages=self.prefix_pages, prefix_len=self.prefix)
        if any(n != 1 for n in self.news):
            a.update(q_indptr=self.q_indptr, max_q_len=max(self.news))
        a.update(kw)
        return (self.q, self.cache, self.table, self.seq_len), a

    def run(self, **kw):
        pos, named = self.args(**kw)
        return P.prefix_attention(*pos, **named)

    def check(self, out, lse=None, causal=True, scale=None):
        scale = self.dim ** -0.5 if scale is None else scale
        u, t0 = U[self.dtype], 0
        assert out.dtype == self.dtype and out.shape == self.q.shape
        for (k, v), n, length in zip(self.own, self.news, self.lens):
            if n == 0:
                continue
            k, v = (torch.cat((s, o)).double() for s, o in zip(self.shared, (k, v)))
            total = k.shape[0]
            q = self.q[t0:t0 + n].double().view(n, self.kv_heads, -1, self.dim)
            sc = torch.einsum("nhgd,khd->nhgk", q, k) * scale
            seen = torch.arange(total, device="cuda")[None] < total - n + 1 + torch.arange(n, device="cuda")[:, None]
            seen = (seen if causal else torch.ones_like(seen))[:, None, None]
            big = (torch.einsum("nhgd,khd->nhgk", q.abs(), k.abs()) * scale).nan_to_num(0, 0, 0)
            e = 2.0 ** -18 * (1 + big.masked_fill(~seen, 0).amax(-1)) if total else torch.zeros(())
            p = sc.masked_fill(~seen, -math.inf).softmax(-1).masked_fill(~seen, 0) if total else sc
            none = ~seen.any(-1).expand(sc.shape[:-1])
            p = p.masked_fill(none[..., None], 0)
            # a key that a query does not see has no part in its sum, whatever its value
            pe, ve = p.permute(1, 0, 2, 3).flatten(1, 2), v.permute(1, 0, 2)
            hidden = (~seen).expand(sc.shape).permute(1, 0, 2, 3).flatten(1, 2)
            finite = ve.isfinite().all(-1)
            ref = pe @ ve.masked_fill(~finite[..., None], 0)
            for h, key in (~finite).nonzero().tolist():
                add = torch.where(hidden[h, :, key, None], 0.0, pe[h, :, key, None] * ve[h, key])
                ref[h] += add
            mag = pe @ ve.abs().masked_fill(~finite[..., None], 0)
            shape = (self.kv_heads, n, -1, self.dim)
            ref, mag = (x.view(shape).permute(1, 0, 2, 3) for x in (ref, mag))
            got = out[t0:t0 + n].double().view(n, self.kv_heads, -1, self.dim)
            ok = ref.isfinite()
            assert torch.equal(got.isfinite(), ok)
            tol = u * ref.abs() + (u + 4 * (e[..., None] if e.dim() else e)) * mag + (2.0 ** -25 if self.dtype == F16 else 0)
            err = (got - ref).abs()
            assert bool((err <= tol)[ok].all()), "worst %g of its bound" % float((err / tol)[ok].max())
            if lse is not None:
                want = sc.masked_fill(~seen, -math.inf).logsumexp(-1) if total else torch.full(sc.shape[:-1], -math.inf, device="cuda")
                has = lse[t0:t0 + n].double().view(want.shape)
                assert torch.equal(has == -math.inf, want == -math.inf)
                assert bool(((has - want).abs() <= 4 * e)[want > -math.inf].all())
            t0 += n


# ------------------------------------------------------------------ attention
ATTEND = [  # news, lens, prefix, heads, kv heads, dim, page
    ([1], [1], 0, 1, 1, 64, 16),
    ([1], [1], 1, 4, 1, 128, 1),
    ([1, 1, 1], [0, 5, 300], 0, 8, 2, 128, 16),
    ([1, 1, 1], [0, 17, 1], 77, 8, 8, 96, 7),
    ([1] * 9, [3, 64, 65, 127, 128, 129, 255, 600, 0], 1000, 8, 2, 64, 64),
    ([1, 1], [40, 900], 4100, 12, 4, 256, 24),
    ([1, 1], [2000, 33], 0, 10, 2, 128, 100),
    ([1] * 40, [9] * 40, 515, 6, 2, 128, 16),
    ([3, 0, 1, 20], [3, 4, 90, 33], 50, 8, 2, 128, 16),
    ([70, 5], [70, 300], 200, 4, 1, 64, 32),
    ([150, 129, 1], [150, 400, 90], 333, 8, 2, 128, 16),
    ([150, 129, 1], [150, 400, 90], 0, 8, 2, 64, 48),
    ([90, 33], [290, 33], 130, 5, 1, 96, 16),
    ([40, 12], [40, 19], 20, 4, 2, 256, 8),
    ([5, 9], [2, 0], 3, 4, 2, 128, 16),    # queries before the own part, and before everything
    ([30, 300], [20, 100], 150, 4, 2, 128, 16),
    ([300], [1500], 0, 16, 2, 128, 128),
    ([1] * 130, [30] * 130, 700, 16, 4, 128, 16),
    ([1] * 130, [30] * 130, 129, 8, 4, 64, 32),
    ([2] * 70, [30] * 70, 2000, 24, 4, 128, 16),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("case", range(len(ATTEND)))
def test_attention(case, dtype):
    b = Batch(*ATTEND[case], dtype, seed=case)
    out, lse = b.run(lse=True)
    b.check(out, lse)
    assert torch.equal(b.run(max_seq_len=max(b.lens)), b.run(max_seq_len=max(b.lens)))  # the same twice
    b.check(b.run(max_seq_len=max(b.lens)))


@pytest.mark.parametrize("case", [4, 8, 10, 14, 15, 17, 19])
def test_attention_without_a_mask(case):
    b = Batch(*ATTEND[case], BF16, seed=case)
    out, lse = b.run(lse=True, causal=False, scale=0.3)
    b.check(out, lse, causal=False, scale=0.3)


@pytest.mark.parametrize("case", [4, 8, 10, 13, 17])
def test_attention_strides(case):
    """A cache stored head by head, queries inside a joint projection, outputs inside a larger
    buffer."""
    b = Batch(*ATTEND[case], BF16, seed=case, heads_first=True)
    t, h, d = b.q.shape
    wide = torch.zeros(t, h + 2 * b.kv_heads, d, dtype=BF16, device="cuda")
    wide[:, :h] = b.q
    b.q = wide[:, :h]
    buf = torch.full((t, h + 1, d + 8), 7.0, dtype=BF16, device="cuda")
    out = buf[:, :h, :d]
    assert b.run(out=out) is out
    b.check(out)
    assert bool((buf[:, h] == 7).all()) and bool((buf[..., d:] == 7).all())
    heads_first = b.q.transpose(0, 1).contiguous().transpose(0, 1)
    b.q = heads_first
    b.check(b.run())


@pytest.mark.parametrize("news,lens,prefix", [([6, 40], [30, 90], 0), ([200, 100], [200, 260], 100), ([150], [150], 0),
                                              ([3, 2], [1, 2], 40)])
@pytest.mark.parametrize("dim", [64, 128])
def test_values_after_a_querys_token_do_not_reach_it(news, lens, prefix, dim):
    """NaN and infinities at keys that only later queries see."""
    b = Batch(news, lens, prefix, 8, 2, dim, 16, BF16, seed=5)
    for s, (n, length) in enumerate(zip(news, lens)):
        for at, what in ((length - 1, math.nan), (max(length - n // 2, 0), math.inf)):
            if at >= length:
                continue
            b.own[s][1][at, 0, 3] = what
            b.own[s][0][length - 1, 1, 5] = math.nan  # and a key
        b.write(b.rows[s], *b.own[s])
    out = b.run()
    t0 = 0
    for s, n in enumerate(news):  # the last queries see the NaN key: all of that head is NaN
        assert bool(out[t0 + n - 1, b.heads // 2:].isnan().all())
        assert bool(out[t0:t0 + n - 1, b.heads // 2:].isfinite().all())
        t0 += n
    for s in range(len(news)):
        b.own[s][0][:, 1] = 0.0
    half = b.heads // 2
    cut = Batch(news, lens, prefix, 8, 2, dim, 16, BF16, seed=5)
    cut.own, cut.q = [[k[:, :1], v[:, :1]] for k, v in b.own], b.q[:, :half]
    cut.shared = [x[:, :1] for x in cut.shared]
    cut.heads, cut.kv_heads = half, 1
    cut.check(out[:, :half].contiguous())


def test_infinite_values_that_are_seen():
    b = Batch([1, 1], [40, 50], 30, 4, 2, 128, 16, BF16, seed=2)
    b.shared[1][3, 0, 7] = math.inf
    b.write(b.prefix_pages.tolist(), *b.shared)
    out = b.run()
    assert bool((out[:, :2, 7] == math.inf).all())
    assert int(out.isfinite().logical_not().sum()) == 4


def test_large_scores_do_not_overflow():
    b = Batch([1, 1, 1], [200, 3, 65], 400, 4, 2, 128, 16, BF16, seed=2)
    b.q *= 64
    out, lse = b.run(lse=True)
    b.check(out, lse)


def test_cache_offsets_beyond_32_bits():
    """Pages past 2^31 elements of the cache (k and v share the memory)."""
    page, heads, dim = 64, 8, 128
    pages = (1 << 31) // (page * heads * dim) + 40
    flat = torch.zeros(pages, page, heads, dim, dtype=BF16, device="cuda")
    b = Batch([1, 2], [100, 130], 200, 16, heads, dim, page, BF16, seed=1)
    moved = torch.arange(pages - b.cache.pages, pages, device="cuda")
    flat[moved] = b.cache.k
    other = torch.zeros_like(flat)
    other[moved] = b.cache.v
    b.cache = P.PagedKV(flat, other)
    b.table = P.PageTable(b.table.indptr, moved[b.table.indices])
    b.prefix_pages = moved[b.prefix_pages]
    b.check(b.run())
    k = normal(gen(2), 3, heads, dim, dtype=BF16)
    P.kv_append(b.cache, b.table, b.seq_len, k, k, q_indptr=b.q_indptr)
    last = b.table.indices[b.table.indptr[1:] - 1]
    assert torch.equal(flat[last[0], 99 % page], k[0]) and torch.equal(other[last[1], 129 % page], k[2])


@pytest.mark.parametrize("news,dim,page", [([1, 1], 128, 16), ([1, 1], 64, 7), ([40, 30], 128, 16), ([40, 90], 64, 24), ([200, 9], 64, 8)])
def test_pages_outside_the_cache_read_as_zeros(news, dim, page):
    """Lengths beyond the listed pages are cut to them, pages that do not exist hold zeros."""
    b = Batch(news, [200, 150], 90, 8, 2, dim, page, BF16, seed=3)
    bad = b.table.indices.clone()
    bad[1], bad[int(b.table.indptr[1]) + 2] = b.cache.pages + 3, -2
    b.table = P.PageTable(b.table.indptr, bad)
    pre = b.prefix_pages.clone()
    pre[-1] = 1 << 40
    b.prefix_pages = pre
    for s, i in ((0, 1), (1, 2)):
        for x in b.own[s]:
            x[i * page:(i + 1) * page] = 0
    for x in b.shared:
        x[(len(pre) - 1) * page:] = 0
    b.check(b.run())
    b.seq_len = torch.tensor([10 ** 12, -4], device="cuda")
    b.lens = [len(b.rows[0]) * page, 0]
    b.own[1] = [x[:0] for x in b.own[1]]
    for x in (b.cache.k, b.cache.v):  # the last page's free slots are seen now
        x[b.rows[0][-1]] = x[b.rows[0][-1]].nan_to_num(0.0)
    b.own[0] = [torch.cat((x, x.new_zeros(b.lens[0] - x.shape[0], *x.shape[1:]))) for x in b.own[0]]
    b.check(b.run())


def test_attention_on_another_stream_and_workspace():
    b = Batch(*ATTEND[9], BF16, seed=4)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    pos, named = b.args()
    n = P.prefix_attention_workspace_bytes(*pos, **named)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    st.wait_stream(torch.cuda.current_stream())
    out = b.run(stream=st, workspace=ws)
    st.synchronize()
    b.check(out)
    with pytest.raises(ValueError, match="workspace"):
        b.run(workspace=ws[: n - 16])


def test_a_decoding_step_in_a_graph():
    """Captured once, replayed with other contents and lengths."""
    b = Batch([1] * 5, [30, 7, 64, 2, 90], 300, 8, 2, 128, 16, BF16, seed=8)
    pos, named = b.args(max_seq_len=96)
    ws = torch.empty(P.prefix_attention_workspace_bytes(*pos, **named), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(b.q)
    b.run(max_seq_len=96, out=out, workspace=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        b.run(max_seq_len=96, out=out, workspace=ws)
    g.replay()
    b.check(out)
    b.q.copy_(normal(gen(9), *b.q.shape, dtype=BF16))
    b.lens = [29, 1, 33, 0, 81]
    b.seq_len.copy_(torch.tensor(b.lens))
    b.own = [[k[:n], v[:n]] for (k, v), n in zip(b.own, b.lens)]
    g.replay()
    b.check(out)


def test_attention_empty_and_refusals():
    b = Batch([1, 1], [5, 6], 20, 4, 2, 64, 16, BF16)
    e = Batch([], [], 20, 4, 2, 64, 16, BF16)
    assert e.run().shape == (0, 4, 64)
    pos, named = b.args()
    q, cache, table, seq_len = pos
    f32 = P.PagedKV(cache.k.float(), cache.v.float())
    for bad in (lambda: P.prefix_attention(q.float(), cache, table, seq_len), lambda: P.prefix_attention(q[:1], cache, table, seq_len),
                lambda: P.prefix_attention(q, f32, table, seq_len), lambda: P.prefix_attention(q, cache, table, seq_len[:1]),
                lambda: P.prefix_attention(q, cache, table, seq_len.int()),
                lambda: P.prefix_attention(q, P.PagedKV(cache.k, cache.v[:-1]), table, seq_len),
                lambda: P.prefix_attention(q, cache, table, seq_len, lse=torch.empty(2, 3, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(lib.TgError, match="prefix_len"):
        P.prefix_attention(q, cache, table, seq_len, prefix_pages=b.prefix_pages, prefix_len=33)
    with pytest.raises(lib.TgError, match="multiple"):
        P.prefix_attention(q[:, :3], cache, table, seq_len)


def test_index_check():
    b = Batch([1, 2], [5, 16], 20, 4, 2, 64, 16, BF16)
    b.check(b.run(check=True))
    good = b.table, b.seq_len, b.prefix_pages, b.q_indptr

    def raises(word, **kw):
        with pytest.raises(lib.TgError, match=word) as e:
            b.run(check=True, **kw)
        assert e.value.status == lib.TG_EBOUNDS

    ip, ix = b.table.indptr, b.table.indices
    b.table = P.PageTable(ip, torch.full_like(ix, b.cache.pages))
    raises("page out of range")
    b.table = P.PageTable(ip.flip(0), ix)
    raises("indptr")
    b.table = good[0]
    b.seq_len = torch.tensor([5, 17], device="cuda")
    raises("seq_len")
    b.seq_len = good[1]
    raises("seq_len", max_seq_len=15)
    b.prefix_pages = torch.full_like(b.prefix_pages, -1)
    raises("prefix page")
    b.prefix_pages = good[2]
    raises("q_indptr", max_q_len=1)
    b.q_indptr = torch.tensor([0, 1, 2], device="cuda")
    raises("q_indptr")
    k = normal(gen(0), 3, 2, 64, dtype=BF16)
    with pytest.raises(lib.TgError, match="more new tokens"):
        P.kv_append(b.cache, b.table, torch.tensor([0, 5], device="cuda"), k, k, q_indptr=good[3], check=True)


def test_index_checks_of_several_threads_keep_apart():
    """Checked calls of good and bad tables, paged and sparse, each from a thread and a stream of its
    own: every bad one is refused and no good one.  (The bad matrix is bad by its column count alone,
    and a page outside the cache reads as zeros, so a check that failed to tell would do no harm.)"""
    import threading

    from tilegen_b200 import codegen, device

    b = Batch([1, 2], [5, 16], 20, 4, 2, 64, 16, BF16)
    (q, cache, table, seq_len), named = b.args()
    off = P.PageTable(table.indptr, torch.full_like(table.indices, cache.pages))
    sched = codegen.generate("spmv", codegen.Config(bounds_check=True))
    ip = torch.arange(0, 2 * 500 + 1, 2, device="cuda")
    ix = torch.arange(1000, device="cuda") % 400
    x = torch.ones(400, dtype=torch.float64, device="cuda")
    good = device.DeviceCSR(ip, ix, torch.ones(1000, dtype=torch.float64, device="cuda"), (500, 400))
    bad = device.DeviceCSR(ip, ix, good.data, (500, 399))
    calls = [(True, lambda st: P.prefix_attention(q, cache, table, seq_len, check=True, stream=st, **named)),
             (False, lambda st: P.prefix_attention(q, cache, off, seq_len, check=True, stream=st, **named)),
             (True, lambda st: device.spmv(good, x, sched=sched, stream=st)),
             (False, lambda st: device.spmv(bad, x[:399], sched=sched, stream=st))] * 2
    wrong = []

    def work(fine, call):
        st = torch.cuda.Stream()
        for _ in range(300):
            try:
                call(st)
                refused = False
            except lib.TgError as e:
                refused = e.status == lib.TG_EBOUNDS
                if not refused:
                    wrong.append(str(e))
            if refused == fine:
                wrong.append("refused" if refused else "let pass")
        st.synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=c) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, "%d of %d: %s" % (len(wrong), 300 * len(calls), sorted(set(wrong)))


@pytest.mark.parametrize("prefix", [0, 90])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim,heads,news,lens,max_q", [
    (64, 8, [3, 1, 2], [20, 9, 2], 2),          # the kernel for few rows, one part without a prefix
    (96, 4, [40, 7], [300, 7], 12),             # several chunks of own keys
    (128, 16, [150, 40], [150, 210], 70),       # the tcgen05 kernel, one part without a prefix
    (64, 16, [200, 3, 0, 90], [700, 3, 5, 90], 128),
])
def test_more_tokens_than_max_q_len(dim, heads, news, lens, max_q, causal, prefix):
    """The first max_q_len tokens of a sequence see what they see without the bound; the others,
    and tokens that no sequence holds, see nothing: zeros, and -inf in lse."""
    b = Batch(news, lens, prefix, heads, 2, dim, 16, BF16, seed=7)
    whole, whole_lse = b.run(lse=True, causal=causal)
    b.check(whole, whole_lse, causal=causal)
    head, tail = 3, 5  # tokens before the first sequence and after the last one
    q = torch.cat((normal(gen(1), head, heads, dim, dtype=BF16), b.q, normal(gen(2), tail, heads, dim, dtype=BF16)))
    indptr = b.q_indptr + head
    out = torch.full_like(q, math.nan)
    lse = torch.full(q.shape[:2], math.nan, device="cuda")
    P.prefix_attention(q, b.cache, b.table, b.seq_len, prefix_pages=b.prefix_pages, prefix_len=prefix, q_indptr=indptr,
                       max_q_len=max_q, causal=causal, out=out, lse=lse)
    held = torch.zeros(q.shape[0], dtype=torch.bool, device="cuda")
    for first, n in zip(indptr[:-1].tolist(), news):
        held[first:first + min(n, max_q)] = True
    inside = held[head:head + sum(news)]
    got = torch.where(inside[:, None, None], out[head:head + sum(news)], whole)
    b.check(got, torch.where(inside[:, None], lse[head:head + sum(news)], whole_lse), causal=causal)
    assert bool((out[~held] == 0).all()) and bool((lse[~held] == -math.inf).all())


@pytest.mark.parametrize("dim,n,max_q", [(64, 3, 4), (128, 150, 160), (256, 3, 4)])
@pytest.mark.parametrize("own", [True, False])
def test_tokens_past_the_last_sequence(dim, n, max_q, own):
    """A padded batch, with a prefix alone and with own pages alone."""
    b = Batch([n, 2], [n, 2] if own else [0, 0], 0 if own else 40, 8, 2, dim, 16, F16, seed=3)
    pad = 700
    q = torch.cat((b.q, normal(gen(1), pad, 8, dim, dtype=F16)))
    for causal in (True, False):
        out, lse = torch.full_like(q, math.nan), torch.full(q.shape[:2], math.nan, device="cuda")
        P.prefix_attention(q, b.cache, b.table, b.seq_len, prefix_pages=b.prefix_pages, prefix_len=b.prefix,
                           q_indptr=b.q_indptr, max_q_len=max_q, max_seq_len=max(b.lens), causal=causal, out=out, lse=lse)
        b.check(out[:n + 2], lse[:n + 2], causal=causal)
        assert bool((out[n + 2:] == 0).all()) and bool((lse[n + 2:] == -math.inf).all())


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_many_small_weights_beside_a_large_one(dtype, many):
    """One key takes nearly all of the softmax, and all others 2^-26 of it each: together, they are
    what the output is made of (their values are 8, the large key's are 0).  A weight rounded to
    float16 beside a largest weight of 1 would be lost, being below half of the type's smallest
    number.  The kernels keep the largest weight of a part at 2^7 or above in float16, so that what
    rounding to a multiple of 2^-24 may cost is keys * 2^-32 of the largest value."""
    heads, dim, page = 64, 64, 256
    gap = 26 * math.log(2.0)
    if many:  # one CTA a pair of head and row tile goes over all of the prefix
        rows, prefix, own = 300, 65536, 0
    else:     # as many (sequence, head) pairs as fill the GPU: few and long chunks of own keys
        rows, prefix, own = 40, 0, 65536
    pages = 65536 // page
    k = torch.zeros(pages, page, heads, dim, dtype=dtype, device="cuda")
    v = torch.full_like(k, 8.0)
    k[0, 0, :, 0] = 16.0
    v[0, 0] = 0.0
    q = torch.zeros(rows, heads, dim, dtype=dtype, device="cuda")
    q[..., 0] = 16.0
    ids = torch.arange(pages, device="cuda")
    if many:
        table = P.PageTable(torch.zeros(rows + 1, dtype=torch.int64, device="cuda"), ids[:0])
        named = dict(prefix_pages=ids, prefix_len=prefix)
    else:     # all sequences list the same pages
        table = P.PageTable(torch.arange(rows + 1, device="cuda") * pages, ids.repeat(rows))
        named = dict(max_seq_len=own)
    seq_len = torch.full((rows,), own, device="cuda")
    out, lse = P.prefix_attention(q, P.PagedKV(k, v), table, seq_len, scale=gap / 256, lse=True, **named)
    w = 65535 * 2.0 ** -26
    ref = 8 * w / (1 + w)
    u, e = U[dtype], 2.0 ** -18 * (1 + gap)
    tol = u * ref + (u + 4 * e) * ref + (2.0 ** -25 + 65536 * 2.0 ** -32 * 8 if dtype == F16 else 0)
    assert float((out.double() - ref).abs().max()) <= tol
    assert float((lse.double() - (gap + math.log1p(w))).abs().max()) <= 4 * e


def test_strides_of_dimensions_of_one():
    """Nothing is multiplied by the stride of a dimension of one, so it may be anything: one token or
    one page cut out of a buffer whose rows are off the 16-byte grid."""
    b = Batch([1], [11], 20, 4, 1, 64, 32, BF16, seed=6)
    q, out = (torch.zeros(5, 259, dtype=BF16, device="cuda")[:, :256].unflatten(1, (4, 64))[:1] for _ in range(2))
    q.copy_(b.q)
    b.q = q
    assert q.stride() == (259, 64, 1)
    assert b.run(out=out) is out
    b.check(out)
    lone = Batch([2], [11], 0, 1, 1, 64, 32, BF16, seed=6, spare=0)
    assert lone.cache.pages == 1
    odd = [torch.as_strided(x, x.shape, (x.stride(0) + 1, 64, 3, 1)) for x in (lone.cache.k, lone.cache.v)]
    lone.cache = P.PagedKV(*odd)
    lone.q = torch.as_strided(lone.q, lone.q.shape, (64, 5, 1))
    lone.check(lone.run())
    r = P.Rope(P.rope_frequencies(64))
    pos = torch.tensor([9], device="cuda")
    check_rotated(P.rope(q, r, pos), *rotate64(q, pos, r), BF16)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [1, 6, 7, 130])
@pytest.mark.parametrize("news,lens,prefix", [([150, 129, 1], [150, 400, 90], 333), ([90, 70], [290, 71], 0), ([1] * 50, [9] * 50, 300)])
def test_pages_with_few_rows_in_common_with_a_tile(news, lens, prefix, page, dim, dtype):
    """The tcgen05 kernel with 64 or 128 boxes a tile of 128 keys, lengths that end inside one, and
    pages outside the cache, which read as zeros."""
    b = Batch(news, lens, prefix, 8, 2, dim, page, dtype, seed=page)
    out, lse = b.run(lse=True)
    b.check(out, lse)
    bad = b.table.indices.clone()
    bad[0] = b.cache.pages
    b.table = P.PageTable(b.table.indptr, bad)
    for x in b.own[0]:
        x[:page] = 0
    if prefix:
        b.prefix_pages = b.prefix_pages.clone()
        b.prefix_pages[2] = -1
        for x in b.shared:
            x[2 * page:3 * page] = 0
    b.check(b.run())


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("news,lens,page,dim,rot,layout,heads_first", [
    ([1], [1], 1, 64, 64, "half", False),
    ([1] * 5, [1, 16, 17, 40, 9], 16, 128, 128, "half", False),
    ([1, 1], [9, 8], 8, 96, 48, "interleaved", True),
    ([3, 0, 50, 1], [3, 7, 70, 33], 24, 128, 64, "interleaved", False),
    ([700], [900], 64, 64, 64, "half", True),
    ([5, 2], [5, 9], 16, 36, 10, "half", False),
    ([20, 9], [30, 9], 7, 80, 0, "half", False),
])
def test_append(news, lens, page, dim, rot, layout, heads_first, dtype):
    b = Batch(news, lens, 0, 6, 2, dim, page, dtype, seed=dim, heads_first=heads_first)
    g = gen(1)
    t = sum(news)
    kv = normal(g, t, 2 * 2, dim, dtype=dtype)
    k, v = kv[:, :2], kv[:, 2:]
    r = P.Rope(P.rope_frequencies(rot), layout, 1.5)
    before = b.cache.k.clone(), b.cache.v.clone()
    base = 1000
    kw = {} if all(n == 1 for n in news) else {"q_indptr": b.q_indptr}
    q = P.kv_append(b.cache, b.table, b.seq_len, k, v, rope=r, q=b.q, position_base=base, **kw)
    at = torch.cat([torch.arange(l - n, l) for n, l in zip(news, lens)]).cuda()
    check_rotated(q, *rotate64(b.q, at + base, r), dtype)
    pages = torch.cat([torch.tensor(row, dtype=torch.int64)[torch.arange(l - n, l) // page]
                       for row, n, l in zip(b.rows, news, lens)]).cuda()
    got = b.cache.k[pages, at % page]
    check_rotated(got, *rotate64(k, at + base, r), dtype)
    assert torch.equal(b.cache.v[pages, at % page], v)
    # nothing else was written
    for now, old in zip((b.cache.k, b.cache.v), before):
        now[pages, at % page] = old[pages, at % page]
        assert torch.equal(now.nan_to_num(9.0), old.nan_to_num(9.0))
    # positions of the caller, in place, and without a rotation
    pos = torch.randint(0, 9999, (t,), generator=g, device="cuda")
    q2 = b.q.clone()
    assert P.kv_append(b.cache, b.table, b.seq_len, k, v, rope=r, q=q2, q_out=q2, positions=pos, **kw) is q2
    check_rotated(q2, *rotate64(b.q, pos, r), dtype)
    assert P.kv_append(b.cache, b.table, b.seq_len, k, v, **kw) is None
    assert torch.equal(b.cache.k[pages, at % page], k)


def test_append_drops_what_has_no_slot():
    """Lengths beyond the listed pages, pages outside the cache, tokens before slot 0."""
    b = Batch([1, 1, 3, 1], [5, 20, 2, 16], 0, 4, 2, 64, 16, BF16)
    before = b.cache.k.clone()
    bad = b.table.indices.clone()
    bad[0], bad[-1] = b.cache.pages, -7
    lens = torch.tensor([5, 33, 2, 16], device="cuda")
    k = normal(gen(0), 6, 2, 64, dtype=BF16)
    P.kv_append(b.cache, P.PageTable(b.table.indptr, bad), lens, k, k, q_indptr=b.q_indptr)
    page = b.rows[2][0]
    assert torch.equal(b.cache.k[page, 0], k[3]) and torch.equal(b.cache.k[page, 1], k[4])  # token 2 of 3 has slot 0
    b.cache.k[page, :2] = before[page, :2]
    assert torch.equal(b.cache.k.nan_to_num(9.0), before.nan_to_num(9.0))


def test_append_refusals():
    b = Batch([1, 1], [5, 6], 0, 4, 2, 64, 16, BF16)
    k = normal(gen(0), 2, 2, 64, dtype=BF16)
    r = P.Rope(P.rope_frequencies(64))
    for bad in (lambda: P.kv_append(b.cache, b.table, b.seq_len, k[:1], k[:1]), lambda: P.kv_append(b.cache, b.table, b.seq_len, k, k[:, :1]),
                lambda: P.kv_append(b.cache, b.table, b.seq_len, k.float(), k.float()),
                lambda: P.kv_append(b.cache, b.table, b.seq_len, k, k, q_out=b.q),
                lambda: P.kv_append(b.cache, b.table, b.seq_len, k, k, rope=r, positions=b.seq_len[:1])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(lib.TgError):
        P.kv_append(b.cache, b.table, b.seq_len, k, k, rope=P.Rope(P.rope_frequencies(128)))


# ------------------------------------------------------------------ together
def test_prompts_then_decoding_steps():
    """The prefix and the prompts are appended and attended to, then two decoding steps; each is
    compared with attention over the plainly rotated keys."""
    g = gen(21)
    kvh, heads, dim, page, prefix = 2, 8, 64, 16, 75
    r = P.Rope(P.rope_frequencies(dim, scaling="linear", factor=2.0))
    lens = [9, 30, 1]
    per = [4, 5, 3]
    ids = torch.randperm(40, generator=g, device="cuda").tolist()
    pre, own = ids[:5], [ids[5:5 + per[0]], ids[10:10 + per[1]], ids[20:20 + per[2]]]
    cache = P.PagedKV(*(torch.full((40, page, kvh, dim), math.nan, dtype=BF16, device="cuda") for _ in range(2)))
    k, v = normal(g, prefix, kvh, dim, dtype=BF16), normal(g, prefix, kvh, dim, dtype=BF16)
    P.kv_append(cache, P.PageTable.from_lists([pre]), torch.tensor([prefix], device="cuda"), k, v, rope=r,
                q_indptr=torch.tensor([0, prefix], device="cuda"))
    shared = [P.rope(k, r, torch.arange(prefix, device="cuda")), v]
    table = P.PageTable.from_lists(own)
    b = Batch([1], [1], 0, heads, kvh, dim, page, BF16)  # only its check() is used
    b.own, b.shared = [[torch.empty(0, kvh, dim, dtype=BF16, device="cuda")] * 2 for _ in lens], shared
    b.lens = [0] * 3
    for news in (lens, [1, 1, 1], [1, 1, 1]):
        b.news, b.lens = list(news), [x + y for x, y in zip(b.lens, news)]
        seq_len = torch.tensor(b.lens, device="cuda")
        indptr = torch.tensor([0] + b.news, device="cuda").cumsum(0)
        q, k, v = (normal(g, sum(news), h, dim, dtype=BF16) for h in (heads, kvh, kvh))
        q = P.kv_append(cache, table, seq_len, k, v, rope=r, q=q, position_base=prefix, q_indptr=indptr)
        pos = torch.cat([torch.arange(l - n, l, device="cuda") + prefix for n, l in zip(news, b.lens)])
        kr, t0 = P.rope(k, r, pos), 0
        for s, n in enumerate(news):
            b.own[s] = [torch.cat((b.own[s][0], kr[t0:t0 + n])), torch.cat((b.own[s][1], v[t0:t0 + n]))]
            t0 += n
        b.q = q
        b.check(P.prefix_attention(q, cache, table, seq_len, prefix_pages=torch.tensor(pre, device="cuda"), prefix_len=prefix,
                                   q_indptr=indptr, max_q_len=max(news)))


@pytest.mark.parametrize("kw", [dict(batch=5, prefix=100, steps=3), dict(batch=40, prefix=515, steps=20, prompt=(1, 30)),
                                dict(batch=2, prefix=1, steps=2, heads=8, kv_heads=8, dim=128, page=8)])
def test_the_decoding_example(kw):
    """Three 16-bit roundings of the block's output (projections, attention, sum): 4 half ulps."""
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "shared_prefix_decode.py")
    spec = importlib.util.spec_from_file_location("shared_prefix_decode", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    assert example.check(*example.generate(**kw)) < 4 * U[BF16]
