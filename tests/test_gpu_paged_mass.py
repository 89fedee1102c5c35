"""The attention weight that cached keys gather, against a plain implementation in 64 bits, with the
log-sum-exp that the attention left.

Bound, derived before the first run: a weight p = exp(s - lse) has a relative error of at most
2 e + 2^-22 |lse| + 2^-20 (e = 2^-18 (1 + scale sum_d |q_d k_d|): the score's 32-bit sum; lse's product
with log2 e; the exponential), and the sum over n rows one of (n / 4 + 64) 2^-24 more.  The old weight's
product and the last addition: 2^-22 of the result's terms.
"""

from __future__ import annotations

import math
import os
import subprocess
import sys

import pytest
import torch

from test_gpu_paged import ATTEND, BF16, F16, Batch, gen, normal
from tilegen_b200 import lib
from tilegen_b200 import paged as P

pytestmark = pytest.mark.gpu


class Weighed(Batch):
    """A batch with a mass: NaN where nothing may be read, kept apart to see what is written."""

    def __init__(self, *a, heads_last=False, **kw):
        super().__init__(*a, **kw)
        self.mass = P.empty_mass(self.cache)
        if heads_last:
            self.mass = self.mass.contiguous()
        self.mass.fill_(math.nan)
        g = gen(99)
        self.old = []
        for pages, n, length in zip(self.rows, self.news, self.lens):
            old = torch.rand(length, self.kv_heads, generator=g, device="cuda")
            old[max(length - n, 0):] = math.nan  # what the new tokens' slots held before
            self.old.append(old)
            for i, pg in enumerate(pages):
                part = old[i * self.page:(i + 1) * self.page]
                self.mass[pg, :part.shape[0]] = part
        self.before = self.mass.clone()

    def lse(self, **kw):
        return self.run(lse=True, **kw)[1]

    def gather(self, lse, decay=1.0, causal=True, scale=None, max_q=None, **kw):
        pos, named = self.args(**kw)
        named = {k: v for k, v in named.items() if not k.startswith("prefix")}
        out = P.attention_mass(self.mass, pos[0], *pos[1:], lse, causal=causal, decay=decay, scale=scale, **named)
        assert out is self.mass

    def check(self, lse, decay=1.0, causal=True, scale=None, asked=None):
        scale = self.dim ** -0.5 if scale is None else scale
        t0, want_all = 0, self.before.clone()
        for (k, _), old, pages, n, length in zip(self.own, self.old, self.rows, self.news, self.lens):
            k = k.double()
            q = self.q[t0:t0 + n].double().view(n, self.kv_heads, self.heads // self.kv_heads, self.dim)
            L = lse[t0:t0 + n].double().view(n, self.kv_heads, self.heads // self.kv_heads, 1)
            sc = torch.einsum("nhgd,khd->nhgk", q, k) * scale
            seen = torch.arange(length, device="cuda")[None] < length - n + 1 + torch.arange(n, device="cuda")[:, None]
            seen = (seen if causal else torch.ones_like(seen)) & (torch.arange(n, device="cuda") < (n if asked is None else asked))[:, None]
            seen = seen[:, None, None] & (L > -math.inf)
            p = torch.where(seen, (sc - L).exp(), 0.0)
            e = 2.0 ** -18 * (1 + torch.einsum("nhgd,khd->nhgk", q.abs(), k.abs()) * scale)
            rel = 2 * e + 2.0 ** -22 * L.abs() + 2.0 ** -20 + (n * p.shape[2] / 4 + 64) * 2.0 ** -24
            tol = torch.where(seen, p * rel, 0.0).sum((0, 2)).T
            gathered = p.sum((0, 2)).T  # [key, head]
            kept = old.double().clone()
            if causal:
                kept[max(length - n, 0):] = 0.0
            if decay == 0:
                kept[:] = 0.0
            ref = decay * kept + gathered
            tol += 2.0 ** -22 * (decay * kept + gathered)
            at = torch.arange(length, device="cuda")
            where = torch.tensor(pages, device="cuda", dtype=torch.int64)[at // self.page], at % self.page
            got = self.mass[where].double()
            ok = ref.isfinite()
            assert torch.equal(got.isfinite(), ok)
            err = (got - ref).abs()
            assert bool((err <= tol)[ok].all()), "worst %g of its bound" % float((err / tol)[ok].max())
            want_all[where] = self.mass[where]
            t0 += n
        # slots that no sequence holds are as they were
        assert torch.equal(want_all.nan_to_num(-7.0), self.mass.nan_to_num(-7.0))


MORE = [
    ([1, 1], [500, 1300], 40, 300, 1, 64, 16),     # more heads a key head than a row tile has rows
    ([3, 70], [50, 90], 0, 130, 1, 256, 16),
    ([2, 1], [77, 200], 0, 25, 5, 128, 16),        # groups that do not divide a tile
    ([700, 1], [900, 130], 0, 8, 2, 128, 32),      # several row tiles, shared out
    ([33, 1000], [40, 2100], 100, 6, 2, 64, 48),
    ([1] * 200, [200] * 200, 0, 8, 8, 64, 8),
    ([1, 1, 1], [1, 4000, 129], 0, 4, 2, 128, 6),  # 64 boxes a tile
    ([1] * 700, list(range(700)), 30, 8, 2, 64, 16),  # more sequences than one launch takes
    ([90] * 530, [90 + i % 70 for i in range(530)], 0, 4, 1, 64, 32),
    ([300, 90, 1], [700, 90, 400], 0, 4, 2, 256, 16),  # many rows of heads of 256 and 96, shared out
    ([600, 0, 31], [900, 300, 31], 50, 8, 2, 96, 24),
    ([400, 700], [100, 650], 0, 8, 2, 128, 16),    # more queries than keys, many rows
]
CASES = ATTEND + MORE


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_mass(case, dtype):
    b = Weighed(*CASES[case], dtype, seed=case)
    lse = b.lse()
    for kw in ({}, {"max_seq_len": max(b.lens)}):
        b.mass.copy_(b.before)
        b.gather(lse, 0.75, **kw)
        b.check(lse, 0.75)
    first = b.mass.clone()
    b.mass.copy_(b.before)
    b.gather(lse, 0.75, max_seq_len=max(b.lens))
    assert torch.equal(first.nan_to_num(-7.0), b.mass.nan_to_num(-7.0))  # the same twice


@pytest.mark.parametrize("case", [4, 8, 10, 14, 16, 20, 22, 23, 29, 30, 31])
def test_without_a_mask(case):
    b = Weighed(*CASES[case], BF16, seed=case)
    lse = b.lse(causal=False, scale=0.3)
    for old, pages in zip(b.old, b.rows):  # without a mask no token is new: all old weights count
        old.nan_to_num_(0.5)
        for i, pg in enumerate(pages):
            part = old[i * b.page:(i + 1) * b.page]
            b.mass[pg, :part.shape[0]] = part
    b.before = b.mass.clone()
    b.gather(lse, causal=False, scale=0.3)
    b.check(lse, causal=False, scale=0.3)


@pytest.mark.parametrize("case", [4, 9, 10, 17, 23])
def test_decay_of_zero_reads_nothing(case):
    b = Weighed(*CASES[case], BF16, seed=case)
    lse = b.lse()
    b.mass.fill_(math.nan)
    b.before = b.mass.clone()
    b.gather(lse, 0.0)
    b.check(lse, 0.0)


@pytest.mark.parametrize("case", [4, 8, 10, 13, 17, 20])
def test_strides(case):
    """A cache stored head by head, queries inside a joint projection or heads first, a mass with heads
    side by side and one inside a larger buffer."""
    b = Weighed(*CASES[case], BF16, seed=case, heads_first=True, heads_last=True)
    lse = b.lse()
    t, h, d = b.q.shape
    wide = torch.zeros(t, h + 3, d, dtype=BF16, device="cuda")
    wide[:, 1:h + 1] = b.q
    for q in (wide[:, 1:h + 1], b.q.transpose(0, 1).contiguous().transpose(0, 1)):
        b.q = q
        b.mass.copy_(b.before)
        b.gather(lse)
        b.check(lse)
    big = torch.full((b.cache.pages, b.page + 1, b.kv_heads, 3), 5.0, device="cuda")
    b.mass = big[:, :b.page, :, 1].copy_(b.before)
    b.gather(lse)
    b.check(lse)
    assert bool((big[..., 0] == 5).all()) and bool((big[:, b.page] == 5).all())


def test_the_weights_of_a_query_sum_to_one():
    """Without a prefix each row's weights sum to one; behind one, to the own keys' share."""
    b = Weighed([1] * 5, [1, 50, 128, 300, 2000], 0, 8, 2, 128, 16, BF16, seed=1)
    b.gather(b.lse(), 0.0)
    for pages, n in zip(b.rows, b.lens):
        total = sum(b.mass[pg, :min(b.page, n - i * b.page)].sum(0) for i, pg in enumerate(pages))
        assert bool(((total - 4).abs() < 4 * 2.0 ** -14).all())


def test_tokens_past_the_bound_and_rows_that_see_nothing():
    b = Weighed([5, 300, 2], [5, 310, 40], 0, 8, 2, 64, 16, BF16, seed=2)
    lse = b.lse()
    b.gather(lse, 0.5, max_q_len=3)
    b.check(lse, 0.5, asked=3)
    b.mass.copy_(b.before)
    lse[6:40] = -math.inf  # rows that saw nothing, by their lse
    b.gather(lse, 0.5)
    b.check(lse, 0.5)


def test_sequences_without_new_tokens_decay():
    b = Weighed([0, 2, 0], [130, 9, 5], 0, 8, 2, 64, 16, BF16, seed=2)
    lse = b.lse()
    b.gather(lse, 0.25)
    b.check(lse, 0.25)
    empty = Weighed([0, 0], [130, 9], 0, 8, 2, 64, 16, BF16, seed=2)
    empty.gather(torch.empty(0, 8, device="cuda"), 0.5, max_q_len=None)
    empty.check(torch.empty(0, 8, device="cuda"), 0.5)


def test_nan_and_infinite_keys_stay_their_own():
    """A key that is not finite spoils its own weight, a query that is not finite its own rows' keys; what
    lies behind a query's token does not reach it."""
    b = Weighed([40], [300], 0, 4, 1, 128, 16, BF16, seed=3)
    lse = b.lse()
    b.gather(lse)
    clean = b.mass.clone()
    row = b.rows[0]
    b.cache.k[row[2], 3, 0, 5] = math.nan
    b.cache.k[row[-1], 299 % 16, 0, 5] = math.inf  # only the last token sees it
    b.mass.copy_(b.before)
    b.gather(lse)
    bad = torch.zeros_like(clean, dtype=torch.bool)
    bad[row[2], 3] = bad[row[-1], 299 % 16] = True
    assert bool(b.mass[row[2], 3].isnan().all())
    assert torch.equal(b.mass[~bad].nan_to_num(-7.0), clean[~bad].nan_to_num(-7.0))


@pytest.mark.parametrize("page", [16, 7])
def test_pages_outside_the_cache(page):
    """Keys of pages that do not exist count as zeros and their weights are dropped; lengths are cut."""
    b = Weighed([1, 1], [200, 150], 0, 8, 2, 64, page, BF16, seed=3)
    lse = b.lse()
    bad = b.table.indices.clone()
    bad[1], bad[int(b.table.indptr[1]) + 2] = b.cache.pages + 3, -2
    table, b.table = b.table, P.PageTable(b.table.indptr, bad)
    b.seq_len = torch.tensor([10 ** 12, -4], device="cuda")
    b.gather(lse)
    changed = (b.mass != b.before) & ~(b.mass.isnan() & b.before.isnan())
    pages = set(changed.any(-1).any(-1).nonzero().flatten().tolist())
    assert pages <= set(b.rows[0]) - {b.rows[0][1]}
    with pytest.raises(lib.TgError) as e:
        b.gather(lse, check=True)
    assert e.value.status == lib.TG_EBOUNDS
    b.table = table


def test_offsets_beyond_32_bits():
    page, heads, dim = 64, 8, 128
    pages = (1 << 31) // (page * heads * dim) + 40
    b = Weighed([1, 2], [100, 130], 0, 16, heads, dim, page, BF16, seed=1)
    lse = b.lse()
    flat = torch.zeros(pages, page, heads, dim, dtype=BF16, device="cuda")
    moved = torch.arange(pages - b.cache.pages, pages, device="cuda")
    flat[moved] = b.cache.k
    b.cache = P.PagedKV(flat, flat)
    b.table = P.PageTable(b.table.indptr, moved[b.table.indices])
    far = torch.empty(pages, page, heads, 1 + (1 << 31) // (pages * page * heads), device="cuda")[..., 0]
    small, b.mass = b.mass, far
    far[moved] = small
    b.gather(lse)
    b.mass = far[moved]
    b.check(lse)


def test_queries_of_one_number_for_all_tokens():
    """Strides of zero, as an expanded tensor has them: taken or refused, never misread."""
    b = Weighed([1, 1], [200, 90], 0, 8, 2, 64, 16, BF16, seed=3)
    b.q = b.q[:1].expand(2, 8, 64)
    lse = b.lse()
    try:
        b.gather(lse)
    except lib.TgError as e:
        assert e.status == lib.TG_ECUDA and torch.equal(b.mass.nan_to_num(-7.0), b.before.nan_to_num(-7.0))
    else:
        b.check(lse)
    with pytest.raises(ValueError):  # one place for all heads
        P.attention_mass(b.mass[..., :1].expand(b.mass.shape), b.q.contiguous(), b.cache, b.table, b.seq_len, lse)


def test_graph_streams_and_workspace():
    b = Weighed(*MORE[3], BF16, seed=4)
    lse = b.lse()
    b.gather(lse, 0.5)
    want = b.mass.clone()
    pos, named = b.args()
    n = P.attention_mass_workspace_bytes(*pos, q_indptr=b.q_indptr, max_q_len=max(b.news))
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.gather(lse, 0.5, workspace=ws)
    for _ in range(2):
        b.mass.copy_(b.before)
        graph.replay()
        assert torch.equal(b.mass.nan_to_num(-7.0), want.nan_to_num(-7.0))
    b.mass.copy_(b.before)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    b.gather(lse, 0.5, stream=st)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(b.mass.nan_to_num(-7.0), want.nan_to_num(-7.0))


def test_refusals():
    b = Weighed([1, 1], [9, 3], 0, 4, 2, 64, 16, BF16)
    lse = b.lse()
    for bad in (lambda: b.gather(lse.double()), lambda: b.gather(lse[:1]), lambda: b.gather(lse.T.contiguous().T),
                lambda: P.attention_mass(b.mass[:2], b.q, b.cache, b.table, b.seq_len, lse),
                lambda: P.attention_mass(b.mass.half(), b.q, b.cache, b.table, b.seq_len, lse),
                lambda: P.attention_mass(b.mass, b.q[:1], b.cache, b.table, b.seq_len, lse),
                lambda: P.attention_mass(b.mass, b.q.float(), b.cache, b.table, b.seq_len, lse)):
        with pytest.raises(ValueError):
            bad()
    for bad, status in ((lambda: b.gather(lse, -0.5), lib.TG_EINVAL), (lambda: b.gather(lse, math.nan), lib.TG_EINVAL),
                        (lambda: b.gather(lse, scale=0.0), lib.TG_EINVAL), (lambda: b.gather(lse, max_seq_len=-1), lib.TG_EINVAL)):
        with pytest.raises(lib.TgError) as e:
            bad()
        assert e.value.status == status
    off = torch.empty(2 * 4 * 64 + 1, dtype=BF16, device="cuda")[1:].view(2, 4, 64)
    with pytest.raises(lib.TgError) as e:
        P.attention_mass(b.mass, off, b.cache, b.table, b.seq_len, lse)
    assert e.value.status == lib.TG_EINVAL
    wide = Weighed([1], [9], 0, 4, 2, 64, 16, BF16)
    cache = P.PagedKV(torch.zeros(4, 16, 2, 80, dtype=BF16, device="cuda"), torch.zeros(4, 16, 2, 80, dtype=BF16, device="cuda"))
    with pytest.raises(lib.TgError) as e:
        P.attention_mass(P.empty_mass(cache), torch.zeros(1, 4, 80, dtype=BF16, device="cuda"), cache, wide.table, wide.seq_len, lse[:1])
    assert e.value.status == lib.TG_EUNSUPPORTED


def test_a_workspace_kept_by_a_small_batch_serves_a_long_prompt():
    """Asked for with one token, with and without a q_indptr; then parts of one long prompt are kept in it."""
    small = Weighed([1], [9], 0, 32, 8, 128, 16, BF16, seed=1)
    pos, _ = small.args()
    n = P.attention_mass_workspace_bytes(*pos, max_q_len=2048)
    starts = torch.tensor([0, 1], device="cuda")
    assert n == P.attention_mass_workspace_bytes(*pos, q_indptr=starts, max_q_len=2048) > 0
    assert P.attention_mass_workspace_bytes(*pos) == P.attention_mass_workspace_bytes(*pos, q_indptr=starts) == 0
    ws = torch.full((n,), 255, dtype=torch.uint8, device="cuda")
    b = Weighed([2048, 1], [2100, 50], 0, 32, 8, 128, 16, BF16, seed=2)
    lse = b.lse()
    b.gather(lse, 0.5, workspace=ws)
    b.check(lse, 0.5)
    small.gather(small.lse(), workspace=ws)


GIVE_UP = [
    ([1] * 5, [1, 50, 128, 300, 2000], 40, 8, 2, 128, 16),
    ([32, 7], [3000, 90], 0, 8, 1, 64, 16),                  # two halves of rows
    ([700, 1], [900, 130], 0, 8, 2, 128, 32),                # parts that are joined
    ([90] * 530, [90 + i % 70 for i in range(530)], 0, 4, 1, 64, 32),  # more sequences than one launch takes
    ([2, 1], [77, 200], 0, 300, 1, 256, 16),                 # several row tiles a token
    ([300, 9], [700, 1900], 0, 16, 8, 96, 24),
]


def test_a_wait_that_runs_out_leaves_nan():
    """Where a wait has run out (here: as if at once, in every CTA) no key keeps a number that may be wrong,
    and nothing else is written."""
    code = """
import sys
sys.path[:0] = %r
from test_gpu_paged_mass import *
for case, shape in enumerate(GIVE_UP):
    for dtype in (BF16, F16):
        b = Weighed(*shape, dtype, seed=case)
        lse = b.lse()
        for decay in (0.5, 0.0):
            b.mass.copy_(b.before.nan_to_num(3.0))
            b.gather(lse, decay, max_seq_len=max(b.lens))
            want = b.before.nan_to_num(3.0)
            for pages, length in zip(b.rows, b.lens):
                at = torch.arange(length, device="cuda")
                want[torch.tensor(pages, device="cuda")[at // b.page], at %% b.page] = math.nan
            assert torch.equal(b.mass.nan_to_num(-7.0), want.nan_to_num(-7.0)), (case, dtype, decay)
print("all", len(GIVE_UP))
""" % [os.path.dirname(os.path.abspath(__file__)), os.path.dirname(os.path.dirname(os.path.abspath(__file__)))]
    r = subprocess.run([sys.executable, "-c", code], env={**os.environ, "TG_MASS_WAIT_MS": "0"}, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "all %d" % len(GIVE_UP) in r.stdout, r.stdout + r.stderr


def test_a_unit_may_take_longer_than_a_wait():
    """4000 tokens of 256 heads a key head pass 512 keys, 20 milliseconds for a CTA's unit, of which it has
    several: with a limit of five milliseconds nothing runs out, as all waits but those for a whole unit are
    microseconds.  The bound is that of the other cases, for 1024000 rows."""
    code = """
import sys
sys.path[:0] = %r
from test_gpu_paged_mass import *
n, kvh, group, dim, keys, page, batch = 4000, 8, 256, 64, 512, 32, 40
g = gen(7)
pages = batch * keys // page
cache = P.PagedKV(normal(g, pages, page, kvh, dim, dtype=BF16), None)
cache.v = cache.k
table = P.PageTable.from_lists([list(range(b * keys // page, (b + 1) * keys // page)) for b in range(batch)])
news = [0 if b %% 5 == 1 else n for b in range(batch)]
starts = torch.tensor([0] + news, device="cuda").cumsum(0)
one = normal(g, 1, kvh * group, dim, dtype=BF16)
sc = torch.einsum("xhgd,bkhd->bhgk", one.double().view(1, kvh, group, dim), cache.k.double().view(batch, keys, kvh, dim)) * dim ** -0.5
lse = sc.logsumexp(-1).float()  # [sequence, key head, head]
rows = lse.flatten(1).repeat_interleave(torch.tensor(news, device="cuda"), 0).contiguous()
mass = P.empty_mass(cache).fill_(2.0)
lens = torch.full((batch,), keys, device="cuda")
P.attention_mass(mass, one.expand(sum(news), kvh * group, dim), cache, table, lens, rows, q_indptr=starts, max_q_len=n,
                 max_seq_len=keys, causal=False, decay=0.5)
p = (sc - lse.double()[..., None]).exp()
e = 2.0 ** -18 * (1 + torch.einsum("xhgd,bkhd->bhgk", one.double().abs().view(1, kvh, group, dim),
                                   cache.k.double().abs().view(batch, keys, kvh, dim)) * dim ** -0.5)
rel = 2 * e + 2.0 ** -22 * lse.double().abs()[..., None] + 2.0 ** -20 + (n * group / 4 + 64) * 2.0 ** -24
count = torch.tensor(news, device="cuda", dtype=torch.float64)[:, None, None]
gathered, tol = p.sum(2) * count, (p * rel).sum(2) * count
got = mass.double().reshape(batch, keys, kvh).transpose(1, 2)
err, tol = (got - gathered - 1.0).abs(), tol + 2.0 ** -22 * (gathered + 1.0)
assert bool(got.isfinite().all()), int(got.isnan().sum())
assert bool((err <= tol).all()), float((err / tol).max())
print("all", batch)
""" % [os.path.dirname(os.path.abspath(__file__)), os.path.dirname(os.path.dirname(os.path.abspath(__file__)))]
    r = subprocess.run([sys.executable, "-c", code], env={**os.environ, "TG_MASS_WAIT_MS": "5"}, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "all 40" in r.stdout, r.stdout + r.stderr


@pytest.mark.parametrize("case", [0, 3])
@pytest.mark.parametrize("how", ["tokens", "heads", "both", "overlapping"])
def test_queries_of_any_strides(how, case):
    """Expanded queries and rows that overlap are taken as they are, as the attention takes them."""
    b = Weighed(*MORE[case], BF16, seed=6)
    t, h, d = b.q.shape
    b.q = {"tokens": lambda q: q[:1].expand(t, h, d), "heads": lambda q: q[:, :1].expand(t, h, d),
           "both": lambda q: q[:1, :1].expand(t, h, d), "overlapping": lambda q: torch.as_strided(q, (t, h, d), (d, d, 1))}[how](b.q)
    lse = b.lse()
    b.gather(lse, 0.5)
    b.check(lse, 0.5)
