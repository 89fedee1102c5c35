"""Eviction from a paged cache against a plain implementation, place by place.  Everything is moved or
compared, nothing computed: results are equal bit for bit."""

from __future__ import annotations

import math

import pytest
import torch

from tilegen_b200 import lib
from tilegen_b200 import paged as P

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


class Cache:
    """Sequences of `lens` keys on pages in random order, some pages spare."""

    def __init__(self, lens, heads, dim, page, dtype, seed=0, heads_first=False, levels=0, mass_first=True):
        g = gen(seed)
        self.lens, self.page, self.heads = lens, page, heads
        own = [-(-n // page) for n in lens]
        total = sum(own) + 3
        order = torch.randperm(total, generator=g, device="cuda").tolist()
        self.rows = [[order.pop() for _ in range(n)] for n in own]
        self.table = P.PageTable.from_lists(self.rows)
        shape = (total, heads, page, dim) if heads_first else (total, page, heads, dim)
        k, v = (torch.randn(shape, generator=g, device="cuda").to(dtype) for _ in range(2))
        if heads_first:
            k, v = k.transpose(1, 2), v.transpose(1, 2)
        self.cache = P.PagedKV(k, v)
        self.mass = P.empty_mass(self.cache) if mass_first else torch.zeros(total, page, heads, device="cuda")
        x = torch.randn(self.mass.shape, generator=g, device="cuda")
        # levels: so many different weights, else hardly two alike
        self.mass.copy_((x * levels / 4).round() if levels else (2 * x).exp())
        self.seq_len = torch.tensor(lens, dtype=torch.int64, device="cuda")

    def tensors(self):
        return self.cache.k, self.cache.v, self.mass

    def sources(self, budget, first, recent):
        """[sequence][head] -> the old place of each new one."""
        out = []
        for pages, length in zip(self.rows, self.lens):
            size = min(length, budget)
            last = min(recent, size)
            lead = min(first, size - last)
            heavy = size - last - lead
            at = torch.arange(length, device="cuda")
            heads = []
            for h in range(self.heads):
                source = at[:size].clone()
                if length > size:
                    where = torch.tensor(pages, device="cuda")[at // self.page], at % self.page, torch.full_like(at, h)
                    m = self.mass[where][lead:length - last]
                    # NaN before all, then by weight (-0 is 0), then by place
                    order = sorted(range(m.numel()), key=lambda i, x=m.tolist(): (not math.isnan(x[i]), -x[i] if not math.isnan(x[i]) else 0.0, i))
                    chosen = sorted(lead + i for i in order[:heavy])
                    stay = [c for c in chosen if c < lead + heavy]
                    move = [c for c in chosen if c >= lead + heavy]
                    free = sorted(set(range(lead, lead + heavy)) - set(stay))
                    source[torch.tensor(free, dtype=torch.int64, device="cuda")] = torch.tensor(move, dtype=torch.int64, device="cuda")
                    source[lead + heavy:] = at[length - last:]
                heads.append(source)
            out.append(heads)
        return out

    def check(self, budget, first, recent, separate=False, **kw):
        sources = self.sources(budget, first, recent)
        k, v, mass = (x.clone() for x in self.tensors())
        want = [x.clone() for x in (k, v, mass)]
        loose = torch.zeros(mass.shape, dtype=torch.bool, device="cuda")  # behind the new length: anything
        for pages, length, heads in zip(self.rows, self.lens, sources):
            to = torch.tensor(pages, dtype=torch.int64, device="cuda")
            for h, source in enumerate(heads):
                at = torch.arange(source.numel(), device="cuda")
                for x, y in zip((k, v, mass), want):
                    y[to[at // self.page], at % self.page, h] = x[to[source // self.page], source % self.page, h]
                rest = torch.arange(source.numel(), length, device="cuda")
                loose[to[rest // self.page], rest % self.page, h] = True
        out = torch.full_like(self.mass, -7.0) if separate else None
        got_len, kept = P.kv_evict(self.cache, self.table, self.seq_len, self.mass, budget, first=first, recent=recent, kept=True,
                                   mass_out=out, **kw)
        assert got_len.tolist() == [min(n, budget) for n in self.lens]
        for b, heads in enumerate(sources):
            for h, source in enumerate(heads):
                row = kept[b, h]
                assert torch.equal(row[:source.numel()].long(), source), (b, h)
                assert bool((row[source.numel():] == -1).all())
        for x, y in zip(self.tensors(), want):
            if separate and x is self.mass:
                assert torch.equal(x.nan_to_num(9.0), mass.nan_to_num(9.0))
                continue
            hide = loose if x.dim() == 3 else loose[..., None].expand(x.shape)
            assert torch.equal(x.masked_fill(hide, 0).nan_to_num(9.0), y.masked_fill(hide, 0).nan_to_num(9.0))
        if separate:  # the kept keys' weights and nothing else
            alone = torch.full_like(out, -7.0)
            for pages, heads in zip(self.rows, sources):
                to = torch.tensor(pages, dtype=torch.int64, device="cuda")
                for h, source in enumerate(heads):
                    at = torch.arange(source.numel(), device="cuda")
                    alone[to[at // self.page], at % self.page, h] = mass[to[source // self.page], source % self.page, h]
            assert torch.equal(out.nan_to_num(9.0), alone.nan_to_num(9.0))
        return got_len, kept


CASES = [  # lens, heads, dim, page; budget, first, recent
    (([1], 1, 64, 16), (1, 0, 0)),
    (([2, 0, 1], 2, 64, 16), (1, 0, 0)),
    (([5, 9, 3], 2, 64, 16), (4, 1, 1)),
    (([300, 20, 129], 2, 128, 16), (100, 4, 16)),
    (([300, 20, 129], 2, 128, 16), (100, 0, 0)),
    (([300, 280], 2, 128, 7), (270, 4, 200)),      # recent keys overlap their new places
    (([300, 301, 302], 1, 96, 24), (299, 1, 250)),
    (([300, 90], 3, 64, 1), (60, 50, 40)),         # first and recent alone are more
    (([300, 90], 3, 64, 8), (60, 50, 10)),         # exactly the budget
    (([300, 90], 3, 64, 8), (60, 0, 100)),
    (([300, 90], 3, 64, 8), (0, 3, 3)),            # nothing is kept
    (([2100, 4000, 17], 4, 64, 32), (1000, 4, 300)),
    (([9000], 2, 64, 16), (2500, 4, 32)),
    (([20000, 31], 1, 64, 64), (19999, 4, 9000)),  # all but one, a long list in order
    (([1100] * 40, 8, 16, 16), (1024, 4, 64)),
    (([70, 300], 2, 5, 16), (50, 2, 9)),           # rows of 10 bytes
    (([70, 300], 2, 6, 16), (50, 2, 9)),           # rows of 12 bytes
    (([150, 300], 1, 2048, 8), (50, 2, 9)),        # rows longer than a CTA
]


@pytest.mark.parametrize("separate", [False, True])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_evict(case, separate):
    what, cut = CASES[case]
    Cache(*what, (BF16, F16, F32)[case % 3], seed=case).check(*cut, separate=separate)
    c = Cache(*what, F32 if case % 2 else F16, seed=case, heads_first=True, mass_first=False)
    c.check(*cut, separate=separate, max_seq_len=max(c.lens), check=True)


@pytest.mark.parametrize("levels", [1, 2, 40])
@pytest.mark.parametrize("case", [2, 3, 5, 7, 11, 12, 14])
def test_ties_go_to_the_lowest_place(case, levels):
    """Weights of a few values, zeros of both signs and negative ones among them."""
    what, cut = CASES[case]
    c = Cache(*what, F16, seed=case, levels=levels)
    c.mass[c.mass == 0] *= torch.where(torch.rand(int((c.mass == 0).sum()), generator=gen(1), device="cuda") < 0.5, -1.0, 1.0)
    c.check(*cut)


def test_all_weights_alike_and_weights_that_are_no_numbers():
    for value in (0.0, 1.0, math.inf, -math.inf, math.nan):
        c = Cache([500, 1300], 2, 64, 16, BF16, seed=3)
        c.mass.fill_(value)
        c.check(400, 2, 30)
    c = Cache([500, 1300], 2, 64, 16, BF16, seed=3)
    pick = torch.rand(c.mass.shape, generator=gen(2), device="cuda")
    c.mass[pick < 0.1] = math.nan
    c.mass[(pick > 0.1) & (pick < 0.2)] = -math.nan
    c.mass[(pick > 0.2) & (pick < 0.3)] = math.inf
    c.mass[(pick > 0.3) & (pick < 0.4)] = -math.inf
    c.mass[(pick > 0.4) & (pick < 0.5)] = 1e-42  # below the normal range
    c.check(400, 2, 30)


@pytest.mark.parametrize("levels", [0, 3])
@pytest.mark.parametrize("lens,budget,recent", [([130000], 20000, 64), ([350000, 9], 300000, 5000), ([70000, 60000], 6000, 3000)])
def test_long_sequences(lens, budget, recent, levels):
    """Clusters of CTAs, weights that do not fit in shared memory, long lists, thousands of equal weights."""
    c = Cache(lens, 1, 8, 64, BF16, seed=5, levels=levels)
    k, v, mass = (x.clone() for x in c.tensors())
    got_len, kept = P.kv_evict(c.cache, c.table, c.seq_len, c.mass, budget, first=4, recent=recent, kept=True,
                               max_seq_len=max(lens))
    assert got_len.tolist() == [min(n, budget) for n in lens]
    for b, length in enumerate(lens):
        size = min(length, budget)
        at = torch.arange(length, device="cuda")
        pages = torch.tensor(c.rows[b], device="cuda")
        where = pages[at // 64], at % 64, torch.zeros_like(at)
        m = mass[where]
        source = at[:size].clone()
        if length > size:
            heavy, end = size - recent - 4, size - recent
            order = torch.sort(m[4:length - recent], descending=True, stable=True).indices[:heavy] + 4
            chosen = torch.zeros(length, dtype=torch.bool, device="cuda")
            chosen[order] = True
            free = (~chosen[4:end]).nonzero().flatten() + 4
            source[free] = chosen[end:].nonzero().flatten() + end
            source[end:] = at[length - recent:]
        assert torch.equal(kept[b, 0, :size].long(), source)
        to, old = tuple(w[:size] for w in where), tuple(w[source] for w in where)
        for x, y in zip((k, v, mass), c.tensors()):
            assert torch.equal(y[to], x[old])


def test_again_and_again():
    """Steps of a server: keys are appended, the longest sequences are cut, lengths in place."""
    g = gen(8)
    c = Cache([200, 230, 100], 2, 64, 16, BF16, seed=8)
    c.rows = [list(range(i * 16, (i + 1) * 16)) for i in range(3)]
    k = torch.randn(48, 16, 2, 64, generator=g, device="cuda").to(BF16)
    c.cache = P.PagedKV(k, k.clone())
    c.mass = P.empty_mass(c.cache).copy_(torch.rand(48, 16, 2, generator=g, device="cuda"))
    c.table = P.PageTable.from_lists(c.rows)
    for step in range(6):
        c.lens = [min(n + 7, 256) for n in c.lens]
        c.seq_len += 7
        c.seq_len.clamp_(max=256)
        got, _ = c.check(210, 4, 50, seq_len_out=c.seq_len)
        assert got is c.seq_len
        c.lens = got.tolist()


def test_offsets_beyond_32_bits():
    page, heads, dim = 64, 8, 128
    pages = (1 << 31) // (page * heads * dim) + 40
    c = Cache([500, 700], heads, dim, page, BF16, seed=1)
    moved = torch.arange(pages - c.cache.pages, pages, device="cuda")
    big = [torch.zeros(pages, page, heads, dim, dtype=BF16, device="cuda") for _ in range(2)]
    for x, y in zip(big, (c.cache.k, c.cache.v)):
        x[moved] = y
    mass = torch.zeros(pages, page, heads, device="cuda")
    mass[moved] = c.mass
    small = Cache([500, 700], heads, dim, page, BF16, seed=1)
    want = P.kv_evict(small.cache, small.table, small.seq_len, small.mass, 300, 4, 20)
    got = P.kv_evict(P.PagedKV(*big), P.PageTable(c.table.indptr, moved[c.table.indices]), c.seq_len, mass, 300, 4, 20)
    assert torch.equal(got, want)
    assert torch.equal(big[0][moved], small.cache.k) and torch.equal(big[1][moved], small.cache.v)
    assert torch.equal(mass[moved], small.mass)


def test_bad_pages_and_lengths():
    """Pages that do not exist read as zeros, writes to them are dropped, lengths are cut."""
    c = Cache([300, 200, 90], 2, 64, 16, BF16, seed=3)
    ix = c.table.indices.clone()
    ix[1], ix[-1] = c.cache.pages + 5, -3
    table = P.PageTable(c.table.indptr, ix)
    lens = torch.tensor([10 ** 12, -4, 90], device="cuda")
    before = [x.clone() for x in c.tensors()]
    got = P.kv_evict(c.cache, table, lens, c.mass, 100, 4, 10)
    assert got.tolist() == [100, 0, 90]
    mine = set(c.rows[0])
    for x, y in zip(c.tensors(), before):
        changed = (x != y).flatten(1).any(1).nonzero().flatten().tolist()
        assert set(changed) <= mine - {c.rows[0][1]}
    with pytest.raises(lib.TgError) as e:
        P.kv_evict(c.cache, table, lens, c.mass, 100, 4, 10, check=True)
    assert e.value.status == lib.TG_EBOUNDS


def test_graph_streams_and_workspace():
    what, cut = CASES[11]
    c, plain = Cache(*what, BF16, seed=11), Cache(*what, BF16, seed=11)
    first = [x.clone() for x in c.tensors()]
    want = P.kv_evict(plain.cache, plain.table, plain.seq_len, plain.mass, *cut)
    ws = torch.empty(P.kv_evict_workspace_bytes(c.cache, c.table, c.seq_len, cut[0]), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(c.seq_len)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        P.kv_evict(c.cache, c.table, c.seq_len, c.mass, *cut, seq_len_out=out, workspace=ws)
    for _ in range(2):
        for x, y in zip(c.tensors(), first):
            x.copy_(y)
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)
        assert all(torch.equal(x, y) for x, y in zip(c.tensors(), plain.tensors()))
    for x, y in zip(c.tensors(), first):
        x.copy_(y)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    got = P.kv_evict(c.cache, c.table, c.seq_len, c.mass, *cut, stream=st)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(got, want) and all(torch.equal(x, y) for x, y in zip(c.tensors(), plain.tensors()))


def test_refusals():
    c = Cache([30, 20], 2, 64, 16, BF16)

    def call(**kw):
        a = dict(cache=c.cache, table=c.table, seq_len=c.seq_len, mass=c.mass, budget=10)
        a.update(kw)
        return P.kv_evict(**a)

    for bad in (dict(mass=c.mass.half()), dict(mass=c.mass[1:]), dict(mass_out=c.mass[..., :1]), dict(seq_len=c.seq_len[:1]),
                dict(seq_len=c.seq_len.int()), dict(kept=torch.empty(2, 2, 9, dtype=torch.int32, device="cuda")),
                dict(kept=torch.empty(2, 2, 10, device="cuda")), dict(workspace=torch.empty(8, dtype=torch.uint8, device="cuda")),
                dict(seq_len_out=torch.empty(3, dtype=torch.int64, device="cuda")),
                dict(cache=P.PagedKV(c.cache.k.double(), c.cache.v.double()))):
        with pytest.raises(ValueError):
            call(**bad)
    for bad in (dict(budget=-1), dict(first=-1), dict(recent=-2), dict(max_seq_len=-1)):
        with pytest.raises(lib.TgError) as e:
            call(**bad)
        assert e.value.status == lib.TG_EINVAL


def test_empty():
    c = Cache([], 2, 64, 16, BF16)
    got, kept = P.kv_evict(c.cache, c.table, c.seq_len, c.mass, 10, kept=True)
    assert got.shape == (0,) and kept.shape == (0, 2, 0)
    none = Cache([0, 0], 2, 64, 16, BF16)
    assert P.kv_evict(none.cache, none.table, none.seq_len, none.mass, 10).tolist() == [0, 0]


def test_a_view_of_the_mass_is_the_mass():
    """The stride of a dimension of one tells nothing: another view of the same weights is the mass itself."""
    c = Cache([40, 9], 1, 64, 16, BF16, seed=5)
    want = Cache([40, 9], 1, 64, 16, BF16, seed=5)
    lens = P.kv_evict(want.cache, want.table, want.seq_len, want.mass, 20, first=2, recent=5)
    view = torch.as_strided(c.mass, c.mass.shape, (16, 1, 3))
    assert view.stride() != c.mass.stride() and view.data_ptr() == c.mass.data_ptr()
    assert torch.equal(P.kv_evict(c.cache, c.table, c.seq_len, c.mass, 20, first=2, recent=5, mass_out=view), lens)
    for x, y, pages, n in ((x, y, pages, int(n)) for x, y in zip(c.tensors(), want.tensors()) for pages, n in zip(c.rows, lens)):
        at = torch.arange(n, device="cuda")
        where = torch.tensor(pages, device="cuda")[at // 16], at % 16
        assert torch.equal(x[where], y[where])
    with pytest.raises(ValueError, match="share"):
        P.kv_evict(c.cache, c.table, c.seq_len, c.mass, 20, mass_out=torch.as_strided(c.mass, c.mass.shape, (8, 1, 1)))
