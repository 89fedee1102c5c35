"""A bounded cache as it is used: norms on the way into the cache, attention, gathered weight and eviction,
step after step."""

from __future__ import annotations

import importlib.util
import math
import os

import pytest
import torch

from tilegen_b200 import paged as P

pytestmark = pytest.mark.gpu


def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "bounded_cache_decode.py")
    spec = importlib.util.spec_from_file_location("bounded_cache_decode", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("kw", [dict(), dict(batch=3, prompt=700, budget=200, steps=25, dim=128, page=24, slack=1),
                                dict(batch=5, prompt=90, budget=64, steps=30, recent=40, first=40, heads=4, kv_heads=4)])
def test_the_example(kw):
    """Three 16-bit roundings of the block's output (projections, attention, sum): 4 half ulps."""
    e = example()
    s, *rest = result = e.generate(**kw)
    assert max(s.lens) <= s.budget + s.slack
    assert e.check(*result) < 4 * 2.0 ** -8


def test_steps_of_a_server_against_64_bits():
    """The weights that all kept keys have gathered over prompts, steps and evictions, and what was kept:
    a key's weight is that of the formula with the log-sum-exps that the calls returned, summed over the
    steps since it came, wherever it has moved.  Each of at most 41 weights has a relative error below
    2 * 2^-18 (1 + 16) + 2^-20 + 2^-22 * 8 (scores of normed heads of 64 are below 8 * 1.5^2), their sum
    41 * 2^-24 more."""
    e = example()
    s = e.Server([150, 40, 9], 96, recent=20, slack=5, seed=3)
    width = s.qkv.shape[0]
    total = [[{} for _ in range(s.kv_heads)] for _ in range(3)]  # token -> weight, 64 bits
    origin = [[[] for _ in range(s.kv_heads)] for _ in range(3)]
    keys = [{} for _ in range(3)]
    x = torch.randn(199, width, generator=s.g, device="cuda").to(s.qkv.dtype)
    count, news = [0, 0, 0], [150, 40, 9]
    group = s.heads // s.kv_heads
    for step in range(41):
        if step:
            kept = s.evict()
            if kept is not None:
                for b, row in enumerate(kept.tolist()):
                    for h in range(s.kv_heads):
                        origin[b][h] = [origin[b][h][i] for i in row[h] if i >= 0]
        y, q, lse = s.step(x, news)
        t = 0
        for b, n in enumerate(news):
            pages = torch.tensor(s.rows[b], device="cuda")
            at = torch.arange(s.lens[b], device="cuda")
            now = s.cache.k[pages[at // s.page], at % s.page]  # [place, key head, dim]
            for i in range(n):
                keys[b][count[b] + i] = now[s.lens[b] - n + i].clone()
            w = min(32, n)  # a prompt's last tokens weigh it
            for h in range(s.kv_heads):
                origin[b][h] += range(count[b], count[b] + n)
                k = torch.stack([keys[b][o][h] for o in origin[b][h]])
                assert torch.equal(k, now[:, h])  # each key is where it should be
                rows, L = q[t + n - w:t + n, h * group:(h + 1) * group].double(), lse[t + n - w:t + n, h * group:(h + 1) * group].double()
                p = (torch.einsum("ngd,kd->ngk", rows, k.double()) / math.sqrt(s.dim) - L[..., None]).exp()
                sees = torch.arange(len(origin[b][h]), device="cuda") < (len(origin[b][h]) - w + 1 + torch.arange(w, device="cuda"))[:, None]
                for o, v in zip(origin[b][h], (p * sees[:, None]).sum((0, 1)).tolist()):
                    total[b][h][o] = total[b][h].get(o, 0.0) + v
                got = s.mass[pages[at // s.page], at % s.page, h].double()
                want = torch.tensor([total[b][h][o] for o in origin[b][h]], dtype=torch.float64, device="cuda")
                rel = 2 * 2.0 ** -18 * (1 + 16) + 2.0 ** -20 + 2.0 ** -22 * 8 + 41 * 2.0 ** -24
                assert bool(((got - want).abs() <= rel * want).all())
            count[b] += n
            t += n
        x = y[torch.tensor(news, device="cuda").cumsum(0) - 1]
        news = [1, 1, 1]


def test_a_step_in_a_captured_graph():
    """Append, attention, weight and eviction of one decoding step, captured once and replayed: the lengths
    stay on the GPU and grow and shrink by themselves."""
    e = example()
    s = e.Server([100, 80], 90, recent=10, slack=4, seed=5)
    plain = e.Server([100, 80], 90, recent=10, slack=4, seed=5)
    width = s.qkv.shape[0]
    x = torch.randn(180, width, generator=s.g, device="cuda").to(s.qkv.dtype)
    for v in (s, plain):
        v.step(x, [100, 80])
    qkv = torch.randn(2, s.heads + 2 * s.kv_heads, s.dim, generator=s.g, device="cuda").to(s.qkv.dtype)
    positions = s.seen.clone()

    def step(v, lens, out):
        q, k, val = qkv.split((v.heads, v.kv_heads, v.kv_heads), 1)
        lens += 1
        q = P.kv_append(v.cache, v.table, lens, k, val, rope=v.rope, q=q, positions=positions, q_norm=v.q_norm, k_norm=v.k_norm)
        o, lse = P.prefix_attention(q, v.cache, v.table, lens, max_seq_len=101, lse=True)
        P.attention_mass(v.mass, q, v.cache, v.table, lens, lse, max_seq_len=101)
        P.kv_evict(v.cache, v.table, lens, v.mass, 90, first=4, recent=10, max_seq_len=101, seq_len_out=lens)
        out.copy_(o)

    out, want = (torch.empty(2, s.heads, s.dim, dtype=s.qkv.dtype, device="cuda") for _ in range(2))
    step(s, s.seq_len, out)  # sets the kernels' limits
    step(plain, plain.seq_len, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(s, s.seq_len, out)
    for i in range(15):
        qkv.copy_(torch.randn(qkv.shape, generator=s.g, device="cuda"))
        positions += 1
        graph.replay()
        step(plain, plain.seq_len, want)
        assert torch.equal(out, want) and torch.equal(s.seq_len, plain.seq_len)
        assert torch.equal(s.mass, plain.mass)
    assert s.seq_len.tolist() == [90, 90]
