"""Decoding with a bounded cache: one attention block of random weights, its queries and keys normed for
each head.

Each sequence brings a prompt, whose last tokens weigh the keys; what a key gathers from then on is added
at every step.  Every few steps the sequences that have grown over their budget are cut to it: the first
and the last keys stay and, for each key head by itself, those that gathered most.

    python examples/bounded_cache_decode.py [--batch 16] [--prompt 900] [--budget 512] [--steps 64] [--check]

``--check`` compares the last step with attention in 64 bits over the keys that were kept.
"""

from __future__ import annotations

import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from tilegen_b200 import paged  # noqa: E402


class Server:
    """A batch of sequences on a paged cache of at most budget + slack keys each after the prompts."""

    def __init__(self, prompts, budget, first=4, recent=32, slack=8, width=512, heads=8, kv_heads=2, dim=64, page=16, seed=0,
                 dtype=torch.bfloat16):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.heads, self.kv_heads, self.dim, self.page, self.g = heads, kv_heads, dim, page, g
        self.budget, self.first, self.recent, self.slack = budget, first, recent, slack

        def weight(n, m):
            return (torch.randn(n, m, generator=g, device="cuda") / math.sqrt(n)).to(dtype)

        self.qkv, self.out = weight(width, (heads + 2 * kv_heads) * dim), weight(heads * dim, width)
        self.q_norm, self.k_norm = (paged.HeadNorm(1 + 0.2 * torch.randn(dim, generator=g, device="cuda")) for _ in range(2))
        self.rope = paged.Rope(paged.rope_frequencies(dim, 500000.0))
        self.held = [max(n, budget + slack) for n in prompts]  # keys that a sequence's pages hold
        pages = [-(-n // page) for n in self.held]
        order = torch.randperm(sum(pages), generator=g, device="cuda").tolist()
        self.rows = [[order.pop() for _ in range(n)] for n in pages]
        self.table = paged.PageTable.from_lists(self.rows)
        self.cache = paged.PagedKV(*(torch.zeros(sum(pages), page, kv_heads, dim, dtype=dtype, device="cuda") for _ in range(2)))
        self.mass = paged.empty_mass(self.cache)
        self.lens = [0] * len(prompts)  # keys in the cache, as the host knows them
        self.seq_len = torch.zeros(len(prompts), dtype=torch.int64, device="cuda")
        self.seen = torch.zeros(len(prompts), dtype=torch.int64, device="cuda")  # tokens so far: the positions

    def project(self, x):
        y = (x @ self.qkv).view(x.shape[0], -1, self.dim)
        return y.split((self.heads, self.kv_heads, self.kv_heads), 1)

    def step(self, x, news, window=32):
        """New tokens x [tokens, width], news[b] of sequence b: (output, queries, log-sum-exp)."""
        n = torch.tensor(news, device="cuda")
        starts = torch.tensor([0] + news, device="cuda").cumsum(0)
        at = torch.arange(x.shape[0], device="cuda") - starts[:-1].repeat_interleave(n)
        positions = self.seen.repeat_interleave(n) + at
        self.lens = [a + b for a, b in zip(self.lens, news)]
        self.seq_len, self.seen = self.seq_len + n, self.seen + n
        longest, single = max(self.lens), max(news) == 1
        ragged = {} if single else {"q_indptr": starts}
        bound = {} if single else {"max_q_len": max(news)}
        q, k, v = self.project(x)
        q = paged.kv_append(self.cache, self.table, self.seq_len, k, v, rope=self.rope, q=q, positions=positions,
                            q_norm=self.q_norm, k_norm=self.k_norm, **ragged)
        o, lse = paged.prefix_attention(q, self.cache, self.table, self.seq_len, max_seq_len=longest, lse=True, **ragged, **bound)
        if single:
            paged.attention_mass(self.mass, q, self.cache, self.table, self.seq_len, lse, max_seq_len=longest)
        else:  # the prompts' last tokens weigh all keys
            last = [min(window, m) for m in news]
            rows = torch.cat([torch.arange(e - m, e, device="cuda") for e, m in zip(starts[1:].tolist(), last)])
            paged.attention_mass(self.mass, q[rows], self.cache, self.table, self.seq_len, lse[rows], decay=0.0,
                                 q_indptr=torch.tensor([0] + last, device="cuda").cumsum(0), max_q_len=max(last), max_seq_len=longest)
        return x + o.reshape(x.shape[0], -1) @ self.out, q, lse

    def evict(self):
        """Cuts sequences that are `slack` keys over their budget: the old places of their keys, or None."""
        if max(self.lens) < self.budget + self.slack:
            return None
        self.seq_len, kept = paged.kv_evict(self.cache, self.table, self.seq_len, self.mass, self.budget, first=self.first,
                                            recent=self.recent, max_seq_len=max(self.lens), kept=True)
        self.lens = [min(n, self.budget) for n in self.lens]
        return kept


def generate(batch=6, prompt=300, budget=128, steps=40, seed=0, **kw):
    """(server, keys and values by token as they were made, places' tokens, last outputs and queries)."""
    prompts = [max(1, prompt * (i + 1) // batch) for i in range(batch)]
    s = Server(prompts, budget, seed=seed, **kw)
    width = s.qkv.shape[0]
    made = [[] for _ in prompts]                                    # (k, v) of every token
    origin = [[list(range(n)) for _ in range(s.kv_heads)] for n in prompts]  # token at each place, by key head

    def note(news):
        for b, n in enumerate(news):
            at = torch.arange(s.lens[b] - n, s.lens[b], device="cuda")
            where = torch.tensor(s.rows[b], device="cuda")[at // s.page], at % s.page
            made[b].extend(zip(s.cache.k[where].unbind(0), s.cache.v[where].unbind(0)))

    x = torch.randn(sum(prompts), width, generator=s.g, device="cuda").to(s.qkv.dtype)
    y, q, _ = s.step(x, prompts)
    note(prompts)
    x = y[torch.tensor(prompts, device="cuda").cumsum(0) - 1]
    for _ in range(steps):
        kept = s.evict()
        if kept is not None:
            for b, row in enumerate(kept.tolist()):
                for h in range(s.kv_heads):
                    origin[b][h] = [origin[b][h][i] for i in row[h] if i >= 0]
        last = x
        x, q, _ = s.step(x, [1] * batch)
        note([1] * batch)
        for b in range(batch):
            for h in range(s.kv_heads):
                origin[b][h].append(len(made[b]) - 1)
    return s, made, origin, last, x, q


def check(s, made, origin, last, out, q):
    """The largest relative error of the last step's outputs against attention in 64 bits."""
    worst = 0.0
    for b, tokens in enumerate(made):
        o = []
        for j in range(s.heads):
            h = j // (s.heads // s.kv_heads)
            k, v = (torch.stack([tokens[t][i][h] for t in origin[b][h]]).double() for i in range(2))
            o.append((k @ q[b, j].double() / math.sqrt(s.dim)).softmax(0) @ v)
        want = last[b].double() + torch.cat(o) @ s.out.double()
        worst = max(worst, float((out[b].double() - want).norm() / want.norm()))
    return worst


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--batch", type=int, default=16)
    ap.add_argument("--prompt", type=int, default=900)
    ap.add_argument("--budget", type=int, default=512)
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--check", action="store_true")
    a = ap.parse_args(argv)
    result = generate(a.batch, a.prompt, a.budget, a.steps)
    torch.cuda.synchronize()
    s = result[0]
    print("%d sequences, %d to %d tokens each, %d to %d keys kept" % (a.batch, int(s.seen.min()), int(s.seen.max()), min(s.lens),
                                                                      max(s.lens)))
    if a.check:
        print("last step against 64 bits: relative error %.2g" % check(*result))
    return 0


if __name__ == "__main__":
    sys.exit(main())
