"""Decoding of a batch behind a shared prefix: one attention block of random weights.

The prefix (a system prompt, a document) is written to the paged cache once.  Each sequence then
brings a prompt of its own length and generates tokens one by one; every step appends the new keys
and values, rotated, to the sequence's pages and attends to [prefix, own tokens], the prefix being
read once for the whole batch.

    python examples/shared_prefix_decode.py [--batch 16] [--prefix 2048] [--steps 32] [--check]

``--check`` compares the last step with attention over all tokens in 64 bits.
"""

from __future__ import annotations

import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from tilegen_b200 import paged  # noqa: E402


class Block:
    """q, k, v and output projections of random weights, and a paged cache."""

    def __init__(self, width=1024, heads=16, kv_heads=4, dim=64, page=16, pages=4096, context=32768, seed=0,
                 dtype=torch.bfloat16):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.heads, self.kv_heads, self.dim, self.page = heads, kv_heads, dim, page

        def weight(n, m):
            return (torch.randn(n, m, generator=g, device="cuda") / math.sqrt(n)).to(dtype)

        self.qkv = weight(width, (heads + 2 * kv_heads) * dim)
        self.out = weight(heads * dim, width)
        self.cache = paged.PagedKV(*(torch.zeros(pages, page, kv_heads, dim, dtype=dtype, device="cuda") for _ in range(2)))
        self.free = list(range(pages))
        factor = max(1.0, context / 8192)
        self.rope = paged.Rope(paged.rope_frequencies(dim, 500000.0, scaling="yarn", factor=factor),
                               "half", 0.1 * math.log(factor) + 1.0)

    def take(self, tokens):
        """Pages for so many tokens."""
        return [self.free.pop() for _ in range(-(-tokens // self.page))]

    def project(self, x):
        y = (x @ self.qkv).view(x.shape[0], -1, self.dim)
        return y.split((self.heads, self.kv_heads, self.kv_heads), 1)  # views: the calls take strides

    def write_prefix(self, x):
        """The keys and values of the prefix tokens x [tokens, width], as a table of one row."""
        self.prefix_len = x.shape[0]
        pages = self.take(self.prefix_len)
        _, k, v = self.project(x)
        paged.kv_append(self.cache, paged.PageTable.from_lists([pages]), torch.tensor([self.prefix_len], device="cuda"), k, v,
                        rope=self.rope, q_indptr=torch.tensor([0, self.prefix_len], device="cuda"))
        self.prefix_pages = torch.tensor(pages, device="cuda")

    def step(self, x, table, seq_len, max_len, q_indptr=None, max_q_len=None):
        """New tokens x [tokens, width] of the batch, whose sequences are seq_len long after them."""
        q, k, v = self.project(x)
        q = paged.kv_append(self.cache, table, seq_len, k, v, rope=self.rope, q=q, q_indptr=q_indptr,
                            position_base=self.prefix_len)
        o = paged.prefix_attention(q, self.cache, table, seq_len, prefix_pages=self.prefix_pages, prefix_len=self.prefix_len,
                                   q_indptr=q_indptr, max_q_len=max_q_len, max_seq_len=max_len)
        return x + o.reshape(x.shape[0], -1) @ self.out


def generate(batch=16, prefix=2048, steps=32, prompt=(5, 60), seed=0, **kw):
    """(block, every token's input, outputs of the last step, own lengths) of `steps` decoding steps."""
    block = Block(seed=seed, **kw)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    width = block.qkv.shape[0]

    def tokens(n):
        return torch.randn(n, width, generator=g, device="cuda").to(block.qkv.dtype)

    shared = tokens(prefix)
    block.write_prefix(shared)
    lens = [prompt[0] + (prompt[1] - prompt[0]) * i // max(1, batch - 1) for i in range(batch)]
    longest = max(lens) + steps
    table = paged.PageTable.from_lists([block.take(n + steps) for n in lens])
    own = [[] for _ in lens]

    # the prompts, all in one call
    x = tokens(sum(lens))
    for seq, part in zip(own, x.split(lens)):
        seq.append(part)
    seq_len = torch.tensor(lens, device="cuda")
    starts = torch.tensor([0] + lens, device="cuda").cumsum(0)
    y = block.step(x, table, seq_len, longest, starts, max(lens))
    x = y[starts[1:] - 1]  # each sequence goes on from its last token
    # and one token of each sequence a step
    for _ in range(steps):
        for seq, row in zip(own, x):
            seq.append(row[None])
        seq_len += 1
        last, x = x, block.step(x, table, seq_len, longest)
    return block, shared, [torch.cat(seq) for seq in own], last, x


def check(block, shared, own, last, out):
    """The largest relative error of the last step's outputs against attention in 64 bits."""
    worst = 0.0
    for b, seq in enumerate(own):
        x = torch.cat((shared, seq))
        q, k, v = (t.clone() for t in block.project(x))
        pos = torch.arange(x.shape[0], device="cuda")
        q, k = paged.rope(q, block.rope, pos), paged.rope(k, block.rope, pos)
        group = block.heads // block.kv_heads
        k, v = (t.double().repeat_interleave(group, 1) for t in (k, v))
        score = torch.einsum("hd,khd->hk", q[-1].double(), k) / math.sqrt(block.dim)
        o = torch.einsum("hk,khd->hd", score.softmax(-1), v).reshape(1, -1)
        want = last[b].double() + (o @ block.out.double())[0]
        worst = max(worst, float((out[b].double() - want).norm() / want.norm()))
    return worst


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--batch", type=int, default=16)
    ap.add_argument("--prefix", type=int, default=2048)
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--check", action="store_true")
    a = ap.parse_args(argv)
    result = generate(a.batch, a.prefix, a.steps)
    torch.cuda.synchronize()
    print("%d sequences, %d tokens each after their prompts, behind %d shared tokens" % (a.batch, a.steps, a.prefix))
    if a.check:
        print("last step against 64 bits: relative error %.2g" % check(*result))
    return 0


if __name__ == "__main__":
    sys.exit(main())
