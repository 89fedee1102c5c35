"""Head norms, gathered attention weight and eviction without a GPU: refusals that come before anything
touches the device, and the sizes of workspaces."""

from __future__ import annotations

import ctypes
import random

import pytest
import torch
from torch.autograd import forward_ad

from tilegen_b200 import lib
from tilegen_b200 import paged as P

ROWS = lib.TgRows(4096, 256, 64)


def cache(**kw):
    c = dict(k=4096, v=4096, pages=10, page_size=16, heads=2, dim=64, k_page_stride=2048, k_slot_stride=128,
             k_head_stride=64, v_page_stride=2048, v_slot_stride=128, v_head_stride=64)
    c.update(kw)
    return lib.TgPagedKV(**c)


def table(**kw):
    t = dict(rows=3, cols=10, nnz=6, indptr=4096, indices=4096, data=None)
    t.update(kw)
    return lib.TgCsr(**t)


def filled(struct, fields, held=(), **kw):
    a = struct()
    a.held = held
    for k, v in {**fields, **kw}.items():
        setattr(a, k, ctypes.addressof(v) if isinstance(v, ctypes.Structure) and not isinstance(v, (lib.TgRows, lib.TgPagedMass)) else v)
    a.kept_alive = list(fields.values()) + list(kw.values())
    return a


def refused(call, status, msg):
    assert call == status, (call, lib.last_error())
    assert msg in lib.last_error(), lib.last_error()


# ------------------------------------------------------------------ norms
NORM = lib.TgHeadNorm(4096, 0, 1e-6, 0.0)
ROPE = lib.TgRope(4096, 64, 0, 1.0)


def norm(**kw):
    return filled(lib.TgNormRopeArgs, dict(tokens=3, dim=64, q_heads=4, k_heads=2, q=ROWS, k=ROWS, q_out=ROWS, k_out=ROWS,
                                           q_norm=NORM, k_norm=NORM, rope=ROPE, positions=4096), **kw)


def grad(**kw):
    return filled(lib.TgNormRopeGradArgs, dict(tokens=3, dim=64, q_heads=4, k_heads=2, q=ROWS, k=ROWS, dq_out=ROWS, dk_out=ROWS, dq=ROWS,
                                               dk=ROWS, q_norm=NORM, k_norm=NORM, dq_weight=4096, dk_weight=4096, rope=ROPE,
                                               positions=4096), **kw)


NORM_REFUSALS = [
    (dict(tokens=-1), lib.TG_EINVAL, "size"), (dict(dim=0), lib.TG_EINVAL, "size"), (dict(q_heads=-1), lib.TG_EINVAL, "size"),
    (dict(dim=257), lib.TG_EUNSUPPORTED, "256"), (dict(q_heads=1 << 24), lib.TG_EUNSUPPORTED, "2^24"),
    (dict(dim=32), lib.TG_EINVAL, "rot_dim"), (dict(positions=None), lib.TG_EINVAL, "positions"), (dict(flags=1), lib.TG_EINVAL, "flags"),
    (dict(q_norm=lib.TgHeadNorm(4096, 0, -1.0, 0.0)), lib.TG_EINVAL, "eps"),
    (dict(k_norm=lib.TgHeadNorm(4096, 0, float("nan"), 0.0)), lib.TG_EINVAL, "eps"),
    (dict(q=lib.TgRows(None, 256, 64)), lib.TG_EINVAL, "null q"), (dict(k=lib.TgRows(None, 256, 64)), lib.TG_EINVAL, "null k"),
    (dict(rope=lib.TgRope(4096, 64, 7, 1.0)), lib.TG_EINVAL, "layout"),
]


@pytest.mark.parametrize("kw,status,msg", NORM_REFUSALS)
def test_norm_refusals(kw, status, msg):
    L = lib.load()
    refused(L.tg_norm_rope_bf16(norm(**kw), None), status, msg)
    refused(L.tg_norm_rope_backward_f32(grad(**kw), 4096, 1 << 30, None), status, msg)


def test_norm_gradient_workspace():
    L = lib.load()
    ask = L.tg_norm_rope_backward_workspace_bytes
    n = ask(grad())
    assert n == 3 * 2 * 64 * 4 and ask(grad(tokens=0)) == 0 and ask(grad(dim=300)) == 0
    refused(L.tg_norm_rope_backward_f16(grad(), 4096, n - 1, None), lib.TG_ENOMEM, "workspace")
    refused(L.tg_norm_rope_backward_f16(grad(), None, n, None), lib.TG_ENOMEM, "workspace")
    refused(L.tg_norm_rope_backward_f16(grad(), 4104, n, None), lib.TG_EINVAL, "16-byte")
    refused(L.tg_norm_rope_backward_f16(grad(q_norm=None), 4096, n, None), lib.TG_EINVAL, "without its norm")
    sizes = [ask(grad(tokens=t, dim=d)) for t in (1, 100, 100000) for d in (2, 64, 256)]
    assert max(sizes) == ask(grad(tokens=100000, dim=256)) <= 1 << 20
    assert L.tg_norm_rope_bf16(None, None) == L.tg_norm_rope_backward_bf16(None, None, 0, None) == lib.TG_EINVAL
    assert L.tg_norm_rope_bf16(norm(tokens=0, q=lib.TgRows(), positions=None), None) == lib.TG_OK  # nothing to do
    assert L.tg_norm_rope_bf16(norm(q_heads=0, k_heads=0), None) == lib.TG_OK


def test_normed_append_refusals():
    L = lib.load()

    def append(c=None, **kw):
        return filled(lib.TgKvAppendArgs, dict(cache=c or cache(), pages=table(), seq_len=4096, tokens=3, k=ROWS, v=ROWS), **kw)

    bad = lib.TgHeadNorm(4096, 0, -1.0, 0.0)
    refused(L.tg_kv_append_normed_bf16(append(), bad, None, None), lib.TG_EINVAL, "eps")
    refused(L.tg_kv_append_normed_bf16(append(), None, bad, None), lib.TG_EINVAL, "eps")
    refused(L.tg_kv_append_normed_bf16(append(tokens=2), NORM, NORM, None), lib.TG_EINVAL, "q_indptr")
    refused(L.tg_kv_append_normed_bf16(append(k=lib.TgRows(None, 1, 1)), NORM, NORM, None), lib.TG_EINVAL, "null k")
    refused(L.tg_kv_append_normed_bf16(append(cache(dim=600)), NORM, NORM, None), lib.TG_EUNSUPPORTED, "256")
    refused(L.tg_kv_append_normed_bf16(None, NORM, NORM, None), lib.TG_EINVAL, "null")


# ------------------------------------------------------------------ gathered weight
MASS = lib.TgPagedMass(4096, 32, 2, 1)


def mass(**kw):
    return filled(lib.TgAttentionMassArgs, dict(cache=cache(), pages=table(), seq_len=4096, max_seq_len=96, tokens=3, max_q_len=1,
                                                q_heads=4, q=ROWS, lse=4096, scale=0.125, mass=MASS, decay=1.0,
                                                flags=lib.TG_FLAG_CAUSAL), **kw)


@pytest.mark.parametrize("kw,status,msg", [
    (dict(q_heads=3), lib.TG_EINVAL, "multiple"), (dict(q_heads=0), lib.TG_EINVAL, "multiple"),
    (dict(max_seq_len=-1), lib.TG_EINVAL, "max_seq_len"), (dict(tokens=4), lib.TG_EINVAL, "q_indptr"),
    (dict(tokens=-1), lib.TG_EINVAL, "size"), (dict(scale=0.0), lib.TG_EINVAL, "scale"), (dict(scale=float("nan")), lib.TG_EINVAL, "scale"),
    (dict(decay=-0.5), lib.TG_EINVAL, "decay"), (dict(decay=float("inf")), lib.TG_EINVAL, "decay"),
    (dict(flags=2), lib.TG_EINVAL, "flags"), (dict(seq_len=None), lib.TG_EINVAL, "seq_len"), (dict(lse=None), lib.TG_EINVAL, "lse"),
    (dict(q=lib.TgRows(None, 256, 64)), lib.TG_EINVAL, "null q"), (dict(q=lib.TgRows(4098, 256, 64)), lib.TG_EINVAL, "aligned"),
    (dict(q=lib.TgRows(4096, 260, 64)), lib.TG_EINVAL, "aligned"), (dict(mass=lib.TgPagedMass()), lib.TG_EINVAL, "null mass"),
    (dict(cache=cache(dim=80)), lib.TG_EUNSUPPORTED, "head dim"), (dict(cache=cache(k=None)), lib.TG_EINVAL, "null cache"),
    (dict(pages=table(cols=9)), lib.TG_EINVAL, "columns"), (dict(pages=table(indptr=None)), lib.TG_EINVAL, "indptr"),
    (dict(q_indptr=4096, max_q_len=0), lib.TG_EINVAL, "max_q_len"),
    (dict(pages=table(rows=1 << 30, nnz=1 << 34), max_seq_len=1 << 30, tokens=1 << 30), lib.TG_EUNSUPPORTED, "too many"),
])
def test_mass_refusals(kw, status, msg):
    refused(lib.load().tg_attention_mass_bf16(mass(**kw), 4096, 1 << 30, None), status, msg)


def test_mass_workspace():
    L = lib.load()
    ask, needed = L.tg_attention_mass_workspace_bytes, L.tg_attention_mass_needed_bytes
    assert ask(mass()) == 0 and ask(mass(q_indptr=4096, tokens=0, max_q_len=5)) == 0 and ask(mass(q_heads=3)) == 0
    long = mass(pages=table(rows=1, cols=10, nnz=600), tokens=9000, q_indptr=4096, max_q_len=9000, max_seq_len=9600)
    assert 0 < needed(long) <= ask(long) <= 80 << 20
    refused(L.tg_attention_mass_f16(long, 4096, needed(long) - 1, None), lib.TG_ENOMEM, "workspace")
    refused(L.tg_attention_mass_f16(long, None, 1 << 30, None), lib.TG_ENOMEM, "workspace")
    refused(L.tg_attention_mass_f16(long, 4100, 1 << 30, None), lib.TG_EINVAL, "16-byte")
    assert L.tg_attention_mass_f16(mass(pages=table(rows=0, nnz=0), tokens=0), None, 0, None) == lib.TG_OK
    assert L.tg_attention_mass_f16(None, None, 0, None) == lib.TG_EINVAL


def test_a_mass_workspace_serves_every_smaller_call():
    rng = random.Random(3)
    L = lib.load()
    for _ in range(300):
        kv = rng.choice([1, 2, 8])
        heads, dim = kv * rng.choice([1, 4, 5, 300]), rng.choice([64, 96, 128, 256])
        c = cache(pages=1 << 24, heads=kv, dim=dim)
        q = rng.choice([1, 5, 300, 4096, 100000])
        kept = L.tg_attention_mass_workspace_bytes(mass(cache=c, pages=table(rows=2, cols=1 << 24, nnz=1 << 20), q_heads=heads, tokens=q + 1,
                                                        q_indptr=4096, max_q_len=q, max_seq_len=1 << 20))
        for _ in range(20):
            rows, small, seq = rng.choice([1, 3, 64, 700]), rng.randint(1, q), rng.choice([1, 500, 9000, 200000])
            a = mass(cache=c, pages=table(rows=rows, cols=1 << 24, nnz=rows * -(-seq // 16)), q_heads=heads, tokens=rows * small,
                     q_indptr=4096, max_q_len=small, max_seq_len=seq)
            assert L.tg_attention_mass_needed_bytes(a) <= kept <= 80 << 20


def test_a_mass_workspace_does_not_depend_on_the_tokens():
    """What is kept by a first small batch, or by a call without a q_indptr, serves all of the same max_q_len."""
    L = lib.load()
    rng = random.Random(4)
    for _ in range(300):
        kv, top = rng.choice([1, 2, 8]), rng.choice([1, 5, 300, 2048, 100000])
        c = cache(pages=1 << 24, heads=kv, dim=rng.choice([64, 96, 128, 256]))
        heads = kv * rng.choice([1, 4, 5, 300])

        def args(rows, tokens, q, seq, ragged=True):
            return mass(cache=c, pages=table(rows=rows, cols=1 << 24, nnz=rows * -(-seq // 16)), q_heads=heads, tokens=tokens,
                        q_indptr=4096 if ragged else None, max_q_len=q, max_seq_len=seq)

        ask = L.tg_attention_mass_workspace_bytes
        kept = ask(args(1, 0, top, 16))
        assert kept == ask(args(3, 3, top, 500, False)) == ask(args(1, rng.randint(1, top), top, 9000)) == ask(args(1, 1 << 20, top, 9000))
        for _ in range(20):
            rows, q, seq = rng.choice([1, 3, 64, 700]), rng.randint(1, top), rng.choice([1, 500, 9000, 200000])
            assert L.tg_attention_mass_needed_bytes(args(rows, rows * q, q, seq)) <= kept <= 80 << 20
    most = mass(q_indptr=4096, max_q_len=(1 << 63) - 1)
    assert 0 < L.tg_attention_mass_workspace_bytes(most) <= 80 << 20


# ------------------------------------------------------------------ eviction
def evict(**kw):
    return filled(lib.TgKvEvictArgs, dict(cache=cache(), pages=table(), seq_len=4096, max_seq_len=96, budget=40, first=2, recent=5,
                                          mass=MASS, seq_len_out=4096), **kw)


@pytest.mark.parametrize("kw,status,msg", [
    (dict(budget=-1), lib.TG_EINVAL, "negative"), (dict(first=-1), lib.TG_EINVAL, "negative"), (dict(recent=-1), lib.TG_EINVAL, "negative"),
    (dict(max_seq_len=-1), lib.TG_EINVAL, "negative"), (dict(flags=lib.TG_FLAG_CAUSAL), lib.TG_EINVAL, "flags"),
    (dict(seq_len=None), lib.TG_EINVAL, "seq_len"), (dict(seq_len_out=None), lib.TG_EINVAL, "seq_len_out"),
    (dict(mass=lib.TgPagedMass()), lib.TG_EINVAL, "null mass"), (dict(kept=4096, kept_width=39), lib.TG_EINVAL, "kept"),
    (dict(kept=4096, kept_width=-1), lib.TG_EINVAL, "kept_width"), (dict(cache=cache(k=None)), lib.TG_EINVAL, "null cache"),
    (dict(pages=table(cols=9)), lib.TG_EINVAL, "columns"), (dict(pages=table(indptr=None)), lib.TG_EINVAL, "indptr"),
    (dict(pages=table(indices=None)), lib.TG_EINVAL, "indices"), (dict(pages=table(nnz=-1)), lib.TG_EINVAL, "size"),
    (dict(cache=cache(dim=1 << 30)), lib.TG_EUNSUPPORTED, "2^24"),
])
def test_evict_refusals(kw, status, msg):
    refused(lib.load().tg_kv_evict_bf16(evict(**kw), 4096, 1 << 30, None), status, msg)


def test_evict_workspace():
    L = lib.load()
    ask = L.tg_kv_evict_workspace_bytes
    n = ask(evict())
    assert n >= 3 * 2 * (16 + 8 * 40)
    refused(L.tg_kv_evict_f16(evict(), 4096, n - 1, None), lib.TG_ENOMEM, "workspace")
    refused(L.tg_kv_evict_f32(evict(), None, n, None), lib.TG_ENOMEM, "workspace")
    refused(L.tg_kv_evict_f32(evict(), 4100, n, None), lib.TG_EINVAL, "16-byte")
    assert L.tg_kv_evict_f32(evict(pages=table(rows=0, nnz=0)), None, 0, None) == lib.TG_OK
    assert L.tg_kv_evict_f32(None, None, 0, None) == lib.TG_EINVAL
    rng = random.Random(2)
    for _ in range(300):
        rows, seq, budget = rng.choice([1, 5, 300]), rng.choice([10, 3000, 100000]), rng.choice([0, 1, 700, 20000])
        kept = ask(evict(pages=table(rows=rows, nnz=rows * 7000), max_seq_len=seq, budget=budget))
        r = rng.randint(1, rows)
        assert ask(evict(pages=table(rows=r, nnz=r * rng.randint(0, 7000)), max_seq_len=rng.randint(0, seq), budget=budget)) <= kept


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 3, 64)
    kv = P.PagedKV(torch.zeros(4, 16, 2, 64), torch.zeros(4, 16, 2, 64))
    tb, none = P.PageTable(torch.zeros(1, dtype=torch.int64), torch.zeros(0, dtype=torch.int64)), torch.zeros(0, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        P.norm_rope(x, x, P.HeadNorm())
    with pytest.raises(ValueError, match="CUDA"):
        P.norm_rope_backward(x, x, x, x, P.HeadNorm())
    with pytest.raises(ValueError, match="CUDA"):
        P.attention_mass(torch.zeros(4, 16, 2), x, kv, tb, none, torch.zeros(2, 3))
    with pytest.raises(ValueError, match="CUDA"):
        P.kv_evict(kv, tb, none, torch.zeros(4, 16, 2), 10)


def test_forward_mode_tangents_are_refused():
    """A dual tensor has an address like any other, and its tangent would be lost without a word."""
    x, w, pos, r = torch.ones(2, 3, 64), torch.ones(64), torch.zeros(2, dtype=torch.int64), P.Rope(torch.ones(32, dtype=torch.float64))
    n = P.HeadNorm(w)
    with forward_ad.dual_level():
        d, dn = forward_ad.make_dual(x, x.clone()), P.HeadNorm(forward_ad.make_dual(w, w.clone()))
        for call in (lambda: P.rope(d, r, pos), lambda: P.rope_backward(d, r, pos), lambda: P.norm_rope(d, None, n),
                     lambda: P.norm_rope(x, d, n), lambda: P.norm_rope(x, None, dn), lambda: P.norm_rope(x, x, n, dn),
                     lambda: P.norm_rope_backward(d, None, x, None, n), lambda: P.norm_rope_backward(x, None, d, None, n),
                     lambda: P.norm_rope_backward(x, d, x, x, n), lambda: P.norm_rope_backward(x, x, x, x, n, dn),
                     lambda: P.rope(d.clone().requires_grad_(), r, pos)):
            with pytest.raises(NotImplementedError, match="tangent"):
                call()
        for call in (lambda: P.rope(x, r, pos), lambda: P.norm_rope(x, x, n), lambda: P.rope(d, r, pos, out=x)):
            with pytest.raises(ValueError, match="CUDA"):
                call()
    with pytest.raises(ValueError, match="CUDA"):  # the level has ended
        P.rope(d, r, pos)
