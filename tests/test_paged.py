"""The paged-attention calls without a GPU: the C ABI's second header, frequencies, and
refusals that come before anything touches the device."""

from __future__ import annotations

import ctypes
import math
import subprocess

import pytest
import torch

from tilegen_b200 import lib
from tilegen_b200 import paged as P


def test_every_paged_symbol_is_exported_and_typed():
    declared = set(lib.header_symbols(lib.HEADER_PAGED))
    assert declared == set(lib.SIGNATURES_PAGED)
    out = subprocess.run(["nm", "-D", "--defined-only", lib.lib_path()], capture_output=True, text=True).stdout
    exported = {line.split()[-1] for line in out.splitlines() if " T " in line}
    assert declared <= exported
    L = lib.load()
    assert all(getattr(L, n).argtypes == lib.SIGNATURES_PAGED[n][1] for n in declared)


# ------------------------------------------------------------------ frequencies
@pytest.fixture
def on_cpu(monkeypatch):
    monkeypatch.setattr(P, "_dev", torch.device)


def test_frequencies(on_cpu):
    f = P.rope_frequencies(8, 10000.0, device="cpu")
    assert f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14)
    assert P.rope_frequencies(0, device="cpu").numel() == 0
    lin = P.rope_frequencies(64, scaling="linear", factor=4.0, device="cpu")
    assert torch.allclose(lin * 4, P.rope_frequencies(64, device="cpu"), rtol=1e-14)


def test_scaled_base_keeps_the_fastest_pair_and_slows_the_slowest(on_cpu):
    f, g = P.rope_frequencies(64, device="cpu"), P.rope_frequencies(64, scaling="base", factor=8.0, device="cpu")
    assert float(g[0]) == 1.0
    assert math.isclose(float(f[-1] / g[-1]), 8.0, rel_tol=1e-12)


@pytest.mark.parametrize("scaling", ["banded", "yarn"])
def test_banded_scaling(on_cpu, scaling):
    kw = dict(original_len=4096, low=1.0, high=32.0, device="cpu")
    f = P.rope_frequencies(128, 10000.0, **kw)
    g = P.rope_frequencies(128, 10000.0, scaling=scaling, factor=4.0, **kw)
    ratio = f / g
    turns = f * 4096 / (2 * math.pi)
    assert torch.all(ratio[turns > 45] == 1.0)  # kept (45: past the rounding of "yarn" outwards)
    assert torch.allclose(ratio[turns < 0.75], torch.tensor(4.0, dtype=torch.float64))
    assert torch.all(ratio[1:] >= ratio[:-1] - 1e-12)
    assert torch.allclose(P.rope_frequencies(128, 10000.0, scaling=scaling, factor=1.0, **kw), f)


def test_frequency_refusals(on_cpu):
    for kw in (dict(rot_dim=7), dict(rot_dim=8, scaling="cubic"), dict(rot_dim=8, factor=0.5),
               dict(rot_dim=8, scaling="banded", low=4.0, high=4.0)):
        with pytest.raises(ValueError):
            P.rope_frequencies(**kw, device="cpu")


# ------------------------------------------------------------------ refusals of the library
def _cache(**kw):
    c = dict(k=4096, v=4096, pages=10, page_size=16, heads=2, dim=64, k_page_stride=2048, k_slot_stride=128,
             k_head_stride=64, v_page_stride=2048, v_slot_stride=128, v_head_stride=64)
    c.update(kw)
    return lib.TgPagedKV(**c)


def _table(**kw):
    t = dict(rows=3, cols=10, nnz=6, indptr=4096, indices=4096, data=None)
    t.update(kw)
    return lib.TgCsr(**t)


def _attention(cache=None, table=None, **kw):
    a = lib.TgPrefixAttentionArgs()
    a.held = cache or _cache(), table or _table()
    a.cache, a.pages = (ctypes.addressof(x) for x in a.held)
    fields = dict(seq_len=4096, max_seq_len=96, prefix_pages=4096, n_prefix_pages=4, prefix_len=50, tokens=3,
                  q_indptr=None, max_q_len=1, q_heads=4, q=lib.TgRows(4096, 256, 64), out=lib.TgRows(4096, 256, 64),
                  lse=None, scale=0.125, flags=lib.TG_FLAG_CAUSAL)
    fields.update(kw)
    for k, v in fields.items():
        setattr(a, k, v)
    return a


def _refused(status, a, msg, ws=4096, n=1 << 30):
    L = lib.load()
    assert L.tg_prefix_attention_bf16(a, ws, n, None) == status
    assert msg in lib.last_error(), lib.last_error()


def test_attention_workspace_size():
    L = lib.load()
    a = _attention()
    n = L.tg_prefix_attention_workspace_bytes(a)
    parts = 2  # one split of the prefix, one chunk of own keys
    assert n >= parts * 3 * 4 * (64 * 4 + 8) and n % 256 == 0
    assert L.tg_prefix_attention_workspace_bytes(_attention(prefix_len=0)) == 0  # one part: nothing to join
    assert L.tg_prefix_attention_workspace_bytes(_attention(tokens=0, table=_table(rows=0, nnz=0))) == 0
    assert L.tg_prefix_attention_workspace_bytes(_attention(q_heads=3)) == 0


@pytest.mark.parametrize("kw,status,msg", [
    (dict(q_heads=3), lib.TG_EINVAL, "multiple"),
    (dict(q_heads=0), lib.TG_EINVAL, "multiple"),
    (dict(prefix_len=65), lib.TG_EINVAL, "prefix_len"),
    (dict(prefix_len=-1), lib.TG_EINVAL, "prefix_len"),
    (dict(prefix_pages=None), lib.TG_EINVAL, "prefix_pages"),
    (dict(max_seq_len=-1), lib.TG_EINVAL, "max_seq_len"),
    (dict(tokens=4), lib.TG_EINVAL, "q_indptr"),
    (dict(tokens=-1), lib.TG_EINVAL, "size"),
    (dict(scale=0.0), lib.TG_EINVAL, "scale"),
    (dict(scale=float("nan")), lib.TG_EINVAL, "scale"),
    (dict(flags=2), lib.TG_EINVAL, "flags"),
    (dict(seq_len=None), lib.TG_EINVAL, "seq_len"),
    (dict(q=lib.TgRows(None, 256, 64)), lib.TG_EINVAL, "null q"),
    (dict(q=lib.TgRows(4098, 256, 64)), lib.TG_EINVAL, "aligned"),
    (dict(out=lib.TgRows(4096, 260, 64)), lib.TG_EINVAL, "aligned"),
    (dict(cache=_cache(dim=80)), lib.TG_EUNSUPPORTED, "head dim"),
    (dict(cache=_cache(page_size=0)), lib.TG_EINVAL, "page_size"),
    (dict(cache=_cache(k=None)), lib.TG_EINVAL, "null cache"),
    (dict(cache=_cache(pages=0), table=_table(cols=0)), lib.TG_EINVAL, "without pages"),
    (dict(tokens=1 << 30, q_indptr=4096, max_q_len=1, q_heads=64), lib.TG_EUNSUPPORTED, "too many rows"),
    (dict(cache=_cache(v_slot_stride=129)), lib.TG_EINVAL, "aligned"),
    (dict(table=_table(cols=9)), lib.TG_EINVAL, "columns"),
    (dict(table=_table(indptr=None)), lib.TG_EINVAL, "indptr"),
    (dict(table=_table(nnz=-1)), lib.TG_EINVAL, "size"),
])
def test_attention_refusals(kw, status, msg):
    _refused(status, _attention(**kw), msg)


def test_attention_refuses_a_missing_or_small_workspace():
    n = lib.load().tg_prefix_attention_workspace_bytes(_attention())
    _refused(lib.TG_ENOMEM, _attention(), "workspace", 4096, n - 1)
    _refused(lib.TG_ENOMEM, _attention(), "workspace", None, n)
    _refused(lib.TG_EINVAL, _attention(), "16-byte", 4100, n)


_Q = lib.TgRows(4096, 128, 64)


def _append(cache=None, table=None, rope=None, **kw):
    a = lib.TgKvAppendArgs()
    a.held = cache or _cache(), table or _table(), rope
    a.cache, a.pages = (ctypes.addressof(x) for x in a.held[:2])
    if rope is not None:
        a.rope = ctypes.addressof(rope)
    fields = dict(seq_len=4096, tokens=3, q_indptr=None, k=lib.TgRows(4096, 128, 64), v=lib.TgRows(4096, 128, 64))
    fields.update(kw)
    for k, v in fields.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,msg", [
    (dict(tokens=2), "q_indptr"),
    (dict(k=lib.TgRows(None, 128, 64)), "null k"),
    (dict(rope=lib.TgRope(4096, 66, 0, 1.0)), "rot_dim"),
    (dict(rope=lib.TgRope(4096, 31, 0, 1.0)), "rot_dim"),
    (dict(rope=lib.TgRope(4096, 32, 2, 1.0)), "layout"),
    (dict(rope=lib.TgRope(None, 32, 0, 1.0)), "freq"),
    (dict(q=ctypes.addressof(_Q), q_heads=2), "q_out"),
    (dict(flags=lib.TG_FLAG_CAUSAL), "flags"),
    (dict(table=_table(rows=0), tokens=3, q_indptr=4096), "sequence"),
])
def test_append_refusals(kw, msg):
    assert lib.load().tg_kv_append_f32(_append(**kw), None) == lib.TG_EINVAL
    assert msg in lib.last_error()


def test_rope_refusals():
    L = lib.load()
    x, r = lib.TgRows(4096, 128, 64), lib.TgRope(4096, 64, 0, 1.0)
    assert L.tg_rope_f32(r, x, x, 3, 2, 64, None, 0, None) == lib.TG_EINVAL
    assert "positions" in lib.last_error()
    assert L.tg_rope_f32(r, x, x, 3, 2, 64, 4096, 1, None) == lib.TG_EINVAL
    assert L.tg_rope_f32(r, x, x, -3, 2, 64, 4096, 0, None) == lib.TG_EINVAL
    assert L.tg_rope_f32(lib.TgRope(4096, 1 << 15, 0, 1.0), x, x, 3, 2, 1 << 16, 4096, 0, None) == lib.TG_EUNSUPPORTED
    assert L.tg_rope_f32(None, x, x, 3, 2, 64, 4096, 0, None) == lib.TG_EINVAL
    assert L.tg_rope_f32(r, x, x, 0, 2, 64, None, 0, None) == lib.TG_OK  # nothing to do


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 3, 8)
    with pytest.raises(ValueError, match="CUDA"):
        P.rope(x, P.Rope(torch.zeros(4, dtype=torch.float64)), torch.zeros(2, dtype=torch.int64))
    kv = P.PagedKV(torch.zeros(4, 16, 2, 64), torch.zeros(4, 16, 2, 64))
    table = P.PageTable(torch.zeros(1, dtype=torch.int64), torch.zeros(0, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        P.kv_append(kv, table, torch.zeros(0, dtype=torch.int64), x, x)
    with pytest.raises(ValueError, match="CUDA"):
        P.prefix_attention(x, kv, table, torch.zeros(0, dtype=torch.int64))


def test_a_workspace_is_contiguous_and_on_the_calls_device():
    """One byte expanded to many is no workspace: a kernel writes from its address on."""
    from tilegen_b200 import device as D

    cpu = torch.device("cpu")
    ok = torch.empty(512, dtype=torch.uint8)
    assert P._workspace(ok, 512, -1) == (ok.data_ptr(), 512)  # -1: the device number of a CPU tensor
    assert D._ws(512, cpu, ok) == (ok.data_ptr(), 512)
    for bad in (torch.empty(1, dtype=torch.uint8).expand(512), torch.empty(1024, dtype=torch.uint8)[::2],
                torch.empty(32, 32, dtype=torch.uint8).t()[:, ::2]):
        with pytest.raises(ValueError, match="contiguous"):
            P._workspace(bad, 512, -1)
        with pytest.raises(ValueError, match="contiguous"):
            D._ws(512, cpu, bad)
    with pytest.raises(ValueError, match="cuda:0"):
        P._workspace(ok, 512, 0)
    with pytest.raises(ValueError, match="cuda:0"):
        D._ws(512, torch.device("cuda", 0), ok)
    with pytest.raises(ValueError, match="small"):
        P._workspace(ok, 513, -1)


def test_attention_refuses_a_max_q_len_of_zero():
    _refused(lib.TG_EINVAL, _attention(q_indptr=4096, max_q_len=0), "max_q_len")
    empty = _attention(q_indptr=4096, max_q_len=0, tokens=0)
    assert lib.load().tg_prefix_attention_bf16(empty, None, 0, None) == lib.TG_OK


@pytest.mark.parametrize("rows,tokens,heads,kv_heads,dim,seq,listed", [
    (1, 32768, 32, 8, 256, 32768, 32768),            # a long prompt
    (1, 16384, 32, 8, 96, 16384, 16384),
    (1024, 16384, 32, 8, 128, 8192, 1024 * 8192),    # 16 tokens for each of many sequences
    (256, 2048, 32, 8, 128, 65536, 65536 + 255 * 512),  # one long sequence among short ones
    (1024, 16384, 32, 8, 64, 65536, 65536 + 1023 * 512),
])
def test_attention_workspace_stays_small(rows, tokens, heads, kv_heads, dim, seq, listed):
    """Own parts take 1 GiB at most, or one part of each row, whatever the sizes."""
    a = _attention(cache=_cache(pages=1 << 20, heads=kv_heads, dim=dim), table=_table(rows=rows, cols=1 << 20, nnz=listed // 16),
                   tokens=tokens, q_indptr=4096, max_q_len=tokens // rows, q_heads=heads, max_seq_len=seq, prefix_len=0)
    assert lib.load().tg_prefix_attention_workspace_bytes(a) <= max(1 << 30, tokens * heads * (4 * dim + 8)) + 512


def test_a_workspace_serves_every_smaller_call():
    """A buffer taken at the largest sizes of a server, and calls with fewer of everything."""
    import random

    rng = random.Random(5)
    ask = lib.load().tg_prefix_attention_workspace_bytes

    def below(n):
        return rng.choice([n, rng.randint(0, n), int(n ** rng.random())])

    def args(rows, tokens, nnz, heads, kv_heads, dim, page, prefix, seq, q, ragged):
        return _attention(cache=_cache(pages=1 << 24, heads=kv_heads, dim=dim, page_size=page), table=_table(rows=rows, cols=1 << 24, nnz=nnz),
                          tokens=tokens if ragged else rows, q_indptr=4096 if ragged else None, max_q_len=q, q_heads=heads,
                          max_seq_len=seq, prefix_len=prefix, n_prefix_pages=-(-prefix // page))

    for _ in range(300):
        kv_heads, page = rng.choice([1, 2, 8]), rng.choice([1, 7, 16, 64])
        heads, dim = kv_heads * rng.choice([1, 4, 8]), rng.choice([64, 96, 128, 256])
        rows, seq = rng.choice([1, 4, 64, 130, 1024]), rng.choice([1, 256, 2000, 8192, 131072])
        q, prefix = rng.choice([1, 5, 300, 4096]), rng.choice([0, 0, 100, 8192, 131072])
        tokens, nnz = rows + rng.randint(0, rows * (q - 1)), rows * -(-seq // page)
        kept = ask(args(rows, tokens, nnz, heads, kv_heads, dim, page, prefix, seq, q, True))
        for _ in range(30):
            r = max(1, below(rows))
            small = args(r, max(1, below(tokens)), below(nnz), heads, kv_heads, dim, page, below(prefix), below(seq), max(1, below(q)),
                         rng.random() < 0.7)
            assert ask(small) <= kept
            needed = lib.load().tg_prefix_attention_needed_bytes(small)
            assert needed <= ask(small)
