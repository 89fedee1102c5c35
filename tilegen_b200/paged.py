"""Paged attention on torch tensors: rotary positions, appending to a paged key/value cache,
and attention of a batch of sequences that share a prefix.

Which pages hold a sequence's keys and values is a CSR pattern (:class:`PageTable`): row b
lists the pages of sequence b.  The calls follow :mod:`tilegen_b200.device`: asynchronous on
the given (default: current) stream, arguments checked here and in the library, no fallback.

A decoding step of a batch behind a shared prefix::

    q = kv_append(cache, table, seq_len, k, v, rope=rope, q=q, position_base=prefix_len)
    out = prefix_attention(q, cache, table, seq_len, prefix_pages=pages, prefix_len=prefix_len)

and the prefix itself is written once, as a table of one row.
"""

from __future__ import annotations

import contextlib
import ctypes
import math
from dataclasses import dataclass
from typing import List, Optional, Sequence, Tuple, Union

import torch

from . import lib as _lib
from .device import _dev

__all__ = ["Rope", "rope_frequencies", "rope", "rope_backward", "PagedKV", "PageTable", "kv_append",
           "prefix_attention", "prefix_attention_workspace_bytes"]

_SUFFIX = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16"}
_LAYOUT = {"half": _lib.TG_ROPE_HALF, "interleaved": _lib.TG_ROPE_INTERLEAVED}


def rope_frequencies(rot_dim: int, base: float = 10000.0, *, scaling: Optional[str] = None, factor: float = 1.0,
                     original_len: int = 8192, low: float = 1.0, high: float = 32.0,
                     device="cuda") -> torch.Tensor:
    """Angle per position of each of the rot_dim / 2 pairs (float64): base ** (-2 i / rot_dim).

    ``scaling`` stretches them for contexts ``factor`` times ``original_len``:

    * ``"linear"``: every pair turns ``factor`` times slower (positions interpolated);
    * ``"base"``: the base grows so that the slowest pair turns ``factor`` times slower and
      the fastest as before;
    * ``"banded"``: pairs that turn fewer than ``low`` times within ``original_len`` are
      slowed by ``factor``, those that turn more than ``high`` times are kept, and the pairs
      between are blended linearly in their number of turns;
    * ``"yarn"``: the same with the blend linear in the pair's index between the indices that
      turn ``high`` and ``low`` times (rounded outwards).
    """
    if rot_dim < 0 or rot_dim % 2:
        raise ValueError("rot_dim must be even (got %d)" % rot_dim)
    if not factor >= 1.0:
        raise ValueError("factor must be >= 1 (got %r)" % factor)
    if scaling not in (None, "linear", "base", "banded", "yarn"):
        raise ValueError("scaling must be None, 'linear', 'base', 'banded' or 'yarn' (got %r)" % (scaling,))
    if scaling == "base" and rot_dim > 2:
        base = base * factor ** (rot_dim / (rot_dim - 2))
    i = torch.arange(0, rot_dim, 2, dtype=torch.float64)
    f = base ** (-i / max(rot_dim, 1))
    if scaling == "linear":
        f = f / factor
    elif scaling == "banded":
        if not high > low:
            raise ValueError("high must be above low")
        keep = ((f * original_len / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        f = f * (keep + (1 - keep) / factor)
    elif scaling == "yarn":
        if not high > low > 0:
            raise ValueError("high must be above low, and low above 0")

        def index(turns):
            return rot_dim * math.log(original_len / (turns * 2 * math.pi)) / (2 * math.log(base))

        first = max(math.floor(index(high)), 0)
        last = min(math.ceil(index(low)), rot_dim - 1)
        slow = ((i / 2 - first) / max(last - first, 1e-3)).clamp(0, 1)
        f = f * ((1 - slow) + slow / factor)
    return f.to(_dev(device))


@dataclass
class Rope:
    """A rotation of the first 2 * freq.numel() elements of a head: pair i turns by position *
    freq[i] radians (freq: float64 on the GPU) and is multiplied by scale.  ``layout``: pairs
    are (i, i + half) for "half", (2 i, 2 i + 1) for "interleaved"."""

    freq: torch.Tensor
    layout: str = "half"
    scale: float = 1.0

    def desc(self, device: torch.device) -> _lib.TgRope:
        f = self.freq
        if f.dtype != torch.float64 or f.dim() != 1 or not f.is_contiguous() or f.device != device:
            raise ValueError("freq must be a contiguous float64 vector on %s (got %s %s on %s)"
                             % (device, tuple(f.shape), f.dtype, f.device))
        if self.layout not in _LAYOUT:
            raise ValueError("layout must be 'half' or 'interleaved' (got %r)" % (self.layout,))
        return _lib.TgRope(f.data_ptr(), 2 * f.numel(), _LAYOUT[self.layout], float(self.scale))


@dataclass
class PagedKV:
    """Keys and values in pages: [pages, page_size, heads, dim] each, any strides with the last
    one 1 (a cache stored head by head is passed transposed)."""

    k: torch.Tensor
    v: torch.Tensor

    @property
    def pages(self) -> int:
        return int(self.k.shape[0])

    @property
    def page_size(self) -> int:
        return int(self.k.shape[1])

    def desc(self) -> _lib.TgPagedKV:
        k, v = self.k, self.v
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.device != v.device:
            raise ValueError("k and v must be [pages, page_size, heads, dim] of one type on one device (got %s %s and "
                             "%s %s)" % (tuple(k.shape), k.dtype, tuple(v.shape), v.dtype))
        if not k.is_cuda or k.dtype not in _SUFFIX:
            raise ValueError("the cache must be float32, float16 or bfloat16 on a CUDA device (got %s on %s)"
                             % (k.dtype, k.device))
        pages, size, heads, dim = k.shape
        ks, vs = k.stride(), v.stride()
        if dim > 1 and (ks[3] != 1 or vs[3] != 1):
            raise ValueError("the cache's last stride must be 1")
        return _lib.TgPagedKV(k.data_ptr(), v.data_ptr(), pages, size, heads, dim, ks[0], ks[1], ks[2], vs[0], vs[1],
                              vs[2])


@dataclass
class PageTable:
    """CSR table of pages: sequence b holds the pages indices[indptr[b]:indptr[b + 1]], in the
    order of its tokens (int64, on the GPU)."""

    indptr: torch.Tensor
    indices: torch.Tensor

    @property
    def rows(self) -> int:
        return int(self.indptr.numel()) - 1

    @classmethod
    def from_lists(cls, pages: Sequence[Sequence[int]], device="cuda") -> "PageTable":
        d = _dev(device)
        indptr = [0]
        flat: List[int] = []
        for row in pages:
            flat.extend(int(x) for x in row)
            indptr.append(len(flat))
        return cls(torch.tensor(indptr, dtype=torch.int64).to(d), torch.tensor(flat, dtype=torch.int64).to(d))

    def desc(self, device: torch.device, pages: int) -> _lib.TgCsr:
        ip, ix = self.indptr, self.indices
        _vector(ip, "indptr", device)
        _vector(ix, "indices", device)
        if ip.numel() < 1:
            raise ValueError("indptr must have at least one entry")
        return _lib.TgCsr(ip.numel() - 1, pages, ix.numel(), ip.data_ptr(), ix.data_ptr(), None)


def _vector(t: torch.Tensor, name: str, device: torch.device, n: Optional[int] = None) -> int:
    if t.dtype != torch.int64 or t.dim() != 1 or not t.is_contiguous() or t.device != device:
        raise ValueError("%s must be a contiguous int64 vector on %s (got %s %s on %s)"
                         % (name, device, tuple(t.shape), t.dtype, t.device))
    if n is not None and t.numel() != n:
        raise ValueError("%s must have %d entries (got %d)" % (name, n, t.numel()))
    return t.data_ptr()


def _rows(t: torch.Tensor, name: str, shape: Tuple, dtype: torch.dtype, device: torch.device) -> _lib.TgRows:
    if t.shape != shape or t.dtype != dtype or t.device != device:
        raise ValueError("%s must be a %s tensor of shape %s on %s (got %s %s on %s)"
                         % (name, dtype, tuple(shape), device, t.dtype, tuple(t.shape), t.device))
    st = t.stride()
    if st[2] != 1 and shape[2] > 1:
        raise ValueError("%s: the last stride must be 1 (got %d)" % (name, st[2]))
    return _lib.TgRows(t.data_ptr(), st[0], st[1])


@contextlib.contextmanager
def _on(stream: torch.cuda.Stream):
    with torch.cuda.stream(stream):
        yield


def _place(device: torch.device, stream: Optional[torch.cuda.Stream]):
    """(context, stream pointer): the context makes the device and the stream current, so that
    outputs and workspaces allocated inside belong to that stream.  Nothing is entered where
    both are current already."""
    if stream is not None:
        if stream.device != device:
            raise ValueError("the stream is on %s and the tensors on %s" % (stream.device, device))
        return _on(stream), int(stream.cuda_stream)
    if torch.cuda.current_device() != device.index:
        return torch.cuda.device(device), int(torch.cuda.current_stream(device).cuda_stream)
    return contextlib.nullcontext(), int(torch.cuda.current_stream(device).cuda_stream)


def _rope_call(x: torch.Tensor, r: Rope, positions: torch.Tensor, out: Optional[torch.Tensor], flags: int,
               stream) -> torch.Tensor:
    L = _lib.load()
    dev = x.device
    if x.dim() != 3 or dev.type != "cuda" or x.dtype not in _SUFFIX:
        raise ValueError("x must be [tokens, heads, dim], float32, float16 or bfloat16, on a CUDA device (got %s %s on "
                         "%s)" % (tuple(x.shape), x.dtype, dev))
    tokens, heads, dim = x.shape
    xr = _rows(x, "x", x.shape, x.dtype, dev)
    rd = r.desc(dev)
    pos = _vector(positions, "positions", dev, tokens)
    ctx, sp = _place(dev, stream)
    with ctx:
        if out is None:
            out = torch.empty(x.shape, dtype=x.dtype, device=dev)
        yr = _rows(out, "out", x.shape, x.dtype, dev)
        fn = getattr(L, "tg_rope_" + _SUFFIX[x.dtype])
        _lib.check(fn(rd, xr, yr, tokens, heads, dim, pos, flags, sp), "tg_rope")
    return out


def rope(x: torch.Tensor, r: Rope, positions: torch.Tensor, out: Optional[torch.Tensor] = None,
         stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """x [tokens, heads, dim] rotated at positions [tokens] (int64); out may be x."""
    return _rope_call(x, r, positions, out, 0, stream)


def rope_backward(dout: torch.Tensor, r: Rope, positions: torch.Tensor, out: Optional[torch.Tensor] = None,
                  stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """The gradient with respect to x of rope(x, r, positions), for the gradient dout of its
    output; out may be dout."""
    return _rope_call(dout, r, positions, out, _lib.TG_FLAG_ROPE_INVERSE, stream)


def kv_append(cache: PagedKV, table: PageTable, seq_len: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
              rope: Optional[Rope] = None, q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None,
              q_indptr: Optional[torch.Tensor] = None, position_base: int = 0,
              positions: Optional[torch.Tensor] = None, check: bool = False,
              stream: Optional[torch.cuda.Stream] = None) -> Optional[torch.Tensor]:
    """Writes the new tokens' k and v [tokens, heads, dim] into the cache, k rotated on the way,
    and returns q rotated at the same positions (None without q).

    Sequence b brings the tokens q_indptr[b]:q_indptr[b + 1] (without q_indptr: token b) and is
    seq_len[b] tokens long after them; its new token i is token a = seq_len[b] - n + i of its
    pages, at position positions[t] or position_base + a.  ``check`` checks the index arrays
    first (and synchronises)."""
    L = _lib.load()
    kv = cache.desc()
    dev, dt = cache.k.device, cache.k.dtype
    tb = table.desc(dev, kv.pages)
    if k.dim() != 3:
        raise ValueError("k must be [tokens, heads, dim] (got %s)" % (tuple(k.shape),))
    tokens = int(k.shape[0])
    shape = (tokens, kv.heads, kv.dim)
    a = _lib.TgKvAppendArgs()
    a.cache, a.pages = ctypes.pointer(kv), ctypes.pointer(tb)
    a.seq_len = _vector(seq_len, "seq_len", dev, tb.rows)
    a.tokens = tokens
    if q_indptr is not None:
        a.q_indptr = _vector(q_indptr, "q_indptr", dev, tb.rows + 1)
    elif tokens != tb.rows:
        raise ValueError("%d tokens for %d sequences need a q_indptr" % (tokens, tb.rows))
    a.k, a.v = _rows(k, "k", shape, dt, dev), _rows(v, "v", shape, dt, dev)
    if rope is not None:
        a.rope = ctypes.pointer(rope.desc(dev))
    a.position_base = int(position_base)
    if positions is not None:
        a.positions = _vector(positions, "positions", dev, tokens)
    a.flags = _lib.TG_FLAG_BOUNDS_CHECK if check else 0
    ctx, sp = _place(dev, stream)
    with ctx:
        if q is not None:
            if q.dim() != 3:
                raise ValueError("q must be [tokens, q_heads, dim] (got %s)" % (tuple(q.shape),))
            qshape = (tokens, int(q.shape[1]), kv.dim)
            if q_out is None:
                q_out = torch.empty(qshape, dtype=dt, device=dev)
            a.q = ctypes.pointer(_rows(q, "q", qshape, dt, dev))
            a.q_out = ctypes.pointer(_rows(q_out, "q_out", qshape, dt, dev))
            a.q_heads = qshape[1]
        elif q_out is not None:
            raise ValueError("q_out without q")
        _lib.check(getattr(L, "tg_kv_append_" + _SUFFIX[dt])(a, sp), "tg_kv_append")
    return q_out


def _attention_args(q, cache, table, seq_len, prefix_pages, prefix_len, q_indptr, max_q_len, max_seq_len, scale,
                    causal, check):
    kv = cache.desc()
    dev, dt = cache.k.device, cache.k.dtype
    if dt == torch.float32:
        raise ValueError("attention takes float16 or bfloat16 caches (got %s)" % dt)
    tb = table.desc(dev, kv.pages)
    if q.dim() != 3:
        raise ValueError("q must be [tokens, q_heads, dim] (got %s)" % (tuple(q.shape),))
    tokens, heads = int(q.shape[0]), int(q.shape[1])
    a = _lib.TgPrefixAttentionArgs()
    a.cache, a.pages = ctypes.pointer(kv), ctypes.pointer(tb)
    a.seq_len = _vector(seq_len, "seq_len", dev, tb.rows)
    slots = tb.nnz * kv.page_size
    a.max_seq_len = slots if max_seq_len is None else int(max_seq_len)
    if prefix_pages is not None:
        a.prefix_pages, a.n_prefix_pages = _vector(prefix_pages, "prefix_pages", dev), prefix_pages.numel()
    a.prefix_len = int(prefix_len)
    a.tokens = tokens
    if q_indptr is not None:
        a.q_indptr = _vector(q_indptr, "q_indptr", dev, tb.rows + 1)
        a.max_q_len = tokens if max_q_len is None else int(max_q_len)
    else:
        if tokens != tb.rows:
            raise ValueError("%d tokens for %d sequences need a q_indptr" % (tokens, tb.rows))
        a.max_q_len = 1
    a.q_heads = heads
    a.q = _rows(q, "q", (tokens, heads, kv.dim), dt, dev)
    a.scale = kv.dim ** -0.5 if scale is None else float(scale)
    a.flags = (_lib.TG_FLAG_CAUSAL if causal else 0) | (_lib.TG_FLAG_BOUNDS_CHECK if check else 0)
    return a


def prefix_attention_workspace_bytes(q: torch.Tensor, cache: PagedKV, table: PageTable, seq_len: torch.Tensor,
                                     prefix_pages: Optional[torch.Tensor] = None, prefix_len: int = 0,
                                     q_indptr: Optional[torch.Tensor] = None, max_q_len: Optional[int] = None,
                                     max_seq_len: Optional[int] = None) -> int:
    """Bytes of workspace that prefix_attention needs with these arguments."""
    a = _attention_args(q, cache, table, seq_len, prefix_pages, prefix_len, q_indptr, max_q_len, max_seq_len, None,
                        True, False)
    return int(_lib.load().tg_prefix_attention_workspace_bytes(a))


def prefix_attention(q: torch.Tensor, cache: PagedKV, table: PageTable, seq_len: torch.Tensor,
                     prefix_pages: Optional[torch.Tensor] = None, prefix_len: int = 0,
                     q_indptr: Optional[torch.Tensor] = None, max_q_len: Optional[int] = None,
                     max_seq_len: Optional[int] = None, scale: Optional[float] = None, causal: bool = True,
                     out: Optional[torch.Tensor] = None, lse: Union[bool, torch.Tensor] = False,
                     workspace: Optional[torch.Tensor] = None, check: bool = False,
                     stream: Optional[torch.cuda.Stream] = None):
    """softmax(scale * q k^T) v for the queries q [tokens, q_heads, dim] of a batch whose
    sequences share the first prefix_len keys (in prefix_pages), each followed by the seq_len[b]
    keys of its own pages.  The prefix is read once for the whole batch.

    Queries are given as for kv_append: q_indptr, or one for each sequence.  With ``causal`` the
    last query of a sequence sees all its keys, the one before it one key less, and so on; a
    query that sees nothing gives zeros.  max_q_len and max_seq_len bound the tokens and the own
    length of a sequence (defaults: what the arrays' sizes allow; tighter bounds plan better).
    scale defaults to dim ** -0.5.  ``lse=True`` (or a float32 [tokens, q_heads] tensor) returns
    (out, log of the softmax's sum).  ``workspace`` (prefix_attention_workspace_bytes) is
    allocated on the call's stream where it is not given; ``check`` checks the index arrays
    first (and synchronises)."""
    L = _lib.load()
    a = _attention_args(q, cache, table, seq_len, prefix_pages, prefix_len, q_indptr, max_q_len, max_seq_len, scale,
                        causal, check)
    dev, dt = q.device, q.dtype
    ctx, sp = _place(dev, stream)
    with ctx:
        if out is None:
            out = torch.empty(q.shape, dtype=dt, device=dev)
        a.out = _rows(out, "out", q.shape, dt, dev)
        if lse is True:
            lse = torch.empty(q.shape[:2], dtype=torch.float32, device=dev)
        if isinstance(lse, torch.Tensor):
            if lse.shape != q.shape[:2] or lse.dtype != torch.float32 or lse.device != dev or not lse.is_contiguous():
                raise ValueError("lse must be a contiguous float32 tensor of shape %s on %s" % (tuple(q.shape[:2]), dev))
            a.lse = lse.data_ptr()
        nbytes = L.tg_prefix_attention_workspace_bytes(a)
        if workspace is None and nbytes:
            workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        wp, wn = (0, 0) if workspace is None else (workspace.data_ptr(), workspace.numel() * workspace.element_size())
        if workspace is not None and workspace.device != dev:
            raise ValueError("the workspace must be on %s (got %s)" % (dev, workspace.device))
        if wn < nbytes:
            raise ValueError("workspace too small: need %d bytes" % nbytes)
        _lib.check(getattr(L, "tg_prefix_attention_" + _SUFFIX[dt])(a, wp, wn, sp), "tg_prefix_attention")
    return (out, lse) if isinstance(lse, torch.Tensor) else out
