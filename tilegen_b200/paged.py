"""Paged attention on torch tensors: rotary positions, appending to a paged key/value cache,
and attention of a batch of sequences that share a prefix.

Which pages hold a sequence's keys and values is a CSR pattern (:class:`PageTable`): row b
lists the pages of sequence b.  The calls follow :mod:`tilegen_b200.device`: asynchronous on
the given (default: current) stream, arguments checked here and in the library, no fallback.

A decoding step of a batch behind a shared prefix::

    q = kv_append(cache, table, seq_len, k, v, rope=rope, q=q, position_base=prefix_len)
    out = prefix_attention(q, cache, table, seq_len, prefix_pages=pages, prefix_len=prefix_len, max_seq_len=longest)

and the prefix itself is written once, as a table of one row.  max_seq_len is a bound that the
host knows (lengths stay on the GPU); without it a sequence is taken to be as long as all listed
pages together, which plans the work worse.
"""

from __future__ import annotations

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


_CALLS: dict = {}


def _call(name: str):
    """A function of the library, looked up once."""
    fn = _CALLS.get(name)
    if fn is None:
        fn = _CALLS[name] = getattr(_lib.load(), name)
    return fn


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

    def desc(self, index: int) -> _lib.TgRope:
        f, layout = self.freq, _LAYOUT.get(self.layout)
        if f.dtype is not torch.float64 or f.dim() != 1 or not f.is_contiguous() or f.get_device() != index:
            raise ValueError("freq must be a contiguous float64 vector on cuda:%d (got %s %s on %s)"
                             % (index, tuple(f.shape), f.dtype, f.device))
        if layout is None:
            raise ValueError("layout must be 'half' or 'interleaved' (got %r)" % (self.layout,))
        return _lib.TgRope(f.data_ptr(), 2 * f.shape[0], layout, self.scale)


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
        shape, ks, vs = k.shape, k.stride(), v.stride()
        if len(shape) != 4 or shape != v.shape or k.dtype != v.dtype or k.get_device() != v.get_device():
            raise ValueError("k and v must be [pages, page_size, heads, dim] of one type on one device (got %s %s and "
                             "%s %s)" % (tuple(k.shape), k.dtype, tuple(v.shape), v.dtype))
        if not k.is_cuda or k.dtype not in _SUFFIX:
            raise ValueError("the cache must be float32, float16 or bfloat16 on a CUDA device (got %s on %s)"
                             % (k.dtype, k.device))
        if shape[3] > 1 and (ks[3] != 1 or vs[3] != 1):
            raise ValueError("the cache's last stride must be 1")
        return _lib.TgPagedKV(k.data_ptr(), v.data_ptr(), *shape, ks[0], ks[1], ks[2], vs[0], vs[1], vs[2])


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

    def desc(self, index: int, pages: int) -> _lib.TgCsr:
        ip, ix = _vector(self.indptr, "indptr", index), _vector(self.indices, "indices", index)
        rows = self.indptr.shape[0] - 1
        if rows < 0:
            raise ValueError("indptr must have at least one entry")
        return _lib.TgCsr(rows, pages, self.indices.shape[0], ip, ix, None)


# The calls below are made between the kernels of a decoding step, so their checks read what a
# tensor gives without making an object of it (device numbers instead of devices, for one).
def _vector(t: torch.Tensor, name: str, index: int, n: Optional[int] = None) -> int:
    if t.dtype is not torch.int64 or t.dim() != 1 or not t.is_contiguous() or t.get_device() != index:
        raise ValueError("%s must be a contiguous int64 vector on cuda:%d (got %s %s on %s)"
                         % (name, index, tuple(t.shape), t.dtype, t.device))
    if n is not None and t.shape[0] != n:
        raise ValueError("%s must have %d entries (got %d)" % (name, n, t.shape[0]))
    return t.data_ptr()


def _rows(t: torch.Tensor, name: str, shape: Tuple, dtype: torch.dtype, index: int) -> _lib.TgRows:
    if t.shape != shape or t.dtype is not dtype or t.get_device() != index:
        raise ValueError("%s must be a %s tensor of shape %s on cuda:%d (got %s %s on %s)"
                         % (name, dtype, tuple(shape), index, t.dtype, tuple(t.shape), t.device))
    st = t.stride()
    if st[2] != 1 and shape[2] > 1:
        raise ValueError("%s: the last stride must be 1 (got %d)" % (name, st[2]))
    return _lib.TgRows(t.data_ptr(), st[0], st[1])


def _like(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _stream(index: int, stream: Optional[torch.cuda.Stream]) -> int:
    """The stream's handle; raises unless it is on device `index`."""
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(index)  # current_stream(index).cuda_stream, made once a step
    if stream.device.index != index:
        raise ValueError("the stream is on %s and the tensors on cuda:%d" % (stream.device, index))
    return int(stream.cuda_stream)


def _elsewhere(index: int, stream: Optional[torch.cuda.Stream]):
    """The context in which a call's outputs and workspace are allocated and its kernels launched:
    they belong to the call's stream and device.  None where both are current already."""
    if stream is not None:
        return torch.cuda.stream(stream)
    return torch.cuda.device(index) if torch.cuda.current_device() != index else None


def _rope_call(x: torch.Tensor, r: Rope, positions: torch.Tensor, out: Optional[torch.Tensor], flags: int,
               stream) -> torch.Tensor:
    suffix = _SUFFIX.get(x.dtype)
    if x.dim() != 3 or not x.is_cuda or suffix is None:
        raise ValueError("x must be [tokens, heads, dim], float32, float16 or bfloat16, on a CUDA device (got %s %s on "
                         "%s)" % (tuple(x.shape), x.dtype, x.device))
    index, shape = x.get_device(), x.shape
    xr = _rows(x, "x", shape, x.dtype, index)
    rd = r.desc(index)
    pos = _vector(positions, "positions", index, shape[0])
    sp = _stream(index, stream)
    where = _elsewhere(index, stream)
    if where is not None:
        with where:
            return _rope_launch(suffix, x, out, xr, rd, pos, flags, sp)
    return _rope_launch(suffix, x, out, xr, rd, pos, flags, sp)


def _rope_launch(suffix, x, out, xr, rd, pos, flags, sp) -> torch.Tensor:
    if out is None:
        out = _like(x)
    yr = _rows(out, "out", x.shape, x.dtype, x.get_device())
    tokens, heads, dim = x.shape
    _lib.check(_call("tg_rope_" + suffix)(rd, xr, yr, tokens, heads, dim, pos, flags, sp), "tg_rope")
    return out


class _Turn(torch.autograd.Function):
    """The rotation, or with TG_FLAG_ROPE_INVERSE its transpose: each is the other's gradient."""

    @staticmethod
    def forward(ctx, x, freq, positions, layout, scale, flags):
        ctx.save_for_backward(freq, positions)
        ctx.how = layout, scale, flags
        return _rope_call(x, Rope(freq, layout, scale), positions, None, flags, None)

    @staticmethod
    def backward(ctx, dy):
        layout, scale, flags = ctx.how
        if dy.shape[2] > 1 and dy.stride(2) != 1:  # the gradient of a sum is one number, expanded
            dy = dy.contiguous()
        return (_Turn.apply(dy, *ctx.saved_tensors, layout, scale, flags ^ _lib.TG_FLAG_ROPE_INVERSE),) + (None,) * 5


def _turn(x, r, positions, out, flags, stream) -> torch.Tensor:
    if out is None and x.requires_grad and torch.is_grad_enabled():
        if stream is not None:
            _stream(x.get_device(), stream)  # it is on x's device
        with torch.cuda.stream(stream):  # the gradient is taken on the stream of the call (None: no change)
            return _Turn.apply(x, r.freq, positions, r.layout, r.scale, flags)
    return _rope_call(x, r, positions, out, flags, stream)


def rope(x: torch.Tensor, r: Rope, positions: torch.Tensor, out: Optional[torch.Tensor] = None,
         stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """x [tokens, heads, dim] rotated at positions [tokens] (int64); out may be x.

    Differentiable with respect to x, unless the result is written to a given out."""
    return _turn(x, r, positions, out, 0, stream)


def rope_backward(dout: torch.Tensor, r: Rope, positions: torch.Tensor, out: Optional[torch.Tensor] = None,
                  stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """The gradient with respect to x of rope(x, r, positions), for the gradient dout of its
    output; out may be dout.  (What autograd calls for rope; differentiable as rope is.)"""
    return _turn(dout, r, positions, out, _lib.TG_FLAG_ROPE_INVERSE, stream)


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
    first (and synchronises).  A call for serving: no gradient goes through it."""
    kv = cache.desc()
    index, dt = cache.k.get_device(), cache.k.dtype
    tb = table.desc(index, kv.pages)
    if k.dim() != 3:
        raise ValueError("k must be [tokens, heads, dim] (got %s)" % (tuple(k.shape),))
    tokens, rows = k.shape[0], tb.rows
    shape = (tokens, kv.heads, kv.dim)
    a = _lib.TgKvAppendArgs(ctypes.addressof(kv), ctypes.addressof(tb), _vector(seq_len, "seq_len", index, rows), tokens)
    if q_indptr is not None:
        a.q_indptr = _vector(q_indptr, "q_indptr", index, rows + 1)
    elif tokens != rows:
        raise ValueError("%d tokens for %d sequences need a q_indptr" % (tokens, rows))
    a.k, a.v = _rows(k, "k", shape, dt, index), _rows(v, "v", shape, dt, index)
    if rope is not None:
        rd = rope.desc(index)
        a.rope = ctypes.addressof(rd)
    a.position_base = position_base
    if positions is not None:
        a.positions = _vector(positions, "positions", index, tokens)
    if check:
        a.flags = _lib.TG_FLAG_BOUNDS_CHECK
    if q is not None:
        if q.dim() != 3:
            raise ValueError("q must be [tokens, q_heads, dim] (got %s)" % (tuple(q.shape),))
        a.q_heads = q.shape[1]
    elif q_out is not None:
        raise ValueError("q_out without q")
    sp = _stream(index, stream)
    where = _elsewhere(index, stream)
    if where is not None:
        with where:
            return _append_launch(a, q, q_out, (tokens, a.q_heads, kv.dim), dt, index, sp)
    return _append_launch(a, q, q_out, (tokens, a.q_heads, kv.dim), dt, index, sp)


def _append_launch(a, q, q_out, qshape, dt, index, sp) -> Optional[torch.Tensor]:
    if q is not None:
        qr = _rows(q, "q", qshape, dt, index)
        if q_out is None:
            q_out = _like(q)
        qo = _rows(q_out, "q_out", qshape, dt, index)
        a.q, a.q_out = ctypes.addressof(qr), ctypes.addressof(qo)
    _lib.check(_call("tg_kv_append_" + _SUFFIX[dt])(a, sp), "tg_kv_append")
    return q_out


def _attention_args(q, cache, table, seq_len, prefix_pages, prefix_len, q_indptr, max_q_len, max_seq_len, scale,
                    causal, check):
    """(arguments for the library, the descriptors that they point to)."""
    kv = cache.desc()
    index, dt = cache.k.get_device(), cache.k.dtype
    if dt is torch.float32:
        raise ValueError("attention takes float16 or bfloat16 caches (got %s)" % dt)
    tb = table.desc(index, kv.pages)
    if q.dim() != 3:
        raise ValueError("q must be [tokens, q_heads, dim] (got %s)" % (tuple(q.shape),))
    tokens, heads, _ = q.shape
    rows = tb.rows
    a = _lib.TgPrefixAttentionArgs(ctypes.addressof(kv), ctypes.addressof(tb), _vector(seq_len, "seq_len", index, rows),
                                   tb.nnz * kv.page_size if max_seq_len is None else max_seq_len)
    if prefix_pages is not None:
        a.prefix_pages, a.n_prefix_pages = _vector(prefix_pages, "prefix_pages", index), prefix_pages.shape[0]
    a.prefix_len = prefix_len
    a.tokens = tokens
    if q_indptr is not None:
        a.q_indptr = _vector(q_indptr, "q_indptr", index, rows + 1)
        a.max_q_len = tokens if max_q_len is None else max_q_len
    else:
        if tokens != rows:
            raise ValueError("%d tokens for %d sequences need a q_indptr" % (tokens, rows))
        a.max_q_len = 1
    a.q_heads = heads
    a.q = _rows(q, "q", (tokens, heads, kv.dim), dt, index)
    a.scale = kv.dim ** -0.5 if scale is None else scale
    a.flags = (_lib.TG_FLAG_CAUSAL if causal else 0) | (_lib.TG_FLAG_BOUNDS_CHECK if check else 0)
    return a, (kv, tb)


def prefix_attention_workspace_bytes(q: torch.Tensor, cache: PagedKV, table: PageTable, seq_len: torch.Tensor,
                                     prefix_pages: Optional[torch.Tensor] = None, prefix_len: int = 0,
                                     q_indptr: Optional[torch.Tensor] = None, max_q_len: Optional[int] = None,
                                     max_seq_len: Optional[int] = None) -> int:
    """Bytes of a workspace to keep for prefix_attention: enough for a call with these arguments and
    for any of the same head sizes that is smaller (fewer tokens, sequences, listed pages or prefix
    tokens, smaller bounds)."""
    a, _held = _attention_args(q, cache, table, seq_len, prefix_pages, prefix_len, q_indptr, max_q_len, max_seq_len,
                               None, True, False)
    return int(_call("tg_prefix_attention_workspace_bytes")(a))


def prefix_attention(q: torch.Tensor, cache: PagedKV, table: PageTable, seq_len: torch.Tensor,
                     prefix_pages: Optional[torch.Tensor] = None, prefix_len: int = 0,
                     q_indptr: Optional[torch.Tensor] = None, max_q_len: Optional[int] = None,
                     max_seq_len: Optional[int] = None, scale: Optional[float] = None, causal: bool = True,
                     out: Optional[torch.Tensor] = None, lse: Union[bool, torch.Tensor] = False,
                     workspace: Optional[torch.Tensor] = None, check: bool = False,
                     stream: Optional[torch.cuda.Stream] = None):
    """softmax(scale * q k^T) v for the queries q [tokens, q_heads, dim] of a batch whose
    sequences share the first prefix_len keys (in prefix_pages), each followed by the seq_len[b]
    keys of its own pages.  The prefix is fetched once for every 256 rows (tokens times query heads
    of a key head) of a batch of more than 32, for heads of 64 and 128, else once for every 16 or 32.

    Queries are given as for kv_append: q_indptr, or one for each sequence.  With ``causal`` the
    last query of a sequence sees all its keys, the one before it one key less, and so on; a
    query that sees nothing gives zeros, and so does one that no sequence holds.  max_q_len and
    max_seq_len bound the tokens and the own length of a sequence (defaults: what the arrays' sizes
    allow; tighter ones plan better, by up to half of the time): tokens past the first max_q_len
    see nothing, a longer sequence counts as max_seq_len.  Softmax and sums are 32-bit; the weights
    are rounded to the values' type for their product with them.  out may not share memory with q.
    scale defaults to dim ** -0.5.  ``lse=True`` (or a float32 [tokens, q_heads] tensor) returns
    (out, log of the softmax's sum).  ``workspace`` (prefix_attention_workspace_bytes for one to
    keep) is allocated on the call's stream where it is not given; ``check`` checks the index arrays
    first (and synchronises).  A call for serving: no gradient goes through it."""
    a, _held = _attention_args(q, cache, table, seq_len, prefix_pages, prefix_len, q_indptr, max_q_len, max_seq_len,
                               scale, causal, check)
    index = q.get_device()
    sp = _stream(index, stream)
    where = _elsewhere(index, stream)
    if where is not None:
        with where:
            return _attention_launch(a, q, out, lse, workspace, index, sp)
    return _attention_launch(a, q, out, lse, workspace, index, sp)


def _workspace(workspace: torch.Tensor, need: int, index: int) -> Tuple[int, int]:
    """Address and bytes of a caller's workspace of at least `need` bytes."""
    if workspace.get_device() != index:
        raise ValueError("the workspace must be on cuda:%d (got %s)" % (index, workspace.device))
    if not workspace.is_contiguous():  # its bytes would not be the ones from its address on
        raise ValueError("the workspace must be contiguous (got strides %s of shape %s)"
                         % (tuple(workspace.stride()), tuple(workspace.shape)))
    size = workspace.numel() * workspace.element_size()
    if size < need:
        raise ValueError("workspace too small: need %d bytes" % need)
    return workspace.data_ptr(), size


def _attention_launch(a, q, out, lse, workspace, index, sp):
    if out is None:
        out = _like(q)
    a.out = _rows(out, "out", q.shape, q.dtype, index)
    if lse is True:
        lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    if isinstance(lse, torch.Tensor):
        if lse.shape != q.shape[:2] or lse.dtype != torch.float32 or lse.get_device() != index or not lse.is_contiguous():
            raise ValueError("lse must be a contiguous float32 tensor of shape %s on cuda:%d" % (tuple(q.shape[:2]), index))
        a.lse = lse.data_ptr()
    need = _call("tg_prefix_attention_needed_bytes")(a)
    ws = size = 0
    if workspace is None and need:
        workspace, size = torch.empty(need, dtype=torch.uint8, device=q.device), need
        ws = workspace.data_ptr()
    elif workspace is not None:
        ws, size = _workspace(workspace, need, index)
    _lib.check(_call("tg_prefix_attention_" + _SUFFIX[q.dtype])(a, ws, size, sp), "tg_prefix_attention")
    return (out, lse) if isinstance(lse, torch.Tensor) else out
