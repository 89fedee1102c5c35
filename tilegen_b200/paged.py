"""Paged attention on torch tensors: rotary positions, norms of queries and keys with the rotation,
appending to a paged key/value cache, attention of a batch of sequences that share a prefix, the
attention weight that cached keys gather, and eviction of those that gathered least.

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
from torch.autograd import forward_ad

from . import lib as _lib
from .device import _dev

__all__ = ["Rope", "rope_frequencies", "rope", "rope_backward", "HeadNorm", "norm_rope", "norm_rope_backward",
           "norm_rope_backward_workspace_bytes", "PagedKV", "PageTable", "kv_append", "prefix_attention",
           "prefix_attention_workspace_bytes", "empty_mass", "attention_mass", "attention_mass_workspace_bytes", "kv_evict",
           "kv_evict_workspace_bytes"]

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
class HeadNorm:
    """The norm of a head x [dim]: x / sqrt(mean(x^2) + eps) * (offset + weight), or without that factor
    where weight is None.  weight: [dim], float32 or the heads' type, on their GPU; offset is 1 for
    models that keep the weights' distance from one."""

    weight: Optional[torch.Tensor] = None
    eps: float = 1e-6
    offset: float = 0.0

    def desc(self, dim: int, dtype: torch.dtype, index: int) -> _lib.TgHeadNorm:
        w = self.weight
        if w is None:
            return _lib.TgHeadNorm(None, 0, self.eps, self.offset)
        if w.shape != (dim,) or (w.dtype is not dtype and w.dtype is not torch.float32) or not w.is_contiguous() \
                or w.get_device() != index:
            raise ValueError("a norm's weight must be a contiguous %s or float32 vector of %d on cuda:%d (got %s %s on %s)"
                             % (dtype, dim, index, tuple(w.shape), w.dtype, w.device))
        return _lib.TgHeadNorm(w.data_ptr(), w.dtype is not dtype or dtype is torch.float32, self.eps, self.offset)


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
    if st[2] != 1 and shape[2] > 1 and t.numel():
        raise ValueError("%s: the last stride must be 1 (got %d)" % (name, st[2]))
    return _lib.TgRows(t.data_ptr(), st[0], st[1])


def _like(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t, memory_format=torch.contiguous_format)  # half the time of torch.empty with a shape


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


def _no_tangent(name: str, *tensors: Optional[torch.Tensor]) -> None:
    """Refuses tensors that carry a forward-mode tangent, which a call by address would drop.  (Asked for where a
    level of dual tensors is open.)"""
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("%s has no forward-mode derivative: a dual tensor would lose its tangent" % name)


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
    if out is None and forward_ad._current_level >= 0:
        _no_tangent("rope", x)
    if out is None and x.requires_grad and torch.is_grad_enabled():
        if stream is not None:
            _stream(x.get_device(), stream)  # it is on x's device
        with torch.cuda.stream(stream):  # the gradient is taken on the stream of the call (None: no change)
            return _Turn.apply(x, r.freq, positions, r.layout, r.scale, flags)
    return _rope_call(x, r, positions, out, flags, stream)


def rope(x: torch.Tensor, r: Rope, positions: torch.Tensor, out: Optional[torch.Tensor] = None,
         stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """x [tokens, heads, dim] rotated at positions [tokens] (int64); out may be x.

    Differentiable with respect to x, unless the result is written to a given out; a dual tensor of
    forward-mode differentiation is refused."""
    return _turn(x, r, positions, out, 0, stream)


def rope_backward(dout: torch.Tensor, r: Rope, positions: torch.Tensor, out: Optional[torch.Tensor] = None,
                  stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """The gradient with respect to x of rope(x, r, positions), for the gradient dout of its
    output; out may be dout.  (What autograd calls for rope; differentiable as rope is.)"""
    return _turn(dout, r, positions, out, _lib.TG_FLAG_ROPE_INVERSE, stream)


_NO_ROWS = _lib.TgRows()


def _norm_inputs(q, k, q_norm, k_norm, rope, positions):
    """(suffix, device, q's rows, k's rows, k's shape, descriptors of the norms and the rope, positions)."""
    suffix = _SUFFIX.get(q.dtype)
    if q.dim() != 3 or not q.is_cuda or suffix is None:
        raise ValueError("q must be [tokens, heads, dim], float32, float16 or bfloat16, on a CUDA device (got %s %s on %s)"
                         % (tuple(q.shape), q.dtype, q.device))
    index, dt, qs = q.get_device(), q.dtype, q.shape
    qr, kr, ks = _rows(q, "q", qs, dt, index), _NO_ROWS, None
    if k is not None:
        if k.dim() != 3:
            raise ValueError("k must be [tokens, heads, dim] (got %s)" % (tuple(k.shape),))
        ks = (qs[0], k.shape[1], qs[2])
        kr = _rows(k, "k", ks, dt, index)
    elif k_norm is not None:
        raise ValueError("k_norm without k")
    held = (None if q_norm is None else q_norm.desc(qs[2], dt, index), None if k_norm is None else k_norm.desc(qs[2], dt, index),
            None if rope is None else rope.desc(index))
    pos = None
    if rope is not None:
        if positions is None:
            raise ValueError("a rotation needs positions")
        pos = _vector(positions, "positions", index, qs[0])
    return suffix, index, qr, kr, ks, held, pos


def _address(desc) -> Optional[int]:
    return None if desc is None else ctypes.addressof(desc)


def _norm_call(q, k, q_norm, k_norm, rope, positions, q_out, k_out, stream):
    inputs = _norm_inputs(q, k, q_norm, k_norm, rope, positions)
    if k is None and k_out is not None:
        raise ValueError("k_out without k")
    sp = _stream(inputs[1], stream)
    where = _elsewhere(inputs[1], stream)
    if where is not None:
        with where:
            return _norm_launch(inputs, q, k, q_out, k_out, sp)
    return _norm_launch(inputs, q, k, q_out, k_out, sp)


def _norm_launch(inputs, q, k, q_out, k_out, sp):
    suffix, index, qr, kr, ks, held, pos = inputs
    qs, ko = q.shape, _NO_ROWS
    if q_out is None:
        q_out = _like(q)
    qo = _rows(q_out, "q_out", qs, q.dtype, index)
    if k is not None:
        if k_out is None:
            k_out = _like(k)
        ko = _rows(k_out, "k_out", ks, q.dtype, index)
    qn, kn, rd = held
    a = _lib.TgNormRopeArgs(qs[0], qs[2], qs[1], ks[1] if ks else 0, qr, kr, qo, ko, _address(qn), _address(kn), _address(rd), pos)
    _lib.check(_call("tg_norm_rope_" + suffix)(a, sp), "tg_norm_rope")
    return q_out, k_out


class _NormTurn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, freq, positions, how):
        q_norm, k_norm, layout, scale = how
        ctx.save_for_backward(q, k, q_weight, k_weight, freq, positions)
        ctx.how = how
        rope = None if freq is None else Rope(freq, layout, scale)
        return _norm_call(q, k, q_norm and HeadNorm(q_weight, *q_norm), k_norm and HeadNorm(k_weight, *k_norm), rope, positions,
                          None, None, None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, q_weight, k_weight, freq, positions = ctx.saved_tensors
        q_norm, k_norm, layout, scale = ctx.how
        rope = None if freq is None else Rope(freq, layout, scale)
        dq, dk, dqw, dkw = norm_rope_backward(dq_out, dk_out, q, k, q_norm and HeadNorm(q_weight, *q_norm),
                                              k_norm and HeadNorm(k_weight, *k_norm), rope, positions)
        return dq, dk, dqw, dkw, None, None, None


def norm_rope(q: torch.Tensor, k: Optional[torch.Tensor] = None, q_norm: Optional[HeadNorm] = None,
              k_norm: Optional[HeadNorm] = None, rope: Optional[Rope] = None, positions: Optional[torch.Tensor] = None,
              q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None,
              stream: Optional[torch.cuda.Stream] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(q, k) [tokens, heads, dim], each head normed and then rotated at positions [tokens] (int64), in
    one pass over both.  Without a norm that tensor is only rotated, without a rope nothing turns; k
    may be None.  dim is 256 at most.  q_out and k_out may be q and k.

    Differentiable with respect to q, k and the norms' weights (once), unless an out is given; dual
    tensors of forward-mode differentiation are refused."""
    if q_out is None and k_out is None and forward_ad._current_level >= 0:
        _no_tangent("norm_rope", q, k, q_norm and q_norm.weight, k_norm and k_norm.weight)
    if q_out is not None or k_out is not None or not torch.is_grad_enabled() or not any(
            t is not None and t.requires_grad for t in (q, k, q_norm and q_norm.weight, k_norm and k_norm.weight)):
        return _norm_call(q, k, q_norm, k_norm, rope, positions, q_out, k_out, stream)
    if stream is not None:
        _stream(q.get_device(), stream)  # it is on q's device
    how = tuple(n and (n.eps, n.offset) for n in (q_norm, k_norm)) + ((rope.layout, rope.scale) if rope else (None, None))
    with torch.cuda.stream(stream):  # the gradient is taken on the stream of the call (None: no change)
        return _NormTurn.apply(q, k, q_norm and q_norm.weight, k_norm and k_norm.weight, rope and rope.freq,
                               positions if rope else None, how)


def norm_rope_backward(dq_out: torch.Tensor, dk_out: Optional[torch.Tensor], q: torch.Tensor, k: Optional[torch.Tensor] = None,
                       q_norm: Optional[HeadNorm] = None, k_norm: Optional[HeadNorm] = None, rope: Optional[Rope] = None,
                       positions: Optional[torch.Tensor] = None, dq: Optional[torch.Tensor] = None,
                       dk: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None,
                       stream: Optional[torch.cuda.Stream] = None):
    """(dq, dk, gradient of q_norm's weight, of k_norm's weight) of norm_rope(q, k, ...) for the gradients
    dq_out and dk_out of its outputs; None where there is no such tensor.  The weights' gradients have
    the weights' type; their sums are 32-bit and in a fixed order.  dq may be dq_out or q, dk likewise.
    ``workspace``: norm_rope_backward_workspace_bytes, allocated on the call's stream where not given."""
    if forward_ad._current_level >= 0:
        _no_tangent("norm_rope_backward", dq_out, dk_out, q, k, q_norm and q_norm.weight, k_norm and k_norm.weight)
    inputs = _norm_inputs(q, k, q_norm, k_norm, rope, positions)
    if (k is None) != (dk_out is None) or (k is None and dk is not None):
        raise ValueError("k and the gradients of k go together")
    sp = _stream(inputs[1], stream)
    where = _elsewhere(inputs[1], stream)
    if where is not None:
        with where:
            return _norm_grad_launch(inputs, dq_out, dk_out, q, k, q_norm, k_norm, dq, dk, workspace, sp)
    return _norm_grad_launch(inputs, dq_out, dk_out, q, k, q_norm, k_norm, dq, dk, workspace, sp)


def _packed(t: torch.Tensor) -> torch.Tensor:
    """The gradient of a sum is one number, expanded."""
    return t.contiguous() if t.dim() == 3 and t.stride(2) != 1 and t.shape[2] > 1 else t


def _norm_grad_launch(inputs, dq_out, dk_out, q, k, q_norm, k_norm, dq, dk, workspace, sp):
    suffix, index, qr, kr, ks, held, pos = inputs
    qs, dt, gk, ko = q.shape, q.dtype, _NO_ROWS, _NO_ROWS
    dq_out = _packed(dq_out)
    gq = _rows(dq_out, "dq_out", qs, dt, index)
    if dq is None:
        dq = _like(q)
    qo = _rows(dq, "dq", qs, dt, index)
    if k is not None:
        dk_out = _packed(dk_out)
        gk = _rows(dk_out, "dk_out", ks, dt, index)
        if dk is None:
            dk = _like(k)
        ko = _rows(dk, "dk", ks, dt, index)
    dqw = torch.empty_like(q_norm.weight) if q_norm is not None and q_norm.weight is not None else None
    dkw = torch.empty_like(k_norm.weight) if k_norm is not None and k_norm.weight is not None else None
    qn, kn, rd = held
    a = _lib.TgNormRopeGradArgs(qs[0], qs[2], qs[1], ks[1] if ks else 0, qr, kr, gq, gk, qo, ko, _address(qn), _address(kn),
                                None if dqw is None else dqw.data_ptr(), None if dkw is None else dkw.data_ptr(), _address(rd), pos)
    need = _call("tg_norm_rope_backward_workspace_bytes")(a)
    ws = size = 0
    if workspace is None and need:
        workspace, size = torch.empty(need, dtype=torch.uint8, device=q.device), need
        ws = workspace.data_ptr()
    elif workspace is not None:
        ws, size = _workspace(workspace, need, index)
    _lib.check(_call("tg_norm_rope_backward_" + suffix)(a, ws, size, sp), "tg_norm_rope_backward")
    return dq, dk, dqw, dkw


def norm_rope_backward_workspace_bytes(tokens: int, dim: int) -> int:
    """Bytes of a workspace to keep for norm_rope_backward: it serves every call with heads of at most dim
    elements and at most as many tokens."""
    return int(_call("tg_norm_rope_backward_workspace_bytes")(_lib.TgNormRopeGradArgs(tokens, dim)))


def kv_append(cache: PagedKV, table: PageTable, seq_len: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
              rope: Optional[Rope] = None, q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None,
              q_indptr: Optional[torch.Tensor] = None, position_base: int = 0,
              positions: Optional[torch.Tensor] = None, check: bool = False,
              stream: Optional[torch.cuda.Stream] = None, q_norm: Optional[HeadNorm] = None,
              k_norm: Optional[HeadNorm] = None) -> Optional[torch.Tensor]:
    """Writes the new tokens' k and v [tokens, heads, dim] into the cache, k rotated on the way,
    and returns q rotated at the same positions (None without q).  With q_norm or k_norm the heads of
    that tensor are normed before they are rotated (heads of 256 at most).

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
    elif q_out is not None or q_norm is not None:
        raise ValueError("q_out or q_norm without q")
    norms = None
    if q_norm is not None or k_norm is not None:
        norms = tuple(None if n is None else n.desc(kv.dim, dt, index) for n in (q_norm, k_norm))
    sp = _stream(index, stream)
    where = _elsewhere(index, stream)
    if where is not None:
        with where:
            return _append_launch(a, norms, q, q_out, (tokens, a.q_heads, kv.dim), dt, index, sp)
    return _append_launch(a, norms, q, q_out, (tokens, a.q_heads, kv.dim), dt, index, sp)


def _append_launch(a, norms, q, q_out, qshape, dt, index, sp) -> Optional[torch.Tensor]:
    if q is not None:
        qr = _rows(q, "q", qshape, dt, index)
        if q_out is None:
            q_out = _like(q)
        qo = _rows(q_out, "q_out", qshape, dt, index)
        a.q, a.q_out = ctypes.addressof(qr), ctypes.addressof(qo)
    if norms is None:
        _lib.check(_call("tg_kv_append_" + _SUFFIX[dt])(a, sp), "tg_kv_append")
    else:
        _lib.check(_call("tg_kv_append_normed_" + _SUFFIX[dt])(a, *norms, sp), "tg_kv_append")
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


def _mass_desc(mass: torch.Tensor, name: str, cache: PagedKV, index: int) -> _lib.TgPagedMass:
    shape = cache.k.shape[:3]
    if mass.shape != shape or mass.dtype is not torch.float32 or mass.get_device() != index:
        raise ValueError("%s must be a float32 tensor of shape %s on cuda:%d (got %s %s on %s)"
                         % (name, tuple(shape), index, mass.dtype, tuple(mass.shape), mass.device))
    strides = mass.stride()
    if 0 in strides and any(st == 0 and n > 1 for st, n in zip(strides, shape)):
        raise ValueError("%s must have a place of its own for every key (got strides %s)" % (name, strides))
    return _lib.TgPagedMass(mass.data_ptr(), *strides)


def empty_mass(cache: PagedKV) -> torch.Tensor:
    """A mass for the keys of a cache, [pages, page_size, heads] zeros in the order that reads and writes
    fastest (slots side by side)."""
    pages, size, heads, _ = cache.k.shape
    return torch.zeros(pages, heads, size, dtype=torch.float32, device=cache.k.device).transpose(1, 2)


def _mass_args(mass, q, cache, table, seq_len, lse, q_indptr, max_q_len, max_seq_len, scale, causal, decay, check):
    """(arguments for the library, the descriptors that they point to); the checks of _attention_args."""
    kv = cache.desc()
    index, dt = cache.k.get_device(), cache.k.dtype
    if dt is torch.float32:
        raise ValueError("attention takes float16 or bfloat16 caches (got %s)" % dt)
    tb = table.desc(index, kv.pages)
    if q.dim() != 3:
        raise ValueError("q must be [tokens, q_heads, dim] (got %s)" % (tuple(q.shape),))
    tokens, heads, _ = q.shape
    rows, starts = tb.rows, None
    if q_indptr is not None:
        starts = _vector(q_indptr, "q_indptr", index, rows + 1)
        max_q_len = tokens if max_q_len is None else max_q_len
    else:
        if tokens != rows:
            raise ValueError("%d tokens for %d sequences need a q_indptr" % (tokens, rows))
        max_q_len = 1
    if lse is not None and (lse.shape != (tokens, heads) or lse.dtype is not torch.float32 or lse.get_device() != index
                            or not lse.is_contiguous()):
        raise ValueError("lse must be a contiguous float32 tensor of shape %s on cuda:%d (got %s %s on %s)"
                         % ((tokens, heads), index, tuple(lse.shape), lse.dtype, lse.device))
    m = _lib.TgAttentionMassArgs(
        ctypes.addressof(kv), ctypes.addressof(tb), _vector(seq_len, "seq_len", index, rows),
        tb.nnz * kv.page_size if max_seq_len is None else max_seq_len, tokens, starts, max_q_len, heads,
        _rows(q, "q", (tokens, heads, kv.dim), dt, index), None if lse is None else lse.data_ptr(),
        kv.dim ** -0.5 if scale is None else scale, _lib.TgPagedMass() if mass is None else _mass_desc(mass, "mass", cache, index), decay,
        (_lib.TG_FLAG_CAUSAL if causal else 0) | (_lib.TG_FLAG_BOUNDS_CHECK if check else 0))
    return m, (kv, tb)


def attention_mass(mass: torch.Tensor, q: torch.Tensor, cache: PagedKV, table: PageTable, seq_len: torch.Tensor,
                   lse: torch.Tensor, q_indptr: Optional[torch.Tensor] = None, max_q_len: Optional[int] = None,
                   max_seq_len: Optional[int] = None, scale: Optional[float] = None, causal: bool = True,
                   decay: float = 1.0, workspace: Optional[torch.Tensor] = None, check: bool = False,
                   stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """Adds to mass [pages, page_size, heads] (float32, any strides; empty_mass) the attention weight that
    each key of the sequences' own pages gets from the queries q, summed over the tokens that see it and
    the query heads of its key head: mass = decay * mass + sum of exp(scale * q k - lse).  Returns mass.

    q (any strides, 0 too, as an expanded tensor has them), table, seq_len, q_indptr, the bounds, scale and
    causal are those of the prefix_attention call and lse [tokens, q_heads] what it returned (with lse=True); behind a prefix the own keys get their share
    of the whole softmax.  With ``causal`` the queries are the sequence's last tokens, whose keys start
    from nothing: what their slots held is not read.  decay=0 forgets all that came before.  To weigh a
    prompt by its last tokens, pass these as q, with seq_len of the whole prompt, and decay=0.

    No page may be in the table twice.  The cache's values are not read.  float16 or bfloat16, heads of
    64, 96, 128 or 256; scores and sums are 32-bit, in a fixed order.  ``workspace``:
    attention_mass_workspace_bytes, allocated on the call's stream where it is not given.  A call for
    serving: no gradient goes through it."""
    m, _held = _mass_args(mass, q, cache, table, seq_len, lse, q_indptr, max_q_len, max_seq_len, scale, causal, decay, check)
    index = q.get_device()
    sp = _stream(index, stream)
    where = _elsewhere(index, stream)
    if where is not None:
        with where:
            return _mass_launch(m, mass, q, workspace, index, sp)
    return _mass_launch(m, mass, q, workspace, index, sp)


def _mass_launch(m, mass, q, workspace, index, sp):
    need = _call("tg_attention_mass_needed_bytes")(m)
    ws = size = 0
    if workspace is None and need:
        workspace, size = torch.empty(need, dtype=torch.uint8, device=q.device), need
        ws = workspace.data_ptr()
    elif workspace is not None:
        ws, size = _workspace(workspace, need, index)
    _lib.check(_call("tg_attention_mass_" + _SUFFIX[q.dtype])(m, ws, size, sp), "tg_attention_mass")
    return mass


def attention_mass_workspace_bytes(q: torch.Tensor, cache: PagedKV, table: PageTable, seq_len: torch.Tensor,
                                   q_indptr: Optional[torch.Tensor] = None, max_q_len: Optional[int] = None) -> int:
    """Bytes of a workspace to keep for attention_mass: enough for this call and every one of the same
    heads with no larger max_q_len, however many its tokens (0 for few rows).  max_q_len counts without a
    q_indptr too, for calls with one that follow."""
    m, _held = _mass_args(None, q, cache, table, seq_len, None, q_indptr, max_q_len, None, None, True, 1.0, False)
    if max_q_len is not None:
        m.max_q_len = max_q_len
    return int(_call("tg_attention_mass_workspace_bytes")(m))


def _evict_args(cache, table, seq_len, budget, first, recent, max_seq_len, check):
    kv = cache.desc()
    index = cache.k.get_device()
    tb = table.desc(index, kv.pages)
    slots = tb.nnz * kv.page_size
    a = _lib.TgKvEvictArgs(ctypes.addressof(kv), ctypes.addressof(tb), _vector(seq_len, "seq_len", index, tb.rows),
                           slots if max_seq_len is None else max_seq_len, budget, first, recent)
    a.flags = _lib.TG_FLAG_BOUNDS_CHECK if check else 0
    return a, (kv, tb), max(0, min(budget, slots, a.max_seq_len))


def kv_evict(cache: PagedKV, table: PageTable, seq_len: torch.Tensor, mass: torch.Tensor, budget: int, first: int = 0,
             recent: int = 0, max_seq_len: Optional[int] = None, mass_out: Optional[torch.Tensor] = None,
             kept: Union[bool, torch.Tensor] = False, seq_len_out: Optional[torch.Tensor] = None,
             workspace: Optional[torch.Tensor] = None, check: bool = False, stream: Optional[torch.cuda.Stream] = None):
    """Cuts every sequence longer than budget to it, in place, and returns the new lengths (int64;
    seq_len_out, which may be seq_len, or a new tensor).

    For each key head by itself the first `first` keys, the last `recent` ones and, of those between,
    the ones with the largest mass [pages, page_size, heads] stay: equal ones from the lowest place on,
    NaN counts as the largest.  Where the budget is smaller than first + recent, recent goes first.  The
    first keys stay in place; chosen ones that lie within the next budget - first - recent places stay,
    the others fill the free places there, in order; the recent ones follow, in order.  So the order of
    a sequence's keys changes between `first` and `recent`, which attention does not see: keys carry
    their positions.  From then on new tokens' positions are not their places, and kv_append takes
    ``positions``.  Moving the recent keys costs their bytes each time: a server lets sequences grow some
    tokens over their budget and evicts every few steps.

    Keys, values and mass move together; with mass_out (same shape, any strides) the mass of all kept
    keys is written there and mass itself is not changed.  ``kept=True`` (or an int32 [sequences, heads,
    width] tensor, width at least min(budget, max_seq_len)) returns (lengths, old place of each new one,
    -1 behind the length).  Pages behind the new length may be given back; what they and the rest of the
    last page hold is undefined.  No page may be in the table twice.  max_seq_len bounds the lengths (a
    longer sequence counts as that long; default: what the listed pages hold).  ``workspace``:
    kv_evict_workspace_bytes, allocated on the call's stream where it is not given.  No gradient goes
    through it."""
    a, _held, width = _evict_args(cache, table, seq_len, budget, first, recent, max_seq_len, check)
    index = cache.k.get_device()
    a.mass = _mass_desc(mass, "mass", cache, index)
    if mass_out is not None and mass_out is not mass:
        a.mass_out = _mass_desc(mass_out, "mass_out", cache, index)
        if a.mass_out.data == a.mass.data and any(
                n > 1 and x != y for n, x, y in zip(mass.shape, mass.stride(), mass_out.stride())):
            raise ValueError("mass_out must be mass or not share memory with it")
    sp = _stream(index, stream)
    where = _elsewhere(index, stream)
    if where is not None:
        with where:
            return _evict_launch(a, seq_len, seq_len_out, kept, width, workspace, cache, index, sp)
    return _evict_launch(a, seq_len, seq_len_out, kept, width, workspace, cache, index, sp)


def _evict_launch(a, seq_len, seq_len_out, kept, width, workspace, cache, index, sp):
    if seq_len_out is None:
        seq_len_out = torch.empty_like(seq_len)
    a.seq_len_out = _vector(seq_len_out, "seq_len_out", index, seq_len.shape[0])
    shape = (seq_len.shape[0], cache.k.shape[2])
    if kept is True:
        kept = torch.empty(*shape, width, dtype=torch.int32, device=seq_len.device)
    if isinstance(kept, torch.Tensor):
        if kept.dim() != 3 or kept.shape[:2] != shape or kept.shape[2] < width or kept.dtype is not torch.int32 \
                or kept.get_device() != index or not kept.is_contiguous():
            raise ValueError("kept must be a contiguous int32 tensor [%d, %d, at least %d] on cuda:%d (got %s %s on %s)"
                             % (*shape, width, index, tuple(kept.shape), kept.dtype, kept.device))
        a.kept, a.kept_width = kept.data_ptr(), kept.shape[2]
    need = _call("tg_kv_evict_workspace_bytes")(a)
    ws = size = 0
    if workspace is None and need:
        workspace, size = torch.empty(need, dtype=torch.uint8, device=seq_len.device), need
        ws = workspace.data_ptr()
    elif workspace is not None:
        ws, size = _workspace(workspace, need, index)
    _lib.check(_call("tg_kv_evict_" + _SUFFIX[cache.k.dtype])(a, ws, size, sp), "tg_kv_evict")
    return (seq_len_out, kept) if isinstance(kept, torch.Tensor) else seq_len_out


def kv_evict_workspace_bytes(cache: PagedKV, table: PageTable, seq_len: torch.Tensor, budget: int,
                             max_seq_len: Optional[int] = None) -> int:
    """Bytes of a workspace to keep for kv_evict: enough for any call of the same budget on this cache with
    no more sequences and listed pages and no larger max_seq_len."""
    a, _held, _ = _evict_args(cache, table, seq_len, budget, 0, 0, max_seq_len, False)
    return int(_call("tg_kv_evict_workspace_bytes")(a))
