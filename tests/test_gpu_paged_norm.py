"""Norms of queries and keys with the rotation in the same pass: forward, on the way into the paged
cache, and the gradient, against plain implementations in 64 bits.

Bounds, derived before the first run.  u is half an ulp of the type relative to the value (2^-8
bfloat16, 2^-11 float16, 2^-24 float32; float16 below 2^-14 has an absolute 2^-25).

* Forward: the sum of at most 256 squares and its root have a relative error below 2^-18 (a chain of at
  most 16 and a tree), product, weight and rotation a few 2^-24 more (sine, cosine and reduced angle
  2^-22).  With the pair a, b that is turned: u |y| + 2^-17 scale (|a| + |b|).
* dx = r (g' - xh m): the same relative errors of each of its terms, m's among them:
  u |dx| + 2^-16 r (|g'| + |xh| mean |g' xh|), |g'| standing for w scale (|da| + |db|).
* A weight's gradient adds n terms t, in chains of at most n / 16 + 64: u |dw| +
  (2^-16 + (n / 16 + 64) 2^-24) sum |t|.
"""

from __future__ import annotations

import math

import pytest
import torch

from tilegen_b200 import lib
from tilegen_b200 import paged as P

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
U = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F32: 2.0 ** -140, F16: 2.0 ** -25, BF16: 2.0 ** -130}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def pairs(n, layout):
    return (slice(0, n), slice(n, 2 * n)) if layout == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))


def turn64(y, r, pos, sign=1):
    """(y rotated, size of what each element was made of), 64 bits."""
    if r is None:
        return y, y.abs()
    n = r.freq.numel()
    t = (pos.double()[:, None] * r.freq)[:, None]
    c, s = t.cos() * r.scale, t.sin() * r.scale * sign
    ia, ib = pairs(n, r.layout)
    z, mag = y.clone(), y.abs()
    a, b = y[..., ia], y[..., ib]
    z[..., ia], z[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia] = mag[..., ib] = (a.abs() + b.abs()) * abs(r.scale)
    return z, mag


def norm64(x, norm):
    """(x normed, xh, r, factor), 64 bits."""
    x = x.double()
    if norm is None:
        one = torch.ones_like(x[..., :1])
        return x, x, one, one
    r = 1 / (x.square().mean(-1, keepdim=True) + norm.eps).sqrt()
    w = torch.ones(x.shape[-1], dtype=torch.float64, device="cuda") if norm.weight is None else norm.offset + norm.weight.double()
    return x * r * w, x * r, r, w


def check_forward(y, x, norm, r, pos):
    ref, mag = turn64(norm64(x, norm)[0], r, pos)
    tol = U[y.dtype] * ref.abs() + 2.0 ** -17 * mag + TINY[y.dtype]
    err = (y.double() - ref).abs()
    assert bool((err <= tol).all()), "worst %g of its bound" % float((err / tol).max())


def check_gradient(dx, dw, dy, x, norm, r, pos):
    g, gm = turn64(dy.double(), r, pos, -1)
    _, xh, root, w = norm64(x, norm)
    if norm is None:
        ref, tol = g, 2.0 ** -17 * gm
    else:
        ref = root * (g * w - xh * (g * w * xh).mean(-1, keepdim=True))
        tol = 2.0 ** -16 * root * (gm * w.abs() + xh.abs() * (gm * w.abs() * xh.abs()).mean(-1, keepdim=True))
    tol = tol + U[dx.dtype] * ref.abs() + TINY[dx.dtype]
    err = (dx.double() - ref).abs()
    assert bool((err <= tol).all()), "worst %g of its bound" % float((err / tol).max())
    if norm is None or norm.weight is None:
        assert dw is None
        return
    n = x.shape[0] * x.shape[1]
    ref, size = (g * xh).sum((0, 1)), (gm * xh.abs()).sum((0, 1))
    tol = U[dw.dtype] * ref.abs() + (2.0 ** -16 + (n / 16 + 64) * 2.0 ** -24) * size + TINY[dw.dtype]
    err = (dw.double() - ref).abs()
    assert dw.dtype == norm.weight.dtype and bool((err <= tol).all()), "worst %g of its bound" % float((err / tol).max())


SHAPES = [  # tokens, heads, key heads, dim, rotating
    (1, 1, 1, 2, 2), (1, 32, 8, 128, 128), (5, 3, 1, 80, 40), (7, 5, 5, 96, 48), (33, 2, 1, 20, 12), (130, 8, 2, 64, 64),
    (3, 1, 1, 36, 0), (1201, 4, 1, 128, 32), (9, 40, 8, 256, 256), (64, 1, 1, 7, 4), (2000, 1, 0, 64, 64), (301, 0, 3, 72, 72),
    (517, 6, 2, 250, 124), (40, 3, 3, 1, 0), (300, 3, 1, 32, 32), (2500, 16, 4, 128, 128),
]


def problem(case, dtype, layout, wide=False):
    tokens, heads, kv, dim, rot = case
    g = gen(tokens * 1000 + dim)
    q, k = normal(g, tokens, heads, dim, dtype=dtype) * 3, normal(g, tokens, kv, dim, dtype=dtype)
    wt = F32 if wide else dtype
    norms = P.HeadNorm((1 + 0.3 * normal(g, dim)).to(wt), 1e-6), P.HeadNorm((0.3 * normal(g, dim)).to(wt), 1e-5, 1.0)
    r = P.Rope(P.rope_frequencies(rot, scaling="banded", factor=4.0), layout, 1.25)
    pos = torch.randint(0, 1 << 20, (tokens,), generator=g, device="cuda")
    return g, q, k, norms, r, pos


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("case", SHAPES)
def test_forward_and_gradient(case, layout, dtype):
    g, q, k, (qn, kn), r, pos = problem(case, dtype, layout, wide=case[0] % 2 == 0)
    y, z = P.norm_rope(q, k, qn, kn, r, pos)
    check_forward(y, q, qn, r, pos)
    check_forward(z, k, kn, r, pos)
    dy, dz = normal(g, *q.shape, dtype=dtype), normal(g, *k.shape, dtype=dtype)
    dq, dk, dqw, dkw = P.norm_rope_backward(dy, dz, q, k, qn, kn, r, pos)
    check_gradient(dq, dqw, dy, q, qn, r, pos)
    check_gradient(dk, dkw, dz, k, kn, r, pos)
    again = P.norm_rope_backward(dy, dz, q, k, qn, kn, r, pos)
    assert all(torch.equal(a, b) for a, b in zip((dq, dk, dqw, dkw), again))  # the same twice
    # in place
    q2, k2, dy2, k3 = q.clone(), k.clone(), dy.clone(), k.clone()
    assert P.norm_rope(q2, k2, qn, kn, r, pos, q_out=q2, k_out=k2)[0] is q2
    assert torch.equal(q2, y) and torch.equal(k2, z)
    P.norm_rope_backward(dy2, dz, q, k3, qn, kn, r, pos, dq=dy2, dk=k3)
    assert torch.equal(dy2, dq) and torch.equal(k3, dk)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_parts_left_out(dtype):
    """No key tensor, no norm of one, no weight, no rotation."""
    g, q, k, (qn, kn), r, pos = problem((70, 6, 2, 64, 32), dtype, "half")
    dy, dz = normal(g, *q.shape, dtype=dtype), normal(g, *k.shape, dtype=dtype)
    bare = P.HeadNorm(None, 1e-3, 5.0)  # the offset belongs to the weight
    for norms, rope in (((qn, None), r), ((None, kn), r), ((qn, kn), None), ((bare, bare), r), ((None, bare), None)):
        y, z = P.norm_rope(q, k, *norms, rope, pos if rope else None)
        check_forward(y, q, norms[0], rope, pos)
        check_forward(z, k, norms[1], rope, pos)
        dq, dk, dqw, dkw = P.norm_rope_backward(dy, dz, q, k, *norms, rope, pos if rope else None)
        check_gradient(dq, dqw, dy, q, norms[0], rope, pos)
        check_gradient(dk, dkw, dz, k, norms[1], rope, pos)
    y, z = P.norm_rope(q, None, qn, None, r, pos)
    assert z is None and torch.equal(y, P.norm_rope(q, k, qn, kn, r, pos)[0])
    dq, dk, dqw, dkw = P.norm_rope_backward(dy, None, q, None, qn, None, r, pos)
    assert dk is None and dkw is None
    check_gradient(dq, dqw, dy, q, qn, r, pos)
    # what neither turns nor is normed comes back as it was
    assert torch.equal(P.norm_rope(q, k)[0], q) and torch.equal(P.norm_rope(q, k, qn)[1], k)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim", [64, 80, 128])
def test_strides(layout, dim):
    """Views of a joint projection, heads first, outputs inside a larger buffer, rows off the 16-byte
    grid and off the 8-byte grid, gradients of expanded numbers."""
    g = gen(3)
    r = P.Rope(P.rope_frequencies(dim), layout)
    qn, kn = P.HeadNorm(normal(g, dim)), P.HeadNorm(normal(g, dim, dtype=BF16))
    pos = torch.arange(50, device="cuda") * 77
    qkv = normal(g, 50, 8, dim, dtype=BF16)
    q, k = qkv[:, :5], qkv[:, 5:7]
    want = P.norm_rope(q.contiguous(), k.contiguous(), qn, kn, r, pos)
    grads = P.norm_rope_backward(*want, q.contiguous(), k.contiguous(), qn, kn, r, pos)
    for off in (0, 1, 4):
        shift = torch.empty(50 * 8 * dim + off, dtype=BF16, device="cuda")[off:].view(50, 8, dim).copy_(qkv)
        heads_first = shift.transpose(0, 1).contiguous().transpose(0, 1)
        buf = torch.full((50, 6, dim + 8 + off), 7.0, dtype=BF16, device="cuda")
        out = buf[:, :5, off:off + dim]
        for x in (shift, heads_first):
            got = P.norm_rope(x[:, :5], x[:, 5:7], qn, kn, r, pos, q_out=out)
            assert got[0] is out
            check_forward(out, q, qn, r, pos)
            check_forward(got[1], k, kn, r, pos)
            assert bool((buf[:, 5] == 7).all()) and bool((buf[..., off + dim:] == 7).all())
            back = P.norm_rope_backward(*want, x[:, :5], x[:, 5:7], qn, kn, r, pos)
            for a, b in zip(back, grads):
                assert torch.allclose(a.float(), b.float(), rtol=2.0 ** -7, atol=2.0 ** -7 * float(b.float().abs().max()))
    one = torch.ones((), dtype=BF16, device="cuda")
    dq, dk, dqw, dkw = P.norm_rope_backward(one.expand(50, 5, dim), one.expand(50, 2, dim), q, k, qn, kn, r, pos)
    check_gradient(dq, dqw, torch.ones(50, 5, dim, dtype=BF16, device="cuda"), q, qn, r, pos)
    check_gradient(dk, dkw, torch.ones(50, 2, dim, dtype=BF16, device="cuda"), k, kn, r, pos)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_gradient_against_autograd_and_differences(layout):
    g = gen(11)
    q, dy = normal(g, 6, 3, 24), normal(g, 6, 3, 24)
    pos = torch.randint(0, 5000, (6,), generator=g, device="cuda")
    r = P.Rope(P.rope_frequencies(16), layout, 0.75)
    w = normal(g, 24)
    norm = P.HeadNorm(w, 1e-2, 1.0)
    dq, _, dw, _ = P.norm_rope_backward(dy, None, q, None, norm, None, r, pos)

    def loss(x, weight):  # the formula, in 64 bits
        y = x / (x.square().mean(-1, keepdim=True) + 1e-2).sqrt() * (1.0 + weight)
        return (turn64(y, r, pos)[0] * dy.double()).sum()

    leaf, lw = q.double().requires_grad_(), w.double().requires_grad_()
    gx, gw = torch.autograd.grad(loss(leaf, lw), (leaf, lw))
    assert float((dq - gx).abs().max()) < 2.0 ** -18 * float(gx.abs().max()) * 24
    assert float((dw - gw).abs().max()) < 2.0 ** -18 * float(gw.abs().max()) * 24
    # a central difference of step h in 64 bits is off by h^2 / 6 of the third derivative
    h = 1e-4
    sx, sw = normal(g, 6, 3, 24).double(), normal(g, 24).double()
    num = (loss(q.double() + h * sx, w.double() + h * sw) - loss(q.double() - h * sx, w.double() - h * sw)) / (2 * h)
    ana = (dq.double() * sx).sum() + (dw.double() * sw).sum()
    assert abs(float(num - ana)) < 1e-4 * float((dq.double() * sx).abs().sum() + (dw.double() * sw).abs().sum())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_autograd(dtype):
    """The gradients that reach a joint projection and shared weights, on the call's stream; without a
    gradient asked for, none."""
    g, q, k, (qn, kn), r, pos = problem((33, 4, 2, 64, 40), dtype, "half")
    qkv = torch.cat((q, k, k), 1).requires_grad_()
    qw, kw = qn.weight.requires_grad_(), kn.weight.requires_grad_()
    dy, dz = normal(g, *q.shape, dtype=dtype), normal(g, *k.shape, dtype=dtype)
    want = P.norm_rope_backward(dy, dz, q, k, qn, kn, r, pos)
    st = torch.cuda.Stream()
    for stream in (None, st):
        if stream:
            st.wait_stream(torch.cuda.current_stream())
        y, z = P.norm_rope(qkv[:, :4], qkv[:, 4:6], qn, kn, r, pos, stream=stream)
        if stream:
            torch.cuda.current_stream().wait_stream(st)
        gx, gq, gk = torch.autograd.grad((y, z), (qkv, qw, kw), (dy, dz))
        assert torch.equal(gx[:, :4], want[0]) and torch.equal(gx[:, 4:6], want[1]) and not bool(gx[:, 6:].any())
        assert torch.equal(gq, want[2]) and torch.equal(gk, want[3])
    # one weight shared by both, one output used
    shared = P.HeadNorm(qw, 1e-6)
    y, z = P.norm_rope(qkv[:, :4], qkv[:, 4:6], shared, shared, r, pos)
    (gw,) = torch.autograd.grad(z, qw, dz)
    assert torch.equal(gw, P.norm_rope_backward(dy, dz, q, k, shared, shared, r, pos)[3])
    y, none = P.norm_rope(qkv[:, :4], None, qn)
    assert none is None
    (gx,) = torch.autograd.grad(y.sum(), qkv)
    assert torch.equal(gx[:, :4], P.norm_rope_backward(torch.ones_like(y), None, q, None, qn)[0])
    with torch.no_grad():
        assert not P.norm_rope(qkv[:, :4], None, qn)[0].requires_grad
    assert not P.norm_rope(qkv[:, :4], None, qn, q_out=torch.empty_like(y))[0].requires_grad
    with pytest.raises(RuntimeError):  # differentiable once
        torch.autograd.grad(torch.autograd.grad(P.norm_rope(qkv[:, :4], None, qn)[0].sum(), qkv, create_graph=True)[0].sum(), qkv)


def test_rows_of_zeros_infinities_and_nan():
    """A row's trouble stays its own; a row of zeros gives zeros and a finite gradient."""
    g, q, k, (qn, kn), r, pos = problem((20, 4, 2, 128, 128), BF16, "half")
    clean = P.norm_rope(q, k, qn, kn, r, pos)
    q2 = q.clone()
    q2[3, 1] = 0
    q2[5, 2, 7] = math.nan
    q2[6, 0, 9] = math.inf
    y, z = P.norm_rope(q2, k, qn, kn, r, pos)
    assert not bool(y[3, 1].any()) and bool(y[5, 2].isnan().all()) and not bool(y[6, 0].isfinite().all())
    assert torch.equal(z, clean[1])
    keep = torch.ones(20, 4, dtype=torch.bool, device="cuda")
    keep[3, 1] = keep[5, 2] = keep[6, 0] = False
    assert torch.equal(y[keep], clean[0][keep])
    dy = normal(g, *q.shape, dtype=BF16)
    dq = P.norm_rope_backward(dy, z, q2, k, qn, kn, r, pos)
    assert torch.equal(dq[0][keep], P.norm_rope_backward(dy, z, q, k, qn, kn, r, pos)[0][keep])
    assert bool(dq[0][3, 1].isfinite().all()) and bool(dq[2].isnan().all()) and bool(dq[3].isfinite().all())


def test_empty():
    w = torch.ones(64, device="cuda", requires_grad=True)
    x = torch.zeros(0, 3, 64, device="cuda")
    y, z = P.norm_rope(x, x[:, :1], P.HeadNorm(w), P.HeadNorm(w))
    assert y.shape == x.shape and z.shape == (0, 1, 64)
    (gw,) = torch.autograd.grad(y.sum() + z.sum(), w)
    assert not bool(gw.any())
    x = torch.zeros(4, 0, 64, device="cuda")
    dq, _, dw, _ = P.norm_rope_backward(x, None, x, None, P.HeadNorm(w.detach()))
    assert dq.shape == x.shape and not bool(dw.any())


# ------------------------------------------------------------------ on the way into the cache
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("layout,dim,rot,page", [("half", 128, 128, 16), ("interleaved", 64, 32, 7), ("half", 80, 40, 24)])
@pytest.mark.parametrize("norms", ["qk", "q", "k"])
def test_append(norms, layout, dim, rot, page, dtype):
    g = gen(dim + page)
    news, lens, heads, kv = [3, 0, 1, 40], [3, 5, 200, 61], 6, 2
    total = sum(news)
    own = [-(-n // page) for n in lens]
    order = torch.randperm(sum(own) + 2, generator=g, device="cuda").tolist()
    rows = [[order.pop() for _ in range(n)] for n in own]
    table = P.PageTable.from_lists(rows)
    kc, vc = (normal(g, sum(own) + 2, kv, page, dim, dtype=dtype).transpose(1, 2) for _ in range(2))
    cache = P.PagedKV(kc, vc)
    before = kc.clone(), vc.clone()
    qkv = normal(g, total, heads + 2 * kv, dim, dtype=dtype)
    q, k, v = qkv.split((heads, kv, kv), 1)
    qn = P.HeadNorm(normal(g, dim)) if "q" in norms else None
    kn = P.HeadNorm(normal(g, dim, dtype=dtype), 1e-3, 1.0) if "k" in norms else None
    r = P.Rope(P.rope_frequencies(rot), layout, 1.5)
    seq_len = torch.tensor(lens, device="cuda")
    indptr = torch.tensor([0] + news, device="cuda").cumsum(0)
    out = P.kv_append(cache, table, seq_len, k, v, rope=r, q=q, q_indptr=indptr, position_base=11, q_norm=qn, k_norm=kn,
                      check=True)
    t = 0
    for pages, n, length in zip(rows, news, lens):
        pos = torch.arange(length - n, length, device="cuda")
        check_forward(out[t:t + n], q[t:t + n], qn, r, pos + 11)
        if n:
            at = torch.tensor(pages, device="cuda")[pos // page], pos % page
            check_forward(kc[at], k[t:t + n], kn, r, pos + 11)
            assert torch.equal(vc[at], v[t:t + n])
            for x, old in zip((kc, vc), before):
                old[at] = x[at]
        t += n
    assert torch.equal(kc, before[0]) and torch.equal(vc, before[1])  # nothing else was written
    # the same numbers as the norm and the append one after the other, to one rounding more
    q2, k2 = P.norm_rope(q, k, qn, kn)
    again = P.kv_append(cache, table, seq_len, k2, v, rope=r, q=q2, q_indptr=indptr, position_base=11)
    assert torch.allclose(again.float(), out.float(), rtol=2.0 ** -6, atol=2.0 ** -6 * float(out.float().abs().max()))


def test_append_single_tokens_bad_pages_and_no_queries():
    g = gen(5)
    cache = P.PagedKV(*(torch.zeros(6, 16, 2, 64, device="cuda", dtype=BF16) for _ in range(2)))
    table = P.PageTable.from_lists([[1], [9], [3], [-1], [4]])  # two pages that do not exist
    seq_len = torch.tensor([1, 4, 99, 2, 16], device="cuda")     # one place past its pages
    k, v = normal(g, 5, 2, 64, dtype=BF16), normal(g, 5, 2, 64, dtype=BF16)
    kn = P.HeadNorm(normal(g, 64))
    assert P.kv_append(cache, table, seq_len, k, v, k_norm=kn) is None
    want = torch.zeros_like(cache.k)
    normed = P.norm_rope(k, None, kn)[0]
    want[1, 0], want[4, 15] = normed[0], normed[4]
    assert torch.equal(cache.k, want)
    with pytest.raises(lib.TgError) as e:
        P.kv_append(cache, table, seq_len, k, v, k_norm=kn, check=True)
    assert e.value.status == lib.TG_EBOUNDS


def test_graph_capture_and_streams():
    """Forward and gradient in a captured graph, new contents between replays, a kept workspace."""
    g, q, k, (qn, kn), r, pos = problem((65, 4, 2, 128, 128), BF16, "half")
    dy, dz = normal(g, *q.shape, dtype=BF16), normal(g, *k.shape, dtype=BF16)
    P.norm_rope_backward(dy, dz, q, k, qn, kn, r, pos)
    ws = torch.empty(P.norm_rope_backward_workspace_bytes(65, 128), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = P.norm_rope(q, k, qn, kn, r, pos)
        back = P.norm_rope_backward(dy, dz, q, k, qn, kn, r, pos, workspace=ws)
    for seed in (1, 2):
        q.copy_(normal(gen(seed), *q.shape))
        pos.add_(seed)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, P.norm_rope(q, k, qn, kn, r, pos)))
        assert all(torch.equal(a, b) for a, b in zip(back, P.norm_rope_backward(dy, dz, q, k, qn, kn, r, pos)))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    other = P.norm_rope(q, k, qn, kn, r, pos, stream=st)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(other[0], out[0])


def test_one_row_for_all_tokens():
    """Inputs with strides of zero, as an expanded tensor has them."""
    g, q, k, (qn, kn), r, pos = problem((90, 5, 2, 128, 128), BF16, "half")
    wide = q[:1, :1].expand(90, 5, 128)
    check_forward(P.norm_rope(wide, k, qn, kn, r, pos)[0], wide.contiguous(), qn, r, pos)
    one = q[:1, :1].clone().requires_grad_()
    y, _ = P.norm_rope(one.expand(90, 5, 128), None, qn, None, r, pos)
    dy = normal(g, 90, 5, 128, dtype=BF16)
    (gx,) = torch.autograd.grad(y, one, dy)
    each = P.norm_rope_backward(dy, None, wide, None, qn, None, r, pos)[0]
    assert torch.equal(gx, each.sum((0, 1), keepdim=True))


def test_a_training_step_in_a_captured_graph():
    """Forward and gradient by autograd, captured with no eager graph of the same leaves alive."""
    g, q, k, (qn, kn), r, pos = problem((40, 4, 2, 64, 64), BF16, "half")
    dy, dz = normal(g, *q.shape, dtype=BF16), normal(g, *k.shape, dtype=BF16)
    want = P.norm_rope_backward(dy, dz, q, k, qn, kn, r, pos)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        leaves = [t.clone().requires_grad_() for t in (q, k, qn.weight, kn.weight)]
        norms = P.HeadNorm(leaves[2], qn.eps, qn.offset), P.HeadNorm(leaves[3], kn.eps, kn.offset)

        def step():
            return torch.autograd.grad(P.norm_rope(leaves[0], leaves[1], *norms, r, pos), leaves, (dy, dz))

        step()
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        grads = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(grads, want))


def test_refusals():
    g, q, k, (qn, kn), r, pos = problem((4, 3, 1, 64, 64), BF16, "half")
    dy, dz = torch.empty_like(q), torch.empty_like(k)
    short = P.HeadNorm(qn.weight[:63])
    for bad in (lambda: P.norm_rope(q.double(), k, qn, kn, r, pos), lambda: P.norm_rope(q, k.float(), qn, kn, r, pos),
                lambda: P.norm_rope(q, k[:3], qn, kn, r, pos), lambda: P.norm_rope(q, k, short, kn, r, pos),
                lambda: P.norm_rope(q, k, P.HeadNorm(qn.weight.half()), kn, r, pos),
                lambda: P.norm_rope(q, k, P.HeadNorm(qn.weight.cpu()), kn, r, pos),
                lambda: P.norm_rope(q, k, qn, kn, r), lambda: P.norm_rope(q, k, qn, kn, r, pos[:3]),
                lambda: P.norm_rope(q, None, qn, kn, r, pos), lambda: P.norm_rope(q, None, qn, k_out=k),
                lambda: P.norm_rope(q.transpose(1, 2), None), lambda: P.norm_rope(q, k, qn, kn, r, pos, q_out=dy[:, :2]),
                lambda: P.norm_rope_backward(dy, None, q, k, qn, kn, r, pos), lambda: P.norm_rope_backward(dy, dz, q, None, qn),
                lambda: P.norm_rope_backward(dy[:3], dz, q, k, qn, kn, r, pos),
                lambda: P.norm_rope_backward(dy, dz, q, k, qn, kn, r, pos, workspace=torch.empty(8, dtype=torch.uint8, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    for bad, status in ((lambda: P.norm_rope(q, k, P.HeadNorm(eps=-1.0)), lib.TG_EINVAL),
                        (lambda: P.norm_rope(q, k, P.HeadNorm(eps=math.nan)), lib.TG_EINVAL),
                        (lambda: P.norm_rope(q[..., :32], k[..., :32], rope=r, positions=pos), lib.TG_EINVAL),
                        (lambda: P.norm_rope(torch.zeros(2, 1, 257, device="cuda")), lib.TG_EUNSUPPORTED)):
        with pytest.raises(lib.TgError) as e:
            bad()
        assert e.value.status == status
