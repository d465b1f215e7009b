"""Attention with a sliding window and sinks against its definition in 64 bits.

Bounds, element by element, from where the kernels round, with u = half a step of the type (and 3e-5 for 32-bit scores and exponentials):
probabilities and dS are rounded to the type before they enter a product, results once at the end, and D = rowsum(dO o O) is formed from
the rounded O. A probability below the least normal number of fp16 loses up to 2^-25.
"""
import math

import pytest
import torch

import flash_sparse_attn as fsa

pytestmark = pytest.mark.gpu


def reference(q, k, v, window, sinks, mask=None, scale=None, dout=None):
    """(out, dq, dk, dv) and a bound of each for tensors (B, S, heads, d), all in 64 bits."""
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    u = torch.finfo(q.dtype).eps / 2 + 3e-5
    q, k, v = (x.detach().double() for x in (q, k, v))
    B, Sq, H, d = q.shape
    Sk, Hk = k.shape[1:3]
    G = H // Hk
    scale = d ** -0.5 if scale is None else scale
    t = torch.arange(Sq, device=q.device)[:, None] + Sk - Sq
    j = torch.arange(Sk, device=q.device)[None, :]
    seen = ((j <= t) & ((t - j < window) | (j < sinks)))[None, None].expand(B, H, Sq, Sk)
    if mask is not None:
        m = mask.expand(B, mask.shape[1], 1, Sk)
        seen = seen & (m if m.shape[1] == 1 else m.repeat_interleave(H // m.shape[1], 1))
    qh, kh, vh = q.transpose(1, 2), k.transpose(1, 2).repeat_interleave(G, 1), v.transpose(1, 2).repeat_interleave(G, 1)
    x = (qh @ kh.transpose(-1, -2) * scale).masked_fill(~seen, -math.inf)
    p = torch.nan_to_num(torch.softmax(x, -1), nan=0.0)
    out = p @ vh
    # a row's largest probability is at least 2^-8 of the sum's unit when the others are rounded
    p_off = u * p + tiny * 256 * seen / seen.sum(-1, keepdim=True).clamp(min=1)
    o_off = p_off @ vh.abs() + u * out.abs()
    res, off = [out.transpose(1, 2)], [o_off.transpose(1, 2)]
    if dout is None:
        return res, off
    g = dout.double().transpose(1, 2)
    dp = g @ vh.transpose(-1, -2)
    D = (g * out).sum(-1, keepdim=True)
    ds = p * (dp - D)
    ds_off = u * ds.abs() + p * ((g.abs() * o_off).sum(-1, keepdim=True) + 3e-5 * (g.abs() @ vh.abs().transpose(-1, -2))) + tiny * seen

    def group(x):  # over the query heads of a kv head, (B, Sk, Hk, d)
        return x.view(B, Hk, G, Sk, d).sum(2).transpose(1, 2)

    dq = ds @ kh * scale
    dk = group(ds.transpose(-1, -2) @ qh) * scale
    dv = group(p.transpose(-1, -2) @ g)
    res += [dq.transpose(1, 2), dk, dv]
    off += [((ds_off @ kh.abs()) * scale + u * dq.abs()).transpose(1, 2),
            group(ds_off.transpose(-1, -2) @ qh.abs()) * scale + u * dk.abs(),
            group(((u + 3e-5) * p + tiny * seen).transpose(-1, -2) @ g.abs()) + u * dv.abs()]
    return res, off


def tensors(B, Sq, Sk, H, Hk, d, dtype, seed=0, grad=True):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=dtype)

    q, k, v, dout = rnd(B, Sq, H, d), rnd(B, Sk, Hk, d), rnd(B, Sk, Hk, d), rnd(B, Sq, H, d)
    return q.requires_grad_(grad), k.requires_grad_(grad), v.requires_grad_(grad), dout


def check(got, want, off):
    for name, x, y, e in zip(("out", "dq", "dk", "dv"), got, want, off):
        over = (x.detach().double() - y).abs() - e
        at = over.argmax()
        assert torch.isfinite(x).all(), name
        assert over.max() <= 1e-6, (name, float(over.max()), float(e.flatten()[at]), float(y.flatten()[at]))


def padding(B, Sk, heads=1, seed=0):
    """Keys that are there: a part of them, from the left or the right, and none at all in the last row where there are three."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    m = torch.rand((B, heads, 1, Sk), generator=g, device="cuda") < 0.8
    j = torch.arange(Sk, device="cuda")
    m[0] &= j < max(1, Sk - Sk // 3)
    if B > 1:
        m[1] &= j >= Sk // 4
    if B > 2:
        m[2] = False
    return m


# batch, queries, keys, heads, kv heads, head dim, window, sinks
GEOMETRIES = [
    (1, 1, 1, 1, 1, 64, 1, 0),
    (1, 1, 500, 2, 1, 64, 100, 3),
    (2, 5, 7, 2, 2, 32, 2, 1),
    (1, 130, 130, 4, 2, 64, 1, 0),       # a query sees itself alone
    (1, 200, 200, 2, 1, 128, 1, 200),    # sinks do the rest: plain causal
    (2, 300, 300, 4, 4, 128, 64, 4),
    (1, 513, 513, 6, 2, 96, 200, 130),   # sinks beyond a key tile
    (1, 385, 1500, 4, 1, 64, 300, 5),    # keys from before the first query
    (1, 700, 300, 2, 2, 64, 50, 2),      # queries before the first key: rows of zeros
    (3, 256, 256, 8, 2, 128, 128, 128),  # borders of the window on borders of the tiles
    (1, 4500, 4500, 4, 1, 64, 129, 1),   # sinks' gradients from several parts of the queries
    (1, 2300, 2300, 2, 1, 128, 1000, 300),
    (1, 400, 400, 3, 3, 72, 33, 0),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("geometry", GEOMETRIES, ids=str)
def test_forward_and_gradients(geometry, dtype):
    *shape, window, sinks = geometry
    q, k, v, dout = tensors(*shape, dtype)
    out = fsa.flash_sparse_attn_window_func(q, k, v, window, sinks)
    got = [out, *torch.autograd.grad(out, (q, k, v), dout)]
    check(got, *reference(q, k, v, window, sinks, dout=dout))


@pytest.mark.parametrize("heads", ["one", "kv", "query"])
@pytest.mark.parametrize("geometry", [(3, 300, 300, 4, 2, 64, 40, 3), (2, 600, 900, 6, 2, 128, 257, 140), (3, 1, 400, 4, 2, 64, 30, 2)], ids=str)
def test_masks_of_the_keys(geometry, heads):
    *shape, window, sinks = geometry
    q, k, v, dout = tensors(*shape, torch.bfloat16)
    mask = padding(shape[0], shape[2], {"one": 1, "kv": shape[4], "query": shape[3]}[heads])
    out = fsa.flash_sparse_attn_window_func(q, k, v, window, sinks, attn_mask=mask)
    check([out, *torch.autograd.grad(out, (q, k, v), dout)], *reference(q, k, v, window, sinks, mask, dout=dout))


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("geometry", [(1, 300, 300, 4, 1, 256, 70, 5), (2, 200, 333, 2, 2, 192, 300, 0), (1, 2500, 2500, 2, 1, 256, 130, 129),
                                      (1, 90, 40, 2, 1, 136, 9, 2)], ids=str)
def test_wide_heads(geometry, masked):
    *shape, window, sinks = geometry
    q, k, v, dout = tensors(*shape, torch.bfloat16)
    mask = padding(shape[0], shape[2]) if masked else None
    out = fsa.flash_sparse_attn_window_func(q, k, v, window, sinks, attn_mask=mask)
    check([out, *torch.autograd.grad(out, (q, k, v), dout)], *reference(q, k, v, window, sinks, mask, dout=dout))


def packed_reference(q, k, v, cu_q, cu_k, window, sinks, dout):
    parts = []
    for a, b, x, y in zip(cu_q, cu_q[1:], cu_k, cu_k[1:]):
        if y > x and b > a:
            parts.append(reference(q[None, a:b], k[None, x:y], v[None, x:y], window, sinks, dout=dout[None, a:b]))
        else:
            z = [torch.zeros((1, n) + t.shape[1:], dtype=torch.float64, device="cuda") for n, t in ((b - a, q), (b - a, q), (y - x, k), (y - x, v))]
            parts.append((z, z))
    return [[torch.cat([p[w][i][0] for p in parts]) for i in range(4)] for w in range(2)]


@pytest.mark.parametrize("lengths_q,lengths_k,window,sinks,d", [
    ([300, 1, 77, 500, 64], None, 60, 4, 64),
    ([128, 256, 3], None, 128, 130, 128),
    ([40] * 30, None, 16, 1, 32),
    ([2500, 30, 2200], None, 100, 3, 64),          # several parts of the queries beyond the window
    ([100, 7, 200], [300, 9, 200], 50, 2, 128),    # more keys than queries
    ([100, 50], [30, 50], 20, 1, 64),              # fewer: rows of zeros
    ([64, 0, 70], [64, 5, 70], 33, 65, 64),
], ids=str)
def test_packed_sequences(lengths_q, lengths_k, window, sinks, d):
    lengths_k = lengths_k or lengths_q
    cu_q, cu_k = ([sum(x[:i]) for i in range(len(x) + 1)] for x in (lengths_q, lengths_k))
    q, k, v, dout = (x[0].detach().requires_grad_(i < 3) for i, x in enumerate(tensors(1, cu_q[-1], cu_k[-1], 4, 2, d, torch.bfloat16)))
    cu = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (cu_q, cu_k)]
    out = fsa.flash_sparse_attn_window_varlen_func(q, k, v, *cu, max(lengths_q), max(lengths_k), window, sinks)
    check([out, *torch.autograd.grad(out, (q, k, v), dout)], *packed_reference(q, k, v, cu_q, cu_k, window, sinks, dout))


def test_packed_rows_outside_every_sequence_and_no_synchronisation():
    """Tokens before the first boundary and behind the last one, a boundary beyond the tensors; the call is captured, which a synchronisation
    would end."""
    T, window, sinks, lengths = 700, 40, 3, [200, 0, 1, 300]
    q, k, v, dout = (x[0].detach() for x in tensors(1, T, T, 4, 2, 64, torch.bfloat16))
    cu = [50 + sum(lengths[:i]) for i in range(len(lengths) + 1)]
    bounds = torch.tensor(cu, dtype=torch.int32, device="cuda")

    def run(q, k, v):
        q, k, v = (x.detach().requires_grad_() for x in (q, k, v))
        out = fsa.flash_sparse_attn_window_varlen_func(q, k, v, bounds, bounds, max(lengths), max(lengths), window, sinks)
        return [out, *torch.autograd.grad(out, (q, k, v), dout)]

    run(q, k, v)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        run(q, k, v)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            got = run(q, k, v)
    graph.replay()
    torch.cuda.synchronize()
    a, b = cu[0], cu[-1]
    inside = [x - a for x in cu]
    check([x[a:b] for x in got], *packed_reference(q[a:b], k[a:b], v[a:b], inside, inside, window, sinks, dout[a:b]))
    for x in got:
        assert not bool(x[:a].any()) and not bool(x[b:].any())
    bounds.copy_(torch.tensor([0, 100, 100, 400, 2 ** 30]))  # the last sequence ends where the tensors do
    graph.replay()
    torch.cuda.synchronize()
    check(got, *packed_reference(q, k, v, [0, 100, 100, 400, T], [0, 100, 100, 400, T], window, sinks, dout))
