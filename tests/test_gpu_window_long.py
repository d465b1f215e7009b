"""Attention with a sliding window and sinks on long sequences: more key tiles than tables hold, offsets beyond 32 bits. The definition in 64
bits, piece by piece, and the bounds of test_gpu_window.py."""
import pytest
import torch

import flash_sparse_attn as fsa
from test_gpu_window import check

pytestmark = pytest.mark.gpu


def pieces(q, k, v, dout, window, sinks, mask=None, rows=2000):
    """(out, dq, dk, dv) and a bound of each for tensors (1, S, heads, d) with as many kv heads; mask (S,)."""
    u = torch.finfo(q.dtype).eps / 2 + 3e-5
    S, scale = q.shape[1], q.shape[-1] ** -0.5
    q, k, v, g = (x[0].detach().transpose(0, 1).double() for x in (q, k, v, dout))
    res, off = ([torch.zeros_like(q) for _ in range(4)] for _ in range(2))
    for a in range(0, S, rows):
        b = min(S, a + rows)
        lo = max(0, a - window + 1)
        j = torch.cat([torch.arange(min(sinks, lo), device="cuda"), torch.arange(lo, b, device="cuda")])
        t = torch.arange(a, b, device="cuda")[:, None]
        seen = (j <= t) & ((t - j < window) | (j < sinks))
        if mask is not None:
            seen = seen & mask[j]
        Q, K, V, G = q[:, a:b], k[:, j], v[:, j], g[:, a:b]
        p = torch.nan_to_num(torch.softmax((Q @ K.mT * scale).masked_fill(~seen, -torch.inf), -1), nan=0.0)
        out = p @ V
        o_off = (u * p) @ V.abs() + u * out.abs()
        dp = G @ V.mT
        ds = p * (dp - (G * out).sum(-1, keepdim=True))
        ds_off = u * ds.abs() + p * ((G.abs() * o_off).sum(-1, keepdim=True) + 3e-5 * (G.abs() @ V.abs().mT))
        res[0][:, a:b], off[0][:, a:b] = out, o_off
        dq = ds @ K * scale
        res[1][:, a:b], off[1][:, a:b] = dq, ds_off @ K.abs() * scale + u * dq.abs()
        for x, y in ((res[2], ds.mT @ Q * scale), (off[2], ds_off.mT @ Q.abs() * scale), (res[3], p.mT @ G), (off[3], (u + 3e-5) * p.mT @ G.abs())):
            x.index_add_(1, j, y)
    for i in (2, 3):
        off[i] += u * res[i].abs()
    return [x.transpose(0, 1)[None] for x in res], [x.transpose(0, 1)[None] for x in off]


def inputs(S, H, d):
    g = torch.Generator(device="cuda").manual_seed(S)
    return [torch.randn((1, S, H, d), generator=g, device="cuda", dtype=torch.bfloat16).requires_grad_(i < 3) for i in range(4)]


@pytest.mark.parametrize("S,H,d,window,sinks", [(270001, 2, 64, 300, 5), (263000, 1, 128, 1, 140), (270001, 1, 256, 70, 2)])
@pytest.mark.parametrize("masked", [False, True])
def test_more_tiles_than_tables_hold(S, H, d, window, sinks, masked):
    q, k, v, dout = inputs(S, H, d)
    mask = torch.rand(S, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") < 0.7 if masked else None
    out = fsa.flash_sparse_attn_window_func(q, k, v, window, sinks, attn_mask=mask[None, None, None] if masked else None)
    check([out, *torch.autograd.grad(out, (q, k, v), dout)], *pieces(q, k, v, dout, window, sinks, mask))


def test_offsets_beyond_32_bits():
    """More than 2^31 elements a tensor; the last head is compared."""
    S, H, d, window, sinks = 270001, 64, 128, 100, 2
    q, k, v, dout = inputs(S, H, d)
    assert q.numel() > 2 ** 31
    out = fsa.flash_sparse_attn_window_func(q, k, v, window, sinks)
    got = [x[:, :, -1:].clone() for x in (out, *torch.autograd.grad(out, (q, k, v), dout))]
    check(got, *pieces(*(x.detach()[:, :, -1:] for x in (q, k, v, dout)), window, sinks))


def test_a_long_packed_sequence():
    S, H, d, window, sinks = 270001, 1, 64, 500, 3
    q, k, v, dout = inputs(S, H, d)
    q, k, v = (x.detach()[0].requires_grad_() for x in (q, k, v))
    cuts = [0, 1000, 1001, S]
    cu = torch.tensor(cuts, dtype=torch.int32, device="cuda")
    out = fsa.flash_sparse_attn_window_varlen_func(q, k, v, cu, cu, S, S, window, sinks)
    got = [out, *torch.autograd.grad(out, (q, k, v), dout[0])]
    for a, b in zip(cuts, cuts[1:]):
        check([x[None, a:b] for x in got], *pieces(*(x.detach()[None, a:b] for x in (q, k, v, dout[0])), window, sinks))
