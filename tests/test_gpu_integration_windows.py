"""`sliding_window`, as models hand it to the HuggingFace-style caller: dense, padded, packed and cached calls see the last so many keys, with a bias
and a dynamic mask too; a window that hides nothing changes nothing. Definition in 64 bits; bounds as in test_gpu_window.py (a bias adds its own
32-bit rounding to the scores)."""
import math

import pytest
import torch

import flash_sparse_attn as fsa
from flash_sparse_attn.integrations import CachedLayer, flash_sparse_attention_forward
from flash_sparse_attn.utils.mask import create_kept_keys, create_mask
from test_gpu_window import check, packed_reference, reference, tensors

pytestmark = pytest.mark.gpu


class Layer(torch.nn.Module):
    is_causal = True
    layer_idx = 0


def call(q, k, v, *args, **kw):
    return flash_sparse_attention_forward(Layer(), *(x.transpose(1, 2) for x in (q, k, v)), *args, **kw)[0]


def definition(q, k, v, seen, bias=None):
    """(out, bound) for keys that are `seen`, (B|1, H|1, Sq, Sk)."""
    u = torch.finfo(q.dtype).eps / 2 + 3e-5
    G = q.shape[2] // k.shape[2]
    q, k, v = q.double().transpose(1, 2), k.double().transpose(1, 2).repeat_interleave(G, 1), v.double().transpose(1, 2).repeat_interleave(G, 1)
    x = q @ k.mT * q.shape[-1] ** -0.5
    if bias is not None:
        x = x + bias.double().repeat_interleave(q.shape[1] // bias.shape[1], 1)
    p = torch.nan_to_num(x.masked_fill(~seen, -math.inf).softmax(-1), nan=0.0)
    out = p @ v
    return [out.transpose(1, 2)], [(u * p @ v.abs() + u * out.abs()).transpose(1, 2)]


def visible(Sq, Sk, window):
    t, j = torch.arange(Sk - Sq, Sk, device="cuda")[:, None], torch.arange(Sk, device="cuda")
    return ((j <= t) & (t - j < window))[None, None]


@pytest.mark.parametrize("Sq,Sk,d", [(300, 300, 64), (90, 400, 128), (1, 500, 64), (200, 200, 256)])
@pytest.mark.parametrize("window", [1, 70])
def test_dense(Sq, Sk, d, window):
    q, k, v, dout = tensors(2, Sq, Sk, 4, 2, d, torch.bfloat16)
    out = call(q, k, v, None, None, sliding_window=window)
    check([out, *torch.autograd.grad(out, (q, k, v), dout)], *reference(q, k, v, window, 0, dout=dout))


@pytest.mark.parametrize("heads", [1, 2, 4])
@pytest.mark.parametrize("d", [64, 256])
def test_dense_with_a_mask_of_the_keys(heads, d):
    q, k, v, dout = tensors(2, 260, 260, 4, 2, d, torch.bfloat16)
    mask = torch.rand((2, heads, 1, 260), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") < 0.7
    out = call(q, k, v, mask, None, sliding_window=50)
    check([out, *torch.autograd.grad(out, (q, k, v), dout)], *reference(q, k, v, 50, 0, mask, dout=dout))


@pytest.mark.parametrize("rows", ["keys", "queries"])
@pytest.mark.parametrize("kept", [None, 60])
def test_dense_with_a_bias(rows, kept):
    """Of the keys that the bias keeps those in the window; gradients reach the bias."""
    B, S, H, Hk, window = 2, 256, 4, 2, 90
    q, k, v, dout = tensors(B, S, S, H, Hk, 64, torch.bfloat16)
    g = torch.Generator(device="cuda").manual_seed(4)
    n = 1 if rows == "keys" else S
    bias = (torch.argsort(torch.rand((B, Hk, n, S), generator=g, device="cuda"), -1).float() / S - 0.5).to(torch.bfloat16).requires_grad_()
    out = call(q, k, v, None, bias, window_size=kept, sliding_window=window)
    seen = visible(S, S, window)
    if kept:
        mask = create_mask(bias.detach(), None, B, S, S, kept, torch.finfo(torch.bfloat16).min)
        seen = seen & mask.repeat_interleave(H // Hk, 1)
    check([out], *definition(*(x.detach() for x in (q, k, v)), seen, bias.detach()))
    (db,) = torch.autograd.grad(out, bias, dout)
    hidden = ~seen.expand(B, H, S, S).reshape(B, Hk, H // Hk, S, S).any(2)
    if n == S:
        assert not bool(db[hidden].any())
    assert bool(db.any())


@pytest.mark.parametrize("side", ["left", "right"])
@pytest.mark.parametrize("Sq", [200, 1])
def test_padded(side, Sq):
    B, S, window, there = 3, 200, 33, (200, 120, 20)
    q, k, v, dout = tensors(B, Sq, S, 4, 2, 64, torch.bfloat16)
    j = torch.arange(S, device="cuda")
    mask = torch.stack([j >= S - n if side == "left" else j < n for n in there])
    out = call(q, k, v, mask.long(), None, sliding_window=window)
    grads = torch.autograd.grad(out, (q, k, v), dout)
    for b, n in enumerate(there):
        rows = slice(S - n, S) if side == "left" else slice(0, n)
        mine = slice(0, 1) if Sq == 1 else rows
        got = [out[b:b + 1, mine], *(x[b:b + 1, m] for x, m in zip(grads, (mine, rows, rows)))]
        check(got, *reference(q[b:b + 1, mine], k[b:b + 1, rows], v[b:b + 1, rows], window, 0, dout=dout[b:b + 1, mine]))
        assert Sq == 1 or not bool(out[b][~mask[b]].any())


@pytest.mark.parametrize("given", ["position ids", "boundaries"])
@pytest.mark.parametrize("lengths", [[100, 7, 300], [5000, 700]])
def test_packed(given, lengths):
    T, window = sum(lengths), 64
    q, k, v, dout = tensors(1, T, T, 4, 2, 64, torch.bfloat16)
    cuts = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    cu = torch.tensor(cuts, dtype=torch.int32, device="cuda")
    kw = dict(position_ids=torch.cat([torch.arange(n, device="cuda") for n in lengths])[None]) if given == "position ids" else \
        dict(cu_seq_lens_q=cu, cu_seq_lens_k=cu, max_length_q=max(lengths), max_length_k=max(lengths))
    out = call(q, k, v, None, None, sliding_window=window, **kw)
    got = [out, *torch.autograd.grad(out, (q, k, v), dout)]
    check([x[0] for x in got], *packed_reference(q[0], k[0], v[0], cuts, cuts, window, 0, dout[0]))


@pytest.mark.parametrize("heads", [None, 1, 4])
def test_cached(heads):
    R, H, Hk, d, keys, window, dtype = 3, 4, 2, 64, 96, 20, torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(20)
    tables, cache = fsa.block_tables(R, 6, 18, 16, device="cuda"), fsa.quantized_cache(18, Hk, d, 16, device="cuda")
    for new in ([40, 7, 33], [1, 1, 1], [3, 0, 2]):
        total = sum(new)
        step = tables.extend(torch.tensor(new, dtype=torch.int32, device="cuda"), total)
        q, k, v = (torch.randn((1, total, h, d), generator=g, device="cuda", dtype=dtype) for h in (H, Hk, Hk))
        bias = torch.randn((R, heads, 1, keys), generator=g, device="cuda", dtype=dtype) if heads else None
        with torch.no_grad():
            out = call(q, k, v, None, bias, window_size=30, sliding_window=window, kv_cache=CachedLayer(cache, tables, step, None, max(new)))
        kept = None
        if heads:
            valid = torch.arange(keys, device="cuda") < step.lengths[:, None]
            low = torch.finfo(dtype).min
            if heads == H:
                mask = create_mask(bias, valid, R, 1, keys, 30, low)
                bias, kept = bias.masked_fill(~mask, -math.inf), mask.view(R, Hk, H // Hk, 1, keys).any(2)
            else:
                kept = create_kept_keys(bias, valid, R, 1, keys, 30, low)
        want = fsa.flash_sparse_attn_cache_func(q[0], cache, tables, step, attn_mask=kept, attn_bias=bias, sliding_window=window, max_seqlen_q=max(new))
        assert torch.equal(out[0], want)
        plain = fsa.flash_sparse_attn_cache_func(q[0], cache, tables, step, attn_mask=kept, attn_bias=bias, max_seqlen_q=max(new))
        assert not torch.equal(want, plain)


def test_a_window_that_hides_nothing():
    q, k, v, _ = tensors(2, 80, 80, 4, 2, 64, torch.bfloat16, grad=False)
    bias = torch.randn((2, 2, 1, 80), device="cuda", dtype=torch.bfloat16)
    padding = torch.arange(80, device="cuda")[None] < torch.tensor([[80], [50]], device="cuda")
    for args, kw in (((None, None), {}), ((None, bias), {}), ((None, bias), dict(window_size=30)), ((padding, None), {}), ((None, None), dict(is_causal=False))):
        for window in (80, 2 ** 31 - 1):
            assert torch.equal(call(q, k, v, *args, **kw), call(q, k, v, *args, sliding_window=window, **kw))
    one = q[:, :1]
    assert torch.equal(call(one, k, v, None, None, is_causal=False, sliding_window=30), call(one, k, v, None, None, sliding_window=30))
