"""Attention over the 8-bit cache where every key that a query sees carries one large negative bias: the result is the average of
the visible values, whatever the size of the bias, and whatever the scales of the blocks that hold them.

Tolerance, derived: the probabilities are equal, so that nothing in them grows with the bias. A probability is rounded to fp16 (2^-11 of
itself), sums of n products in 32 bits are off by at most n 2^-23 of their magnitudes, and there is one rounding to the type."""
import math

import pytest
import torch

import flash_sparse_attn as fsa
from test_gpu_cache import dev, filled, ints, widen  # noqa: F401

pytestmark = pytest.mark.gpu

LAYOUTS = [  # cached, new, heads, kv heads, head dim, block size
    ([200, 130, 64], [1, 1, 1], 4, 2, 64, 32), ([5000], [1], 8, 2, 128, 64), ([700, 0, 12], [5, 9, 1], 12, 4, 128, 16),
    ([300, 90], [3, 40], 8, 2, 256, 32), ([150] * 140, [1] * 140, 2, 1, 16, 16)]
BIASES = [  # type, bias, whether queries may be other than 0: next to the type's lowest number their scores count for nothing
    (torch.bfloat16, torch.finfo(torch.bfloat16).min, True), (torch.bfloat16, torch.finfo(torch.bfloat16).max, True), (torch.bfloat16, -1e9, False), (torch.bfloat16, -1.2e7, False),
    (torch.float16, torch.finfo(torch.float16).min, False)]


def averages(cache, tables, step, H, visible):
    """(mean of the visible values, of their magnitudes, their number) in 64 bits; visible (requests, kv heads, keys)."""
    T, Hk, d, bs = step.positions.numel(), cache.k.shape[1], cache.k.shape[3], tables.block_size
    mean, size = torch.zeros((2, T, H, d), dtype=torch.float64, device=cache.k.device)
    number = torch.zeros((T, H, 1), dtype=torch.float64, device=cache.k.device)
    cu, length = step.cu_seqlens.tolist(), step.lengths.tolist()
    for r in range(len(length)):
        blocks = tables.table[r, :-(-length[r] // bs)].long()
        n = cu[r + 1] - cu[r]
        seen = torch.arange(length[r], device=mean.device)[None] <= length[r] - n + torch.arange(n, device=mean.device)[:, None]
        for h in range(H):
            hk = h // (H // Hk)
            v = (cache.v[blocks, hk].double() * cache.v_scale[blocks, hk].double()[:, None, None]).reshape(-1, d)[:length[r]]
            w = (seen & visible[r, hk, :length[r]]).double()
            count = w.sum(1, keepdim=True)
            number[cu[r]:cu[r + 1], h] = count
            mean[cu[r]:cu[r + 1], h] = w @ v / count.clamp(min=1)
            size[cu[r]:cu[r + 1], h] = w @ v.abs() / count.clamp(min=1)
    return mean, size, number


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("dtype,value,scores", BIASES)
@pytest.mark.parametrize("cached,new,H,Hk,d,bs", LAYOUTS)
def test_rows_of_one_large_bias_are_averages(dev, cached, new, H, Hk, d, bs, dtype, value, scores, kept, wide):  # noqa: F811
    R, T, keys = len(cached), sum(new), max(a + b for a, b in zip(cached, new))
    tables, cache, step, g = filled(dev, R, cached, new, Hk, d, bs, 31)
    kv = torch.randn((2, T, Hk, d), generator=g, device=dev).to(dtype)
    fsa.cache_append(cache, tables, step, kv[0], kv[1])
    cache.v_scale.copy_(torch.exp2(torch.randint(-12, -2, cache.v_scale.shape, generator=g, device=dev).float()))
    q = torch.randn((T, H, d), generator=g, device=dev).to(dtype) * float(scores)
    bias = torch.full((R, Hk, 1, keys), value, device=dev, dtype=dtype)
    bias[:, -1, :, ::3] = -math.inf
    visible = bias[:, :, 0] > -math.inf
    keep = None
    if kept:
        pos = torch.arange(1, keys, 2, dtype=torch.int32, device=dev).expand(R, Hk, -1).contiguous()
        keep = fsa.KeptKeys(pos, torch.full((R, Hk), pos.shape[-1], dtype=torch.int32, device=dev), None, keys)
        visible = visible & (torch.arange(keys, device=dev) % 2 == 1)
    mean, size, number = averages(cache, tables, step, H, visible)
    if wide:
        tables = widen(tables)
    got = fsa.flash_sparse_attn_cache_func(q, cache, tables, step, keep, bias).double()
    tol = torch.finfo(dtype).eps / 2 * mean.abs() + (2.0 ** -11 + number * 2.0 ** -23) * size + torch.finfo(dtype).tiny
    assert bool(((got - mean).abs() <= tol).all()), ((got - mean).abs() / tol).max().item()
    assert not bool(got[(number == 0).expand_as(got)].any())


@pytest.mark.parametrize("value", [-1e9, -3e4, 3e4, 1e9, torch.finfo(torch.bfloat16).min, torch.finfo(torch.bfloat16).max])
def test_keys_without_the_large_bias(dev, value):  # noqa: F811
    """Keys of two biases far apart: those of the larger one alone count, an average over them with queries of 0."""
    tables, cache, step, g = filled(dev, 2, [900, 70], [1, 3], 2, 128, 16, 32)
    kv = torch.randn((2, 4, 2, 128), generator=g, device=dev).to(torch.bfloat16)
    fsa.cache_append(cache, tables, step, kv[0], kv[1])
    cache.v_scale.copy_(torch.exp2(torch.randint(-12, -2, cache.v_scale.shape, generator=g, device=dev).float()))
    bias = torch.zeros((2, 2, 1, 901), device=dev, dtype=torch.bfloat16)
    bias[:, :, :, ::2] = value
    visible = bias[:, :, 0] == bias.amax()
    mean, size, number = averages(cache, tables, step, 8, visible)
    q = torch.zeros((4, 8, 128), device=dev, dtype=torch.bfloat16)
    for t in (tables, widen(tables)):
        got = fsa.flash_sparse_attn_cache_func(q, cache, t, step, None, bias).double()
        tol = 2.0 ** -8 * mean.abs() + (2.0 ** -11 + number * 2.0 ** -23) * size + 1e-38
        assert bool(((got - mean).abs() <= tol).all())


def test_the_lowest_beside_the_highest(dev):  # noqa: F811
    """Half of the keys at the type's lowest number, the others at its highest: the latter alone count; -inf beside both hides."""
    tables, cache, step, g = filled(dev, 2, [900, 70], [1, 3], 2, 128, 16, 35)
    kv = torch.randn((2, 4, 2, 128), generator=g, device=dev).to(torch.bfloat16)
    fsa.cache_append(cache, tables, step, kv[0], kv[1])
    cache.v_scale.copy_(torch.exp2(torch.randint(-12, -2, cache.v_scale.shape, generator=g, device=dev).float()))
    bias = torch.full((2, 2, 1, 901), torch.finfo(torch.bfloat16).min, device=dev, dtype=torch.bfloat16)
    bias[..., 1::4] = torch.finfo(torch.bfloat16).max
    bias[..., 3::4] = -math.inf
    mean, size, number = averages(cache, tables, step, 8, bias[:, :, 0] > 0)
    q = torch.randn((4, 8, 128), generator=g, device=dev).to(torch.bfloat16)
    for t in (tables, widen(tables)):
        got = fsa.flash_sparse_attn_cache_func(q, cache, t, step, None, bias).double()
        tol = 2.0 ** -8 * mean.abs() + (2.0 ** -11 + number * 2.0 ** -23) * size + 1e-38
        assert bool(((got - mean).abs() <= tol).all())
