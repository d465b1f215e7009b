"""Masks that are made in inference mode, as a server makes them: the same contents as elsewhere, taken by the attention, by the attention
over the 8-bit cache and by the HuggingFace-style caller."""
import pytest
import torch

import flash_sparse_attn as fsa
from flash_sparse_attn.integrations import CachedLayer, flash_sparse_attention_forward
from flash_sparse_attn.utils.mask import create_mask
from test_gpu_cache import attend, check, dev, filled  # noqa: F401

pytestmark = pytest.mark.gpu
LOW = torch.finfo(torch.bfloat16).min


@pytest.mark.parametrize("rows", [1, 130])
def test_attention(dev, rows):  # noqa: F811
    B, S, H, Hk, d = 2, 130, 4, 2, 64
    g = torch.Generator(device=dev).manual_seed(71)
    q, k, v = (torch.randn((B, S, h, d), generator=g, device=dev, dtype=torch.bfloat16) for h in (H, Hk, Hk))
    bias = torch.randn((B, Hk, rows, S), generator=g, device=dev, dtype=torch.bfloat16)
    mask = create_mask(bias, None, B, S, S, 40, LOW)
    want = fsa.flash_sparse_attn_func(q, k, v, mask & True, bias, is_causal=True)  # (a mask without anything tied to it)
    with torch.inference_mode():
        inside = create_mask(bias, None, B, S, S, 40, LOW)
        got = fsa.flash_sparse_attn_func(q, k, v, inside, bias, is_causal=True)
    assert torch.equal(inside, mask) and torch.equal(got, want)


@pytest.mark.parametrize("heads", [1, 2, 4])
def test_cache(dev, heads):  # noqa: F811
    R, H, Hk, d, keys, window = 2, 4, 2, 64, 96, 16
    f = fsa.rotary_frequencies(d, device=dev)
    outs = []
    for mode in (torch.no_grad, torch.inference_mode):
        tables, cache, step, g = filled(dev, R, [90, 40], [1, 2], Hk, d, 16, 72)
        q, k, v = (torch.randn((1, h, 3, d), generator=g, device=dev, dtype=torch.bfloat16) for h in (H, Hk, Hk))
        bias = torch.randn((R, heads, 1, keys), generator=g, device=dev, dtype=torch.bfloat16)

        class Layer(torch.nn.Module):
            is_causal = True

        with mode():
            outs.append(flash_sparse_attention_forward(Layer(), q, k, v, None, bias, window_size=window, kv_cache=CachedLayer(cache, tables, step, f))[0])
            if heads < H:
                mask = create_mask(bias, None, R, 1, keys, window, LOW)
                x = q[0].transpose(0, 1)
                kept = fsa.utils.mask.create_kept_keys(bias, None, R, 1, keys, window, LOW)
                check(fsa.flash_sparse_attn_cache_func(x, cache, tables, step, mask, bias), *attend(x, cache, tables, step, kept, bias))
    assert torch.equal(*outs)
