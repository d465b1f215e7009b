"""The HuggingFace-style caller over the 8-bit cache with a window: a bias for all heads, for each kv head and for each query head, and
refusals that leave the cache as it was."""
import math

import pytest
import torch

import flash_sparse_attn as fsa
from flash_sparse_attn.integrations import CachedLayer, flash_sparse_attention_forward
from flash_sparse_attn.utils.mask import create_mask
from test_gpu_cache import attend, check, dev, filled  # noqa: F401

pytestmark = pytest.mark.gpu


class Layer(torch.nn.Module):
    is_causal = True
    layer_idx = 0


@pytest.mark.parametrize("bias_rows", [1, 3])
@pytest.mark.parametrize("heads", ["one", "kv", "all"])
@pytest.mark.parametrize("cached,new,H,Hk,d", [([300, 0, 90], [1, 1, 1], 8, 2, 64), ([20, 130, 3], [6, 40, 1], 12, 4, 128), ([50, 8, 70], [2, 1, 0], 2, 2, 32)])
def test_windows(dev, cached, new, H, Hk, d, heads, bias_rows):  # noqa: F811
    R, window, dtype, keys = 3, 24, torch.bfloat16, max(cached) + 8  # (of some requests' last keys the bias says nothing)
    tables, cache, step, g = filled(dev, R, cached, new, Hk, d, 16, 33)
    q, k, v = (torch.randn((1, h, sum(new), d), generator=g, device=dev, dtype=dtype) for h in (H, Hk, Hk))
    hb = {"one": 1, "kv": Hk, "all": H}[heads]
    bias = torch.randn((bias_rows, hb, 1, keys), generator=g, device=dev, dtype=dtype)
    f = fsa.rotary_frequencies(d, device=dev)
    with torch.no_grad():
        out, _ = flash_sparse_attention_forward(Layer(), q, k, v, None, bias, window_size=window, kv_cache=CachedLayer(cache, tables, step, f))
    turned = fsa.apply_rotary(q[0].transpose(0, 1), None, f, step.positions)[0]
    valid = torch.arange(keys, device=dev) < step.lengths[:, None]
    rows = bias.expand(R, -1, -1, -1)
    mask = create_mask(rows.contiguous(), valid, R, 1, keys, window, torch.finfo(dtype).min)
    per_head = rows.masked_fill(~mask, -math.inf).repeat_interleave(H // hb, 1)
    assert int((per_head > -math.inf).sum(-1).max()) <= window
    pos = torch.arange(keys, dtype=torch.int32, device=dev).expand(1, 1, -1)
    everything = fsa.KeptKeys(pos, torch.full((1, 1), keys, dtype=torch.int32, device=dev), None, keys)
    check(out[0], *attend(turned, cache, tables, step, everything, per_head))


def test_refusals_write_nothing(dev):  # noqa: F811
    R, H, Hk, d, keys = 2, 4, 2, 64, 64
    tables, cache, step, g = filled(dev, R, [20, 5], [1, 2], Hk, d, 16, 34)
    q, k, v = (torch.randn((1, h, 3, d), generator=g, device=dev, dtype=torch.bfloat16) for h in (H, Hk, Hk))
    bias = torch.randn((R, H, 1, keys), generator=g, device=dev, dtype=torch.bfloat16)
    before = [t.clone().view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t.clone() for t in cache]
    layer = CachedLayer(cache, tables, step)
    for args, kw in [((q, k, v, None, bias[:, :3]), {}), ((q, k, v, None, bias.float()), {}), ((q, k, v, None, bias[0]), {}),
                     ((q, k, v, None, bias.expand(R, H, 3, keys)), {}), ((q, k, v, None, bias[..., :0]), {}), ((q[:, :3], k, v, None, None), {}),
                     ((q, k, v, None, bias.cpu()), {}), ((q, k, v, None, bias.clone().requires_grad_(True)), {}),
                     ((q, k, v, None, bias), dict(kv_cache=layer._replace(max_seqlen_q=-1))), ((q, k, v, None, torch.cat((bias, bias))), {})]:
        for window in (None, 8):
            with pytest.raises((ValueError, RuntimeError)):
                flash_sparse_attention_forward(Layer(), *args, window_size=window, **{"kv_cache": layer, **kw})
    for a, b in zip(before, cache):
        assert torch.equal(a, b.view(torch.uint8) if b.dtype == torch.float8_e4m3fn else b)
