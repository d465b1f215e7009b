"""The HuggingFace-style caller over the 8-bit cache: prompts, then token steps, with and without a dynamic mask, equal the operators
called one by one, and the operators' own tests say what those are."""
import pytest
import torch

import flash_sparse_attn as fsa
from flash_sparse_attn.integrations import CachedLayer, flash_sparse_attention_forward
from flash_sparse_attn.utils.mask import create_kept_keys
from test_gpu_cache import attend, check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda:0")


class Layer(torch.nn.Module):
    is_causal = True
    layer_idx = 0


@pytest.mark.parametrize("window", [None, 24])
def test_prompts_and_tokens(dev, window):
    R, H, Hk, d, keys, dtype = 3, 8, 2, 64, 96, torch.bfloat16
    g = torch.Generator(device=dev).manual_seed(20)
    tables, cache = fsa.block_tables(R, 6, 18, 16, device=dev), fsa.quantized_cache(18, Hk, d, 16, device=dev)
    f = fsa.rotary_frequencies(d, device=dev)
    module = Layer()
    for new in ([40, 7, 33], [1, 1, 1], [3, 0, 2]):
        total = sum(new)
        step = tables.extend(torch.tensor(new, dtype=torch.int32, device=dev), total)
        q, k, v = (torch.randn((1, h, total, d), generator=g, device=dev, dtype=dtype) for h in (H, Hk, Hk))
        bias = torch.randn((R, Hk, 1, keys), generator=g, device=dev, dtype=dtype) if window else None
        layer = CachedLayer(cache, tables, step, f, max(new))
        with torch.no_grad():
            out, weights = flash_sparse_attention_forward(module, q, k, v, None, bias, window_size=window, kv_cache=layer)
        assert weights is None and out.shape == (1, total, H, d)
        turned = fsa.apply_rotary(q[0].transpose(0, 1), None, f, step.positions)[0]
        kept = None
        if window:
            valid = torch.arange(keys, device=dev) < step.lengths[:, None]
            kept = create_kept_keys(bias, valid, R, 1, keys, window, torch.finfo(dtype).min)
        check(out[0], *attend(turned, cache, tables, step, kept, bias))


def test_refusals(dev):
    tables, cache = fsa.block_tables(1, 2, 2, 16, device=dev), fsa.quantized_cache(2, 1, 64, 16, device=dev)
    step = tables.extend(torch.tensor([3], dtype=torch.int32, device=dev), 3)
    x = torch.zeros((1, 1, 3, 64), device=dev, dtype=torch.bfloat16)
    layer = CachedLayer(cache, tables, step)
    with pytest.raises(ValueError):
        flash_sparse_attention_forward(Layer(), x, x, x, torch.ones((1, 3), device=dev), None, kv_cache=layer)
    two = torch.zeros((2, 1, 3, 64), device=dev, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        flash_sparse_attention_forward(Layer(), two, two, two, None, None, kv_cache=layer)
    with pytest.raises(NotImplementedError):
        flash_sparse_attention_forward(Layer(), x, x, x, None, None, softcap=1.0, kv_cache=layer)
