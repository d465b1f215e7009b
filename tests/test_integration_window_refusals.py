"""The HuggingFace-style caller refuses the windows that it cannot show, before anything runs (no GPU needed)."""
import pytest
import torch

import flash_sparse_attn as fsa
from flash_sparse_attn.integrations import CachedLayer, flash_sparse_attention_forward


class Layer(torch.nn.Module):
    is_causal = True
    layer_idx = 0


def call(window, Sq=8, Sk=8, mask=None, bias=None, **kw):
    q, k = (torch.zeros((1, 2, s, 64), dtype=torch.bfloat16) for s in (Sq, Sk))
    return flash_sparse_attention_forward(Layer(), q, k, k, mask, bias, sliding_window=window, **kw)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("window,error", [(0, ValueError), (-3, ValueError), (2 ** 31, ValueError), (4.0, TypeError), (True, TypeError), ("4", TypeError)])
def test_no_windows(window, error, packed):
    kw = dict(position_ids=torch.tensor([[0, 1, 2, 0, 1, 2, 3, 4]])) if packed else {}
    for mask in (None,) if packed else (None, torch.ones((1, 8))):
        with pytest.raises(error):
            call(window, mask=mask, **kw)


@pytest.mark.parametrize("kw", [dict(is_causal=False), dict(softcap=1.0)], ids=str)
def test_not_built(kw):
    for more in (dict(), dict(mask=torch.ones((1, 8))), dict(position_ids=torch.tensor([[0, 1, 2, 0, 1, 2, 3, 4]]))):
        with pytest.raises(NotImplementedError):
            call(4, **kw, **more)


def test_masks_of_other_types():
    with pytest.raises(RuntimeError):
        call(4, mask=torch.zeros((1, 1, 8, 8)))


def test_cached_calls():
    """Nothing is appended: the step and the cache are not even looked at."""
    tables = fsa.BlockTables(*(torch.zeros((1, 4), dtype=torch.int32) for _ in range(5)), block_size=16)
    step = fsa.CacheStep(*(torch.zeros(1, dtype=torch.int32) for _ in range(7)))
    layer = CachedLayer(None, tables, step)
    for window, kw, error in ((0, {}, ValueError), (2.5, {}, TypeError), (63, dict(is_causal=False), NotImplementedError)):
        with pytest.raises(error):
            call(window, kv_cache=layer, **kw)
