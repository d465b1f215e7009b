"""The 8-bit cache has no gradients: a call that would need one raises, whichever tensor it would be the gradient of, and writes
nothing; without gradients the same tensors are served."""
import pytest
import torch

import flash_sparse_attn as fsa
from test_gpu_cache import attend, check, dev, filled  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
def test_scales_that_are_learned(dev, which):  # noqa: F811
    tables, cache, step, g = filled(dev, 2, [20, 5], [1, 2], 2, 64, 16, 51)
    kv = torch.randn((2, 3, 2, 64), generator=g, device=dev, dtype=torch.bfloat16)
    q = torch.randn((3, 4, 64), generator=g, device=dev, dtype=torch.bfloat16)
    learned = cache._replace(**{which: getattr(cache, which).clone().requires_grad_(True)})
    before = [t.detach().clone().view(torch.uint8) for t in learned]
    with pytest.raises(RuntimeError, match="no gradients"):
        fsa.cache_append(learned, tables, step, kv[0], kv[1])
    with pytest.raises(RuntimeError, match="no gradients"):
        fsa.flash_sparse_attn_cache_func(q, learned, tables, step)
    assert all(torch.equal(a, b.detach().view(torch.uint8)) for a, b in zip(before, learned))
    with torch.no_grad():
        fsa.cache_append(learned, tables, step, kv[0], kv[1])
        check(fsa.flash_sparse_attn_cache_func(q, learned, tables, step), *attend(q, learned, tables, step))
