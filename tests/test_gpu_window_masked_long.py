"""Windows of more key tiles than the backward's table of tiles with a kept key holds, and more keys than the calls take. Bounds are those of
test_gpu_window.py."""
import pytest
import torch

import flash_sparse_attn as fsa
from test_gpu_window import check, reference, tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads", ["one", "query"])
@pytest.mark.parametrize("Sq,Sk,window,sinks,d", [(300, 300001, 299000, 3, 64), (130, 280000, 1000, 270000, 128), (40, 270001, 270001, 0, 64), (1, 300001, 290000, 9, 64)])
def test_gradients_under_a_mask(Sq, Sk, window, sinks, d, heads):
    q, k, v, dout = tensors(1, Sq, Sk, 2, 1, d, torch.bfloat16)
    g = torch.Generator(device="cuda").manual_seed(3)
    mask = torch.rand((1, 1 if heads == "one" else 2, 1, Sk), generator=g, device="cuda") < 0.5
    mask[..., 1000:60000] = False
    out = fsa.flash_sparse_attn_window_func(q, k, v, window, sinks, attn_mask=mask)
    check([out, *torch.autograd.grad(out, (q, k, v), dout)], *reference(q, k, v, window, sinks, mask, dout=dout))


def test_too_many_keys():
    q, k = (torch.zeros((1, n, 1, 64), dtype=torch.bfloat16, device="cuda") for n in (100, 2 ** 20 + 1))
    with pytest.raises(RuntimeError):
        fsa.flash_sparse_attn_window_func(q, k, k, 50, 3)
    out = fsa.flash_sparse_attn_window_func(q, k[:, :-1], k[:, :-1], 50, 3)
    assert not bool(out.any())
