"""Rows that see no key: 0, LSE +inf (from which the backward has probabilities of 0), no gradients; with several queries and with one, under
masks, and where there are fewer keys than queries."""
import pytest
import torch

import flash_sparse_attn as fsa
from test_gpu_window import tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("Sq,Sk,masked", [(150, 190, True), (300, 40, False), (300, 40, True), (1, 200, True)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_dense(Sq, Sk, masked, d, dtype):
    q, k, v, dout = tensors(2, Sq, Sk, 4, 2, d, dtype)
    mask = None
    if masked:
        mask = torch.ones((2, 1, 1, Sk), dtype=torch.bool, device="cuda")
        mask[0, ..., :100] = False
        mask[1] = False
    out, lse, _ = fsa.flash_sparse_attn_window_func(q, k, v, 30, 2, attn_mask=mask, return_attn_probs=True)
    t, j = torch.arange(Sk - Sq, Sk, device="cuda")[:, None], torch.arange(Sk, device="cuda")
    seen = ((j <= t) & ((t - j < 30) | (j < 2)))[None, None] & (True if mask is None else mask)
    rows = seen.any(-1).expand(2, 4, Sq)
    assert bool((~rows).any())
    assert bool((lse[~rows] == torch.inf).all()) and bool(torch.isfinite(lse[rows]).all())
    assert not bool(out.transpose(1, 2)[~rows].any())
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), dout)
    assert not bool(dq.transpose(1, 2)[~rows].any())
    keys = seen.any(2).expand(2, 4, Sk)[:, ::2]
    for x in (dk, dv):
        assert bool(torch.isfinite(x).all()) and not bool(x.transpose(1, 2)[~keys].any())


@pytest.mark.parametrize("d", [64, 256])
def test_packed(d):
    q, k, v, dout = (x[0].detach().requires_grad_(i < 3) for i, x in enumerate(tensors(1, 150, 80, 4, 2, d, torch.bfloat16)))
    cu_q, cu_k = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 100, 150], [0, 30, 80]))
    out, lse, _ = fsa.flash_sparse_attn_window_varlen_func(q, k, v, cu_q, cu_k, 100, 50, 20, 1, return_attn_probs=True)
    assert lse.shape == (4, 150) and bool((lse[:, :70] == torch.inf).all()) and bool(torch.isfinite(lse[:, 70:]).all())
    assert not bool(out[:70].any()) and not bool(torch.autograd.grad(out, q, dout)[0][:70].any())
