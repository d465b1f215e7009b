"""The documentation's examples of sliding windows and of drafted tokens run as they are written."""
import pytest
import torch

import flash_sparse_attn as fsa
from test_gpu_documented_calls import Layer, examples

pytestmark = pytest.mark.gpu


def test_training_example():
    dev, H, Hk, d = torch.device("cuda:0"), 4, 2, 64
    q, k, v = (torch.randn((2, 90, h, d), device=dev, dtype=torch.bfloat16, requires_grad=True) for h in (H, Hk, Hk))
    packed = [x.detach().flatten(0, 1).requires_grad_() for x in (q, k, v)]
    texts = examples("fsa.flash_sparse_attn_window_func(")
    assert texts
    for text in texts:
        names = dict(q=q, k=k, v=v, pq=packed[0], pk=packed[1], pv=packed[2], n=100, padding=torch.ones((2, 1, 1, 90), dtype=torch.bool, device=dev),
                     cu_seqlens=torch.tensor([0, 80, 180], dtype=torch.int32, device=dev))
        exec(text, names)
        names["out"].sum().backward()
        assert all(bool(x.grad.isfinite().all()) for x in packed)


def test_serving_example():
    dev, H, Hk, d, V = torch.device("cuda:0"), 4, 2, 64, 1000
    texts = examples("fsa.verify_drafts(")
    assert texts
    w = torch.randn((H * d, V), device=dev, dtype=torch.bfloat16)
    for text in texts:
        tables = fsa.block_tables(requests=3, blocks_per_request=8, num_blocks=24, device=dev)
        new = torch.tensor([4, 0, 2], dtype=torch.int32, device=dev)
        names = dict(torch=torch, layers=[Layer(H, Hk, d, dev) for _ in range(2)], caches=[fsa.quantized_cache(24, Hk, d, device=dev) for _ in range(2)],
                     tables=tables, freqs=fsa.rotary_frequencies(d, device=dev), new_lengths=new, total_tokens=7, n=4, head=lambda x: x @ w,
                     x=torch.randn((7, H * d), device=dev, dtype=torch.bfloat16), token_ids=torch.randint(0, V, (7,), device=dev),
                     draft_probs=torch.full((7, V), 1 / V, device=dev))
        exec(text, names)
        done = names["done"]
        assert torch.equal(done.lengths, tables.lengths) and torch.equal(done.lengths, torch.where(new > 0, done.accepted + 1, 0))
        assert done.next_tokens[1] == -1 and bool((done.next_tokens[[0, 2]] >= 0).all())
