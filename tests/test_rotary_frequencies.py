"""rotary_frequencies refuses what has no meaning (no GPU needed)."""
import pytest
import torch

import flash_sparse_attn as fsa


@pytest.mark.parametrize("args", [
    dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=-2), dict(rotary_dim=64, scaling="dynamic"), dict(rotary_dim=64, factor=0.0),
    dict(rotary_dim=64, scaling="yarn", factor=2.0), dict(rotary_dim=64, scaling="bands", factor=2.0), dict(rotary_dim=64, base=1.0),
    dict(rotary_dim=2, scaling="ntk", factor=2.0), dict(rotary_dim=64, inv_freq=torch.ones(31)),
    dict(rotary_dim=4, inv_freq=torch.tensor([1.0, float("inf")])),
    dict(rotary_dim=64, scaling="bands", factor=2.0, original_length=64, low_freq_factor=4.0, high_freq_factor=1.0)])
def test_refused(args):
    with pytest.raises(ValueError):
        fsa.rotary_frequencies(**args, device="cpu")


def test_own_frequencies():
    inv = torch.tensor([1.0, 0.25, 1e-9], dtype=torch.float64)
    f = fsa.rotary_frequencies(6, inv_freq=inv, device="cpu")
    got = torch.tensor([t % 2 ** 64 for t in f.turns.tolist()], dtype=torch.float64) / 2.0 ** 64 * 2 * torch.pi
    assert torch.allclose(got, inv, rtol=1e-15, atol=0) or torch.allclose(got, inv, rtol=2e-15, atol=2.0 ** -62)
    assert f.amplitude == 1.0 and not f.interleaved


@pytest.mark.parametrize("args", [dict(requests=0, blocks_per_request=1, num_blocks=1), dict(requests=8193, blocks_per_request=1, num_blocks=1),
                                  dict(requests=1, blocks_per_request=0, num_blocks=1), dict(requests=1, blocks_per_request=1, num_blocks=0),
                                  dict(requests=1, blocks_per_request=1, num_blocks=1, block_size=48)])
def test_block_tables_refused(args):
    with pytest.raises(ValueError):
        fsa.block_tables(**args, device="cpu")


@pytest.mark.parametrize("args", [dict(num_blocks=0, kv_heads=1, head_dim=64), dict(num_blocks=1, kv_heads=0, head_dim=64),
                                  dict(num_blocks=1, kv_heads=1, head_dim=72), dict(num_blocks=1, kv_heads=1, head_dim=272),
                                  dict(num_blocks=1, kv_heads=1, head_dim=64, block_size=8)])
def test_quantized_cache_refused(args):
    with pytest.raises(ValueError):
        fsa.quantized_cache(**args, device="cpu")
