"""Blocks beyond 4 GiB of a cache: written, read one by one, gathered and converted, they give what the same blocks of a small cache give."""
import pytest
import torch

import flash_sparse_attn as fsa
from test_gpu_cache import attend, check, dev, ints  # noqa: F401

pytestmark = pytest.mark.gpu


def test_blocks_beyond_4_gib(dev):  # noqa: F811
    H, Hk, d, bs, few, many = 32, 2, 128, 128, 24, 140000
    assert (many - few) * Hk * bs * d > 2 ** 32
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GB")
    g = torch.Generator(device=dev).manual_seed(61)
    f = fsa.rotary_frequencies(d, device=dev)
    small = fsa.block_tables(2, 12, few, bs, device=dev), fsa.quantized_cache(few, Hk, d, bs, device=dev)
    large = fsa.block_tables(2, 12, few, bs, device=dev), fsa.quantized_cache(many, Hk, d, bs, device=dev)
    large[0].free.add_(many - few)
    for new in ([700, 350], [300, 0], [1, 1], [4, 3]):
        T = sum(new)
        x = torch.randn((T, H + 2 * Hk, d), generator=g, device=dev).to(torch.bfloat16)
        outs = []
        for tables, cache in (small, large):
            step = tables.extend(ints(new, dev), T)
            assert bool(step.granted.all())
            q = fsa.cache_append(cache, tables, step, x[:, H:H + Hk], x[:, H + Hk:], query=x[:, :H], frequencies=f)
            most = int(step.lengths.max())
            kept = fsa.KeptKeys(torch.arange(0, most, 3, dtype=torch.int32, device=dev).expand(1, 1, -1).contiguous(),
                                ints([[-(-most // 3)]], dev), None, most)
            outs.append([fsa.flash_sparse_attn_cache_func(q, cache, tables, step, m, max_seqlen_q=max(new)) for m in (None, kept)])
        for a, b in zip(*outs):
            assert torch.equal(a, b) and bool(a.any())
    assert torch.equal(small[0].table + (many - few) * (small[0].table >= 0), large[0].table)
    for a, b in zip(small[1], large[1]):
        assert torch.equal(a.view(torch.uint8), b[many - few:].view(torch.uint8))


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_beyond_2_to_the_31_elements(dev, interleaved):  # noqa: F811
    S, H, d = 70000, 256, 128
    assert S * H * d > 2 ** 31
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GB")
    f = fsa.rotary_frequencies(96, interleaved=interleaved, device=dev)
    x = torch.empty((1, S, H, d), device=dev, dtype=torch.bfloat16)
    g = torch.Generator(device=dev).manual_seed(63)
    for at in (0, S // 2, S - 3):
        x[:, at:at + 3] = torch.randn((1, 3, H, d), generator=g, device=dev).to(torch.bfloat16)
    out = fsa.apply_rotary(x, x[:, :, :1], f)
    for at in (0, S // 2, S - 3):
        part = x[:, at:at + 3].contiguous()
        want = fsa.apply_rotary(part, part[:, :, :1].contiguous(), f, torch.arange(at, at + 3, device=dev))
        assert torch.equal(out[0][:, at:at + 3], want[0]) and torch.equal(out[1][:, at:at + 3], want[1])


def test_tensors_without_elements(dev):  # noqa: F811
    f = fsa.rotary_frequencies(64, device=dev)
    for shape in ((0, 5, 2, 64), (3, 0, 2, 64), (0, 2, 64)):
        q, k = (torch.empty(shape, device=dev, dtype=torch.bfloat16, requires_grad=True) for _ in range(2))
        out = fsa.apply_rotary(q, k, f)
        assert [t.shape for t in out] == [torch.Size(shape)] * 2
        grads = torch.autograd.grad(out, (q, k), [torch.empty_like(t) for t in out])
        assert [t.shape for t in grads] == [torch.Size(shape)] * 2


def test_blocks_that_requests_share(dev):  # noqa: F811
    """Full blocks may be held by several requests (a common prefix); each has blocks of its own behind them."""
    H, Hk, d, bs = 8, 2, 64, 16
    g = torch.Generator(device=dev).manual_seed(62)
    tables, cache = fsa.block_tables(2, 8, 16, bs, device=dev), fsa.quantized_cache(16, Hk, d, bs, device=dev)
    first = torch.randn((48, H + 2 * Hk, d), generator=g, device=dev).to(torch.float16)
    step = tables.extend(ints([48, 0], dev), 48)
    fsa.cache_append(cache, tables, step, first[:, H:H + Hk], first[:, H + Hk:])
    tables.table[1, :3] = tables.table[0, :3]
    tables.lengths[1] = 48
    x = torch.randn((9, H + 2 * Hk, d), generator=g, device=dev).to(torch.float16)
    step = tables.extend(ints([5, 4], dev), 9)
    fsa.cache_append(cache, tables, step, x[:, H:H + Hk], x[:, H + Hk:])
    assert tables.table[0, :3].tolist() == tables.table[1, :3].tolist() and tables.table[0, 3] != tables.table[1, 3]
    check(fsa.flash_sparse_attn_cache_func(x[:, :H], cache, tables, step), *attend(x[:, :H], cache, tables, step))
