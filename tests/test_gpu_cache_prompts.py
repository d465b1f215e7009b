"""Attention of prompt parts over the 8-bit cache, in steps with enough work for the conversion to 16 bits. Every case says how many
keys have to be converted, and the call through the C interface, whose scratch the test can read, says how many were: a threshold
that is tuned cannot empty these tests."""
import ctypes
import math

import pytest
import torch

import flash_sparse_attn as fsa
from flash_sparse_attn import _lib
from test_cabi_cache import Attention, Cache
from test_gpu_cache import attend, check, dev, filled, ints  # noqa: F401

pytestmark = pytest.mark.gpu


def through_c(q, cache, tables, step, max_q=None, max_k=None, causal=True):
    """(result, converted keys whose results were used) of the call through the C interface; the scratch ends with what the conversion
    came upon (256 bytes; not 0 at first: they are computed again) and the converted keys of the requests, summed up (requests + 1,
    in whole 256 bytes)."""
    T, H, d = q.shape
    R, width = tables.table.shape
    c = Cache(k=cache.k.data_ptr(), v=cache.v.data_ptr(), k_scale=cache.k_scale.data_ptr(), v_scale=cache.v_scale.data_ptr(),
              table=tables.table.data_ptr(), requests=R, width=width, num_blocks=cache.k.shape[0], block_size=tables.block_size, tokens=T,
              h_k=cache.k.shape[1], d=d, **{n: getattr(step, n).data_ptr() for n in ("cu_seqlens", "lengths", "cu_blocks", "cu_chunks", "positions")})
    out = torch.full_like(q, math.nan)
    p = Attention(c=c, query=q.data_ptr(), out=out.data_ptr(), query_row_stride=q.stride(0), query_head_stride=q.stride(1),
                  out_row_stride=out.stride(0), out_head_stride=out.stride(1), h=H, dtype=_lib.FDMA_BF16 if q.dtype == torch.bfloat16 else _lib.FDMA_FP16,
                  is_causal=int(causal), max_seqlen_q=T if max_q is None else max_q, max_seqlen_k=width * tables.block_size if max_k is None else max_k,
                  softmax_scale=d ** -0.5)
    lib = _lib.load()
    size, run = lib.fdma_cache_attention_workspace_bytes, lib.fdma_cache_attention
    size.restype, size.argtypes = ctypes.c_size_t, [ctypes.c_void_p]
    run.restype, run.argtypes = ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p]
    n = size(ctypes.byref(p))
    ws = torch.full((max(n, 256),), 0xFF, dtype=torch.uint8, device=q.device)
    p.workspace, p.workspace_bytes = ws.data_ptr(), n
    assert run(ctypes.byref(p), torch.cuda.current_stream().cuda_stream) == 0
    at = n - -(-(R + 1) * 4 // 256) * 256
    if not n:
        return out, 0
    again, keys = int(ws[at - 256:at - 252].view(torch.int32)), int(ws[at:at + 4 * (R + 1)].view(torch.int32)[R])
    assert keys > 0 or again
    return out, 0 if again else keys


def prompts(dev, cached, new, H, Hk, d, bs, dtype, seed):  # noqa: F811
    tables, cache, step, g = filled(dev, len(cached), cached, new, Hk, d, bs, seed)
    T = sum(new)
    kv = torch.randn((2, T, Hk, d), generator=g, device=dev).to(dtype)
    fsa.cache_append(cache, tables, step, kv[0], kv[1])
    return tables, cache, step, torch.randn((T, H, d), generator=g, device=dev).to(dtype), g


CASES = [  # cached, new, heads, kv heads, head dim, block size
    ([500, 37, 0], [200, 260, 300], 32, 8, 128, 64), ([900, 3], [400, 33], 32, 4, 64, 16), ([700, 100, 0, 250], [310, 1, 420, 7], 32, 8, 80, 32),
    ([1000, 0], [256, 1000], 16, 16, 96, 128), ([1500], [300], 16, 1, 256, 128), ([40, 5, 1300, 800], [1, 31, 1, 600], 32, 8, 128, 16),
    ([60] * 40, [1] * 38 + [500, 300], 32, 8, 64, 32), ([0, 511, 77], [513, 32, 5], 16, 2, 256, 64), ([130, 0], [0, 700], 12, 12, 48, 16)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cached,new,H,Hk,d,bs", CASES)
def test_prompt_parts(dev, dtype, cached, new, H, Hk, d, bs):  # noqa: F811
    tables, cache, step, q, _ = prompts(dev, cached, new, H, Hk, d, bs, dtype, 41)
    want = attend(q, cache, tables, step)
    got, keys = through_c(q, cache, tables, step)
    assert keys == sum(a + b for a, b in zip(cached, new) if b >= 32)
    check(got, *want)
    most = max(a + b for a, b in zip(cached, new))
    assert through_c(q, cache, tables, step, max(new), most)[1] == keys
    check(fsa.flash_sparse_attn_cache_func(q, cache, tables, step), *want)
    check(fsa.flash_sparse_attn_cache_func(q, cache, tables, step, max_seqlen_q=max(new), max_seqlen_k=most), *want)
    check(fsa.flash_sparse_attn_cache_func(q, cache, tables, step, is_causal=False, softmax_scale=0.05),
          *attend(q, cache, tables, step, scale=0.05, causal=False))


@pytest.mark.parametrize("d,bs", [(64, 16), (128, 64), (256, 32)])
def test_refused_requests_and_padding(dev, d, bs):  # noqa: F811
    """A refused request of many tokens, padding behind the last one, and single tokens, beside converted ones."""
    H, Hk, dtype = 16, 2, torch.bfloat16
    cached, new = [600, 20, 10, 300], [280, 200, 1, 350]
    tables, cache, _, g = filled(dev, 4, cached, new, Hk, d, bs, 42)
    tables.truncate(ints(cached, dev))
    new[1] = tables.table.shape[1] * bs + 1 - 20  # outgrows its row
    T = sum(new) + 77
    step = tables.extend(ints(new, dev), T)
    assert step.granted.tolist() == [True, False, True, True]
    kv = torch.randn((2, T, Hk, d), generator=g, device=dev).to(dtype)
    fsa.cache_append(cache, tables, step, kv[0], kv[1])
    q = torch.randn((T, H, d), generator=g, device=dev).to(dtype)
    got, keys = through_c(q, cache, tables, step)
    assert keys == 880 + 650
    check(got, *attend(q, cache, tables, step))
    assert not bool(got[280:280 + new[1]].any()) and not bool(got[-77:].any())


def test_captured_and_replayed(dev):  # noqa: F811
    """In a CUDA graph, with contents that change between replays."""
    tables, cache, step, q, g = prompts(dev, [400, 30], [250, 300], 32, 8, 128, 64, torch.bfloat16, 43)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fsa.flash_sparse_attn_cache_func(q, cache, tables, step)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fsa.flash_sparse_attn_cache_func(q, cache, tables, step)
    for _ in range(3):
        q.copy_(torch.randn(q.shape, generator=g, device=dev))
        graph.replay()
        assert torch.equal(out, fsa.flash_sparse_attn_cache_func(q, cache, tables, step))
        check(out, *attend(q, cache, tables, step))


@pytest.mark.parametrize("cached,new,H,Hk,d,bs,max_q,max_k", [
    ([600, 37], [300, 260], 32, 8, 128, 64, 300, 500), ([600, 37], [300, 260], 32, 8, 128, 64, 200, 900), ([500], [400], 16, 2, 64, 16, 400, 700),
    ([700, 100], [310, 1], 32, 8, 80, 32, 300, 1000), ([5, 9], [3, 2], 8, 2, 64, 16, 2, 9)])
def test_requests_beyond_the_bounds(dev, cached, new, H, Hk, d, bs, max_q, max_k):  # noqa: F811
    """Queries from max_seqlen_q on are 0, keys from max_seqlen_k on are not seen, and the causal edge stays where the request's length
    puts it: the same rule for few new tokens and for many."""
    tables, cache, step, q, _ = prompts(dev, cached, new, H, Hk, d, bs, torch.bfloat16, 44)
    seen = fsa.KeptKeys(torch.arange(max_k, dtype=torch.int32, device=dev).expand(1, 1, -1).contiguous(), ints([[max_k]], dev), None, max_k)
    want, tol = attend(q, cache, tables, step, seen)
    for first, n in zip(step.cu_seqlens.tolist(), new):
        want[first + max_q:first + n] = 0
    check(fsa.flash_sparse_attn_cache_func(q, cache, tables, step, max_seqlen_q=max_q, max_seqlen_k=max_k), want, tol)


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("scale", [2.0 ** -1, 2.0 ** 7, 2.0 ** 10])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_numbers_beyond_the_range_of_fp16(dev, dtype, scale, which):  # noqa: F811
    """Keys or values of one block that are larger than fp16 holds count as they are, with fp16 queries too, and so do values that are large
    beside others: results of converted ones are not used then."""
    tables, cache, step, q, _ = prompts(dev, [600, 37], [300, 260], 32, 8, 128, 64, dtype, 45)
    block = tables.table[0, 3].item()
    (cache.k_scale if which == "k" else cache.v_scale)[block] = scale
    x = getattr(cache, which).view(torch.uint8)[block]
    x[:, 5, 7] = 0x7E  # 448
    if which == "k":
        q.mul_(2.0 ** -12)  # (scores near one another)
    want, tol = attend(q, cache, tables, step)
    got, keys = through_c(q, cache, tables, step)
    beyond = want.abs() + tol > 65504  # results that are infinite, or nearly, when they are rounded to fp16
    assert beyond.float().mean() < 0.01
    for out in (got, fsa.flash_sparse_attn_cache_func(q, cache, tables, step)):
        check(out.masked_fill(beyond, 0), want.masked_fill(beyond, 0), tol)
    far = 448 * scale > 65504 or (which == "v" and scale > 2.0 ** -9 * 2.0 ** 8)
    assert (keys == 0) == (dtype == torch.float16 and far)


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,Hk,d,bs", [(32, 8, 128, 64), (32, 4, 64, 16), (16, 2, 256, 32)])
def test_not_a_number_reaches_who_sees_it(dev, dtype, H, Hk, d, bs, which):  # noqa: F811
    """NaN among the last tokens of a prompt: later queries of that request and head become NaN, all others stay as they are."""
    cached, new, G = [500, 37, 700], [300, 260, 310], H // Hk
    tables, cache, step, q, _ = prompts(dev, cached, new, H, Hk, d, bs, dtype, 46)
    want, tol = attend(q, cache, tables, step)
    assert through_c(q, cache, tables, step)[1] == sum(cached) + sum(new)
    for r, token, head in ((0, 270, 0), (1, 101, 1), (1, 200, 1), (2, 309, 0)):
        pos = cached[r] + token
        getattr(cache, which).view(torch.uint8)[tables.table[r, pos // bs], head, pos % bs, 9] = 0xFF
    assert (through_c(q, cache, tables, step)[1] == 0) == (which == "v")
    got = fsa.flash_sparse_attn_cache_func(q, cache, tables, step)
    first = step.cu_seqlens.tolist()
    hit = torch.zeros(got.shape[:2], dtype=torch.bool, device=dev)
    for r, token, head in ((0, 270, 0), (1, 101, 1), (2, 309, 0)):
        hit[first[r] + token:first[r + 1], head * G:(head + 1) * G] = True
    assert bool(got[hit][:, 9].isnan().all()) and (which == "v" or bool(got[hit].isnan().all()))
    assert bool(got[~hit].isfinite().all())
    check(got[~hit], want[~hit], tol[~hit])


def test_scales_that_16_bits_cannot_hold(dev):  # noqa: F811
    """V scales up to 2^127: results that are in bf16's range are what they are with single tokens."""
    tables, cache, step, q, _ = prompts(dev, [600, 37], [300, 260], 32, 8, 128, 64, torch.bfloat16, 47)
    cache.v_scale.mul_(2.0 ** 100)
    cache.v_scale[tables.table[0, 2], 3] = 2.0 ** 123
    cache.v.view(torch.uint8)[tables.table[0, 2], 3] &= 0xB7  # (at most 15, so that 32 bits hold the numbers)
    want, tol = attend(q, cache, tables, step)
    check(fsa.flash_sparse_attn_cache_func(q, cache, tables, step), want, tol)
    assert through_c(q, cache, tables, step)[1] == 0
