"""Attention over the paged 8-bit cache with a sliding window and sinks: single tokens, drafts and prompt parts, against the definition in
64 bits."""
import math

import pytest
import torch

import flash_sparse_attn as fsa
from test_gpu_cache import ATTEND, check, dev, filled, ints, widen  # noqa: F401

pytestmark = pytest.mark.gpu


def attend(query, cache, tables, step, window, sinks, kept=None, bias=None):
    """(result, tolerance) in 64 bits, request by request; roundings as without a window (test_gpu_cache.attend)."""
    T, H, d = query.shape
    Hk, bs, scale = cache.k.shape[1], tables.block_size, query.shape[2] ** -0.5
    out = torch.zeros((T, H, d), dtype=torch.float64, device=query.device)
    tol = torch.zeros_like(out)
    cu, length = step.cu_seqlens.tolist(), step.lengths.tolist()
    u = torch.finfo(query.dtype).eps / 2
    for r, granted in enumerate(step.granted.tolist()):
        n, L = cu[r + 1] - cu[r], length[r]
        if not granted or n == 0:
            continue
        blocks = tables.table[r, :-(-L // bs)].long()
        G = H // Hk
        k, v = ((x[blocks].double() * s[blocks].double()[..., None, None]).transpose(0, 1).reshape(Hk, -1, d)[:, :L].repeat_interleave(G, 0)
                for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
        q = query[cu[r]:cu[r + 1]].double().transpose(0, 1)
        pos, t = torch.arange(L, device=query.device), L - n + torch.arange(n, device=query.device)[:, None]
        seen = ((pos <= t) & ((t - pos < window) | (pos < sinks)))[None].expand(H, n, L).clone()
        if kept is not None:
            there = torch.zeros((H, 1, L), dtype=torch.bool, device=query.device)
            for h in range(H):
                i, j = (r if kept.key_pos.shape[0] > 1 else 0), (h // G if kept.key_pos.shape[1] > 1 else 0)
                p = kept.key_pos[i, j, :int(kept.count[i, j])].long()
                there[h, 0, p[p < L]] = True
            seen &= there
        b = torch.zeros((H, 1, L), dtype=torch.float64, device=query.device)
        if bias is not None:
            row = bias[r if bias.shape[0] > 1 else 0].double().repeat_interleave(H // bias.shape[1], 0)
            m = min(L, row.shape[-1])
            b[..., :m] = row[..., :m]
        k = torch.where(seen.any(1)[..., None], k, 0.0)  # (NaN that nobody sees)
        v = torch.where(seen.any(1)[..., None], v, 0.0)
        s = scale * (q @ k.transpose(1, 2))
        err = scale * d * 2.0 ** -23 * (q.abs() @ k.abs().transpose(1, 2)) + 2.0 ** -22 * (s.abs() + b.abs())
        x = (s + b).masked_fill(~seen, -math.inf)
        top = x.amax(-1, keepdim=True)
        p = (x - top.masked_fill(top == -math.inf, 0.0)).exp()
        l = p.sum(-1, keepdim=True)
        p = p / l.masked_fill(l == 0, 1.0)
        y = p @ v
        worst = torch.where(seen, 2 * err + 2.0 ** -22 * (x - top).abs().clamp(max=1e4), 0.0).nan_to_num(0.0).amax(-1, keepdim=True)
        rounding = 2.0 ** -11 if n < 32 else u
        out[cu[r]:cu[r + 1]] = y.transpose(0, 1)
        tol[cu[r]:cu[r + 1]] = ((rounding + 2 * worst.expm1()) * (p @ v.abs()) + u * y.abs() + 2.0 ** -30 * v.abs().amax()).transpose(0, 1)
    return out, tol + torch.finfo(query.dtype).tiny


def case(dev, cached, new, H, Hk, d, bs, dtype, seed=6):  # noqa: F811
    tables, cache, step, g = filled(dev, len(cached), cached, new, Hk, d, bs, seed)
    T = sum(new)
    kv = torch.randn((2, T, Hk, d), generator=g, device=dev).to(dtype)
    fsa.cache_append(cache, tables, step, kv[0], kv[1])
    return tables, cache, step, torch.randn((T, H, d), generator=g, device=dev).to(dtype), g


WINDOWS = [(1, 0), (64, 4), (100, 70), (1000, 1)]


@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cached,new,H,Hk,d,bs", ATTEND)
def test_windows(dev, dtype, cached, new, H, Hk, d, bs, window, sinks):  # noqa: F811
    tables, cache, step, q, _ = case(dev, cached, new, H, Hk, d, bs, dtype)
    want = attend(q, cache, tables, step, window, sinks)
    args = dict(sliding_window=window, sink_tokens=sinks)
    check(fsa.flash_sparse_attn_cache_func(q, cache, tables, step, **args), *want)
    check(fsa.flash_sparse_attn_cache_func(q, cache, tables, step, max_seqlen_q=max(new), max_seqlen_k=max(step.lengths.tolist()), **args), *want)
    check(fsa.flash_sparse_attn_cache_func(q, cache, widen(tables), step, max_seqlen_q=max(new), **args), *want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cached,new,H,Hk,d,bs,window,sinks", [
    ([2000, 37, 0], [200, 260, 300], 32, 8, 128, 64, 300, 4), ([3000, 3], [400, 33], 32, 4, 64, 16, 64, 100),
    ([1000, 0], [256, 1000], 16, 16, 96, 128, 129, 1), ([4000], [300], 16, 1, 256, 128, 500, 64), ([40, 5, 1300, 800], [1, 31, 1, 600], 32, 8, 128, 16, 200, 0),
    ([5000] * 3, [512] * 3, 32, 8, 128, 32, 1000, 65)])
def test_prompt_parts(dev, dtype, cached, new, H, Hk, d, bs, window, sinks):  # noqa: F811
    tables, cache, step, q, _ = case(dev, cached, new, H, Hk, d, bs, dtype, 41)
    want = attend(q, cache, tables, step, window, sinks)
    got = fsa.flash_sparse_attn_cache_func(q, cache, tables, step, sliding_window=window, sink_tokens=sinks)
    check(got, *want)
    got = fsa.flash_sparse_attn_cache_func(q, cache, tables, step, max_seqlen_q=max(new), max_seqlen_k=max(step.lengths.tolist()),
                                           sliding_window=window, sink_tokens=sinks)
    check(got, *want)


@pytest.mark.parametrize("heads", ["one", "kv", "all"])
@pytest.mark.parametrize("with_bias", [False, True])
def test_with_kept_keys_and_bias(dev, heads, with_bias):  # noqa: F811
    H, Hk, keys = 8, 2, 520
    tables, cache, step, q, g = case(dev, [500, 70, 0], [4, 1, 9], H, Hk, 128, 16, torch.bfloat16)
    hb = {"one": 1, "kv": Hk, "all": H}[heads]
    bias = torch.randn((3, hb, 1, keys), generator=g, device=dev).to(torch.bfloat16) if with_bias else None
    args = dict(sliding_window=90, sink_tokens=20)
    check(fsa.flash_sparse_attn_cache_func(q, cache, tables, step, attn_bias=bias, **args), *attend(q, cache, tables, step, 90, 20, bias=bias))
    mask = torch.rand((3, Hk, 1, keys), generator=g, device=dev) < 0.4
    n = mask.sum(-1)[..., 0].to(torch.int32)
    pos = mask[:, :, 0].to(torch.int32).argsort(dim=-1, descending=True, stable=True).to(torch.int32)
    kept = fsa.KeptKeys(pos.contiguous(), n.contiguous(), None, keys)
    want = attend(q, cache, tables, step, 90, 20, kept, bias)
    check(fsa.flash_sparse_attn_cache_func(q, cache, tables, step, attn_mask=kept, attn_bias=bias, **args), *want)
    check(fsa.flash_sparse_attn_cache_func(q, cache, tables, step, attn_mask=mask, attn_bias=bias, **args), *want)


@pytest.mark.parametrize("n", [1, 5, 40])
def test_not_a_number_behind_the_window_is_not_seen(dev, n):  # noqa: F811
    """Between the sinks and the first key that any query sees, tiles' borders included; one that some query sees reaches those alone."""
    H, Hk, d, bs, window, sinks = 8, 2, 128, 16, 100, 5
    tables, cache, step, q, _ = case(dev, [900], [n], H, Hk, d, bs, torch.bfloat16)
    args = dict(sliding_window=window, sink_tokens=sinks, max_seqlen_q=n)
    want = fsa.flash_sparse_attn_cache_func(q, cache, tables, step, **args)
    row = tables.table[0].tolist()
    first = 900 - window + 1  # of the first query
    for x in (cache.k, cache.v):
        for p in list(range(sinks, 70)) + list(range(first - 60, first)):
            x.view(torch.uint8)[row[p // bs], :, p % bs] = 0x7F
    got = fsa.flash_sparse_attn_cache_func(q, cache, tables, step, **args)
    assert bool(want.isfinite().all()) and torch.equal(got, want)
    cache.v.view(torch.uint8)[row[first // bs], 0, first % bs, 3] = 0x7F
    got = fsa.flash_sparse_attn_cache_func(q, cache, tables, step, **args)
    assert bool(got[0, :H // Hk, 3].isnan().all())
    if n < 32:  # (the conversion of more tokens computes everything again from the 8 bits)
        assert torch.equal(got[1:], want[1:]) and torch.equal(got[0, H // Hk:], want[0, H // Hk:])
    else:
        assert bool(got[1:].isfinite().all())


def test_refused_and_padded_tokens_are_zero(dev):  # noqa: F811
    tables = fsa.block_tables(3, 20, 24, 16, device=dev)
    cache = fsa.quantized_cache(24, 1, 64, 16, device=dev)
    kv = torch.randn((2, 320, 1, 64), device=dev, dtype=torch.bfloat16)
    step = tables.extend(ints([200, 300, 90], dev), 320)  # the second one asks for more than there is
    fsa.cache_append(cache, tables, step, kv[0], kv[1])
    q = torch.randn((320, 2, 64), device=dev, dtype=torch.bfloat16)
    got = fsa.flash_sparse_attn_cache_func(q, cache, tables, step, sliding_window=50, sink_tokens=3)
    check(got, *attend(q, cache, tables, step, 50, 3))
    assert step.granted.tolist() == [True, False, False] and not bool(got[200:].any())


def test_window_as_long_as_the_cache(dev):  # noqa: F811
    tables, cache, step, q, _ = case(dev, [700, 0, 12], [5, 9, 1], 12, 4, 128, 16, torch.bfloat16)
    want = fsa.flash_sparse_attn_cache_func(q, cache, tables, step)
    for window, sinks in ((705, 0), (2 ** 31 - 1, 2 ** 31 - 1), (5, 700)):
        got = fsa.flash_sparse_attn_cache_func(q, cache, tables, step, sliding_window=window, sink_tokens=sinks)
        check(got, *attend(q, cache, tables, step, 705, 0))
        assert torch.equal(got, want) or (got.double() - want.double()).abs().max() <= 2.0 ** -7 * want.abs().max()


def test_refusals(dev):  # noqa: F811
    tables, cache, step, q, _ = case(dev, [70], [1], 2, 1, 64, 16, torch.bfloat16)
    for error, args in ((ValueError, dict(sliding_window=0)), (ValueError, dict(sliding_window=-3)), (ValueError, dict(sliding_window=2 ** 31)),
                        (ValueError, dict(sliding_window=4, sink_tokens=-1)), (ValueError, dict(sink_tokens=4)), (TypeError, dict(sliding_window=4.0)),
                        (TypeError, dict(sliding_window=True)), (ValueError, dict(sliding_window=4, is_causal=False))):
        with pytest.raises(error):
            fsa.flash_sparse_attn_cache_func(q, cache, tables, step, **args)


def test_compiled(dev):  # noqa: F811
    tables, cache, step, q, _ = case(dev, [300, 70, 0], [4, 1, 40], 4, 2, 64, 16, torch.bfloat16)
    want = fsa.flash_sparse_attn_cache_func(q, cache, tables, step, sliding_window=90, sink_tokens=20)
    torch._dynamo.reset()
    fn = torch.compile(lambda q: fsa.flash_sparse_attn_cache_func(q, cache, tables, step, sliding_window=90, sink_tokens=20), backend="aot_eager",
                       fullgraph=True)
    assert torch.equal(fn(q), want)


def test_same_bits_every_time_beside_other_launches(dev):  # noqa: F811
    tables, cache, step, q, _ = case(dev, [3000, 70, 0, 900], [4, 1, 300, 9], 8, 2, 128, 16, torch.bfloat16)

    def run():
        return fsa.flash_sparse_attn_cache_func(q, cache, tables, step, sliding_window=500, sink_tokens=4)

    want = run()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    runs = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                runs.append(run())
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in runs)
