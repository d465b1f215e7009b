"""Verification of drafted tokens against its definition in 64 bits. Tokens and counts are whole numbers and have to be equal: the
kernel compares the random numbers with sums whose errors are some 2^-40, which no case here comes near by chance."""
import math

import pytest
import torch

import flash_sparse_attn as fsa
from test_gpu_cache import dev, ints  # noqa: F401

pytestmark = pytest.mark.gpu


def plan(dev, new, lengths=None, granted=None):  # noqa: F811
    R = len(new)
    cu = [sum(new[:i]) for i in range(R + 1)]
    lengths = [17 + 3 * r + n for r, n in enumerate(new)] if lengths is None else lengths
    z = ints([0] * (R + 1), dev)
    return fsa.CacheStep(ints(cu, dev), ints([0] * cu[-1], dev), z.long(), ints(lengths, dev),
                         torch.tensor(granted or [True] * R, device=dev), z, z)


def definition(step, ids, logits, uniforms, probs, temperature):
    """Request by request on the CPU, in Python's and numpy's 64 bits."""
    cu, lengths, granted = step.cu_seqlens.tolist(), step.lengths.tolist(), step.granted.tolist()
    ids, u = ids.tolist(), uniforms.double().tolist()
    x = logits.double().cpu()
    x = torch.where(x.isnan(), -math.inf, x).clamp(max=torch.finfo(torch.float32).max)
    q = None if probs is None else torch.nan_to_num(probs.double().cpu(), nan=0.0, posinf=math.inf).clamp(min=0.0)
    V = x.shape[1]
    out = []
    for r in range(len(lengths)):
        first, n = cu[r], cu[r + 1] - cu[r]
        if n == 0 or not granted[r]:
            out.append((0, -1, lengths[r]))
            continue
        T = temperature[r].item() if isinstance(temperature, torch.Tensor) else temperature
        T = torch.tensor(T, dtype=torch.float32).double().item()
        acc, nxt = 0, None
        while nxt is None:
            row = x[first + acc]
            empty = bool((row == -math.inf).all())
            draft = ids[first + acc + 1] if acc < n - 1 else None
            if not T > 0:
                best = -1 if empty else int((row == row.max()).nonzero()[0])
                if draft is not None and draft == best:
                    acc += 1
                else:
                    nxt = best
                continue
            p = torch.zeros(V, dtype=torch.float64) if empty else torch.exp((row - row.max()) / T)
            p = p / p.sum() if not empty else p
            if draft is not None and 0 <= draft < V and u[first + acc] * (1.0 if q is None else q[first + acc, draft].item()) < p[draft].item():
                acc += 1
                continue
            left = p
            if draft is not None:
                if q is None:
                    left = p.clone()
                    if 0 <= draft < V:
                        left[draft] = 0.0
                else:
                    left = (p - q[first + acc]).clamp(min=0.0)
                if not left.sum() > 0:
                    left = p
            c = left.cumsum(0)
            above = ((c > u[first + n - 1] * c[-1]) & (left > 0)).nonzero()
            some = (left > 0).nonzero()
            nxt = int(above[0]) if len(above) else int(some[-1]) if len(some) else -1
        out.append((acc, nxt, lengths[r] - (n - 1 - acc)))
    return [list(z) for z in zip(*out)]


def check(dev, step, ids, logits, uniforms, probs=None, temperature=1.0):  # noqa: F811
    got = fsa.verify_drafts(step, ids, logits, uniforms, probs, temperature)
    want = definition(step, ids, logits, uniforms, probs, temperature)
    assert [x.tolist() for x in got] == want
    assert got.next_tokens.dtype == torch.int64 and got.accepted.dtype == got.lengths.dtype == torch.int32
    return got


def drafts(dev, new, V, dtype, probs_dtype, seed, sure=3.0):  # noqa: F811
    g = torch.Generator(device=dev).manual_seed(seed)
    T = sum(new)
    logits = torch.randn((T, V), generator=g, device=dev) * sure
    guess = logits + torch.randn((T, V), generator=g, device=dev) * 0.5
    probs = torch.softmax(guess, -1).to(probs_dtype) if probs_dtype else None
    ids = torch.multinomial(torch.softmax(guess, -1), 1, generator=g)[:, 0].roll(1)
    return ids, logits.to(dtype), torch.rand(T, generator=g, device=dev), probs


@pytest.mark.parametrize("probs", [None, torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("new,V", [([1], 1), ([3, 1, 2], 5), ([4], 1000), ([1, 5, 0, 9, 2], 2049), ([6, 3], 32000), ([40, 17], 777),
                                   ([2, 3, 1] * 60, 1023), ([3] * 3, 50257)], ids=str)
def test_drafts(dev, new, V, dtype, probs):  # noqa: F811
    ids, logits, uniforms, q = drafts(dev, new, V, dtype, probs, 3)
    for temperature in (1.0, 0.0, 0.6, (torch.arange(len(new), device=dev) % 3).float() * 0.5):
        check(dev, plan(dev, new), ids, logits, uniforms, q, temperature)


def test_a_large_vocabulary(dev):  # noqa: F811
    ids, logits, uniforms, q = drafts(dev, [5, 2], 300001, torch.bfloat16, torch.float32, 5)
    check(dev, plan(dev, [5, 2]), ids.to(torch.int32), logits, uniforms, q)
    check(dev, plan(dev, [5, 2]), ids, logits, uniforms)


def test_layouts(dev):  # noqa: F811
    """Rows that begin anywhere, rows of a wider matrix, transposed memory, refused requests, rows behind the last one."""
    new, V = [3, 2, 4, 1], 1237
    ids, logits, uniforms, q = drafts(dev, new + [3], V, torch.bfloat16, torch.float32, 7)
    step = plan(dev, new, granted=[True, False, True, True])
    want = fsa.verify_drafts(step, ids, logits, uniforms, q)
    check(dev, step, ids, logits, uniforms, q)
    for skip in (1, 3, 8):
        wide, wide_q = (torch.full((t.shape[0], V + 20), math.nan, dtype=t.dtype, device=dev) for t in (logits, q))
        wide[:, skip:skip + V], wide_q[:, skip + 1:skip + 1 + V] = logits, q
        got = fsa.verify_drafts(step, ids, wide[:, skip:skip + V], uniforms, wide_q[:, skip + 1:skip + 1 + V])
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    got = fsa.verify_drafts(step, ids, logits.t().contiguous().t(), uniforms, q.t().contiguous().t())
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_special_numbers(dev):  # noqa: F811
    V = 100
    logits = torch.zeros((16, V), device=dev)
    logits[0] = -math.inf                       # nothing to draw from
    logits[1, 1:] = -math.inf                   # one token left, the draft
    logits[2], logits[2, 7] = -math.inf, 2.0
    logits[3, 40] = math.nan
    logits[4, 9], logits[4, 50] = math.inf, math.inf
    logits[5] = torch.finfo(torch.float32).min  # an even row of the lowest numbers
    logits[6, ::2] = -math.inf
    q = torch.full((16, V), 1.0 / V, device=dev)
    q[7] = 0.0                                  # a draft that could not have been drawn
    q[8, 3], q[8, 4] = math.nan, -1.0
    q[9] = 1.0                                  # sure of everything: nothing left over
    q[10, 5] = math.inf
    ids = torch.tensor([3, 3, 0, 7, 40, 9, 99, 0, 8, 3, 4, -1, 100, 2 ** 40, 6, 1], device=dev)
    new = [2] * 8
    for u in (0.0, 0.3, 1 - 2.0 ** -24):
        uniforms = torch.full((16,), u, device=dev)
        for temperature in (1.0, 0.0, 1e-30, 1e30):
            for shift in range(2):  # each row as a draft's own, and as the last one
                x, y = logits.roll(shift, 0), q.roll(shift, 0)
                check(dev, plan(dev, new), ids, x, uniforms, y, temperature)
                check(dev, plan(dev, new), ids, x, uniforms, None, temperature)
    odd = torch.tensor([math.nan, -1.0, math.inf, 0.0, 1e-45, 3e38, 1.0, 1.0], device=dev)
    got = fsa.verify_drafts(plan(dev, new), ids, logits[11:12].expand(16, V), uniforms, None, odd)
    assert got.next_tokens[0].item() == 0 and got.next_tokens[1].item() == 0  # not above 0: the largest, the first of them
    with_inf = logits.clone()
    got = fsa.verify_drafts(plan(dev, new), ids, with_inf, uniforms, q, torch.full((8,), math.inf, device=dev))
    assert bool((got.next_tokens >= -1).all()) and bool((got.next_tokens < V).all())


def test_equal_logits_go_to_the_first(dev):  # noqa: F811
    for V in (3, 1000, 40000):
        logits = torch.randint(0, 3, (8, V), device=dev).to(torch.bfloat16)
        ids = torch.cat([torch.tensor([0], device=dev), logits.float().argmax(-1)[:-1]])
        check(dev, plan(dev, [8]), ids, logits, torch.rand(8, device=dev), None, 0.0)


@pytest.mark.parametrize("V", [10, 3000])
def test_numbers_beside_a_border(dev, V):  # noqa: F811
    """Random numbers that are the 32-bit neighbours of the very ratio p / q: 32-bit sums could not tell them apart."""
    g = torch.Generator(device=dev).manual_seed(V)
    n = 9
    logits = torch.randn((n * 20, V), generator=g, device=dev)
    q = torch.softmax(torch.randn((n * 20, V), generator=g, device=dev), -1)
    ids = torch.randint(0, V, (n * 20,), generator=g, device=dev)
    p = torch.softmax(logits.double(), -1)
    ratio = (p[:-1].gather(1, ids[1:, None]) / q[:-1].double().gather(1, ids[1:, None]))[:, 0].clamp(max=0.999999).float()
    for way in (-1, 0, 1):
        u = ratio if way == 0 else torch.nextafter(ratio, torch.full_like(ratio, float(way)))
        check(dev, plan(dev, [n] * 20), ids, logits, torch.cat([u, u.new_tensor([0.5])]), q)


def test_tokens_are_distributed_as_the_targets(dev):  # noqa: F811
    """One draft each: accepted or replaced, the first new token has the target's probabilities. 200 000 requests, 12 tokens: a count is off by
    less than six standard deviations."""
    R, V = 200000, 12
    g = torch.Generator(device=dev).manual_seed(1)
    p, q = (torch.softmax(torch.randn(V, generator=g, device=dev) * 1.5, -1) for _ in range(2))
    x = torch.multinomial(q, R, replacement=True, generator=g)
    ids = torch.stack((torch.zeros_like(x), x), 1).flatten()
    step = fsa.CacheStep(torch.arange(R + 1, dtype=torch.int32, device=dev) * 2, ids.int(), ids, torch.full((R,), 9, dtype=torch.int32, device=dev),
                         torch.ones(R, dtype=torch.bool, device=dev), ids.int(), ids.int())
    got = fsa.verify_drafts(step, ids, p.log().expand(2 * R, V), torch.rand(2 * R, generator=g, device=dev), q.expand(2 * R, V))
    first = torch.where(got.accepted == 1, x, got.next_tokens)
    count = torch.bincount(first, minlength=V).double()
    want = p.double()
    assert bool(((count - R * want).abs() < 6 * (R * want * (1 - want)).sqrt()).all())
    assert abs(got.accepted.double().mean().item() - torch.minimum(p, q).sum().item()) < 0.01


def test_a_step_with_its_tables(dev):  # noqa: F811
    """extend, append, attend, verify, truncate, captured once and replayed with other drafts: as step by step without a graph."""
    R, V, H, Hk, d, n = 3, 501, 4, 2, 64, 4
    g = torch.Generator(device=dev).manual_seed(2)
    emb, head = torch.randn((V, 3 * H * d), generator=g, device=dev, dtype=torch.bfloat16), torch.randn((H * d, V), generator=g, device=dev, dtype=torch.bfloat16) * 0.1

    def state():
        tables = fsa.block_tables(R, 20, 60, 16, device=dev)
        tables.extend(ints([30, 5, 77], dev), 112)
        cache = fsa.quantized_cache(60, Hk, d, 16, device=dev)
        return tables, cache

    def step_of(tables, cache, new, ids, u):
        step = tables.extend(new, R * n)
        x = emb[ids]
        q, k, v = (y.reshape(-1, h, d) for y, h in zip(x.split((H * d, Hk * d, Hk * d), 1), (H, Hk, Hk)))
        fsa.cache_append(cache, tables, step, k, v)
        out = fsa.flash_sparse_attn_cache_func(q, cache, tables, step, sliding_window=24, sink_tokens=4, max_seqlen_q=n)
        done = fsa.verify_drafts(step, ids, out.flatten(1) @ head, u)
        tables.truncate(done.lengths)
        return done

    emb = emb[:, :(H + 2 * Hk) * d].contiguous()
    new, ids, u = ints([n, n, n], dev), torch.zeros(R * n, dtype=torch.long, device=dev), torch.zeros(R * n, device=dev)
    tables, cache = state()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        keep = [t.clone() for t in tables[:5]]
        step_of(tables, cache, new, ids, u)
        for t, x in zip(tables[:5], keep):
            t.copy_(x)
        for t in cache:
            t.view(torch.uint8).zero_() if t.dtype == torch.float8_e4m3fn else t.fill_(1)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            done = step_of(tables, cache, new, ids, u)
    torch.cuda.synchronize()
    others = state()
    some = 0
    for i in range(5):
        new.copy_(torch.tensor([n, (i % 2) * 2, 1 + i % n]))
        ids.copy_(torch.randint(0, V, (R * n,), generator=g, device=dev))
        u.copy_(torch.rand(R * n, generator=g, device=dev) * 0.01)
        graph.replay()
        want = step_of(*others, new, ids, u)
        torch.cuda.synchronize()
        for x, y in zip(done, want):
            assert torch.equal(x, y)
        assert torch.equal(tables.lengths, others[0].lengths) and torch.equal(tables.lengths, done.lengths)
        some += int(done.accepted.sum())
    assert some > 0


def test_rows_gathered_from_a_step_with_a_prompt_part(dev):  # noqa: F811
    new, V = [300, 4, 0, 1], 700
    step = plan(dev, new)
    ids, logits, u, q = drafts(dev, new, V, torch.bfloat16, torch.float32, 6)
    rows = torch.tensor([299, 300, 301, 302, 303, 304], device=dev)
    part = step._replace(cu_seqlens=ints([0, 1, 5, 5, 6], dev))
    got = check(dev, part, ids[rows], logits[rows], u[rows], q[rows], 0.9)
    assert got.lengths[0] == step.lengths[0] and got.lengths[3] == step.lengths[3]


def test_refusals(dev):  # noqa: F811
    new, V = [2, 3], 50
    ids, logits, u, q = drafts(dev, new, V, torch.float32, torch.float32, 1)
    step = plan(dev, new)
    fsa.verify_drafts(step, ids, logits, u, q)
    for bad in (dict(token_ids=ids[:4]), dict(token_ids=ids.float()), dict(token_ids=ids.cpu()), dict(logits=logits[0]), dict(logits=logits.double()),
                dict(logits=logits[:, :0]), dict(uniforms=u.double()), dict(uniforms=u[:3]), dict(draft_probs=q[:4]), dict(draft_probs=q.double()),
                dict(draft_probs=q[:, :9]), dict(temperature=torch.ones(3, device=dev)), dict(temperature=torch.ones(2)),
                dict(temperature=torch.ones(2, device=dev).double()), dict(step=step._replace(granted=step.granted[:1])),
                dict(step=step._replace(lengths=step.lengths.long())), dict(step=step._replace(cu_seqlens=step.cu_seqlens[:2])),
                dict(logits=logits.clone().requires_grad_())):
        with pytest.raises(RuntimeError):
            fsa.verify_drafts(**{**dict(step=step, token_ids=ids, logits=logits, uniforms=u, draft_probs=q), **bad})
    for t in (-1.0, math.nan, math.inf):
        with pytest.raises(ValueError):
            fsa.verify_drafts(step, ids, logits, u, q, temperature=t)


def test_no_tokens(dev):  # noqa: F811
    step = plan(dev, [0, 0])
    got = fsa.verify_drafts(step, torch.zeros(0, dtype=torch.long, device=dev), torch.zeros((0, 7), device=dev), torch.zeros(0, device=dev))
    assert got.accepted.tolist() == [0, 0] and got.next_tokens.tolist() == [-1, -1] and got.lengths.tolist() == step.lengths.tolist()


def test_compiled(dev):  # noqa: F811
    new = [2, 3]
    ids, logits, u, q = drafts(dev, new, 900, torch.bfloat16, torch.float32, 4)
    step = plan(dev, new)
    want = fsa.verify_drafts(step, ids, logits, u, q, 0.8)
    got = torch.compile(lambda x: fsa.verify_drafts(step, ids, x, u, q, 0.8), fullgraph=True)(logits)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
