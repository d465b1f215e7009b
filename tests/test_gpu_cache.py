"""The paged 8-bit cache: block tables against lists in Python, the writer and the attention against their definitions in 64 bits."""
import math

import pytest
import torch

import flash_sparse_attn as fsa
from test_gpu_rotary import inv_freq, turn

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda:0")


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


# ---- block tables ------------------------------------------------------------------------------------------------------
class Model:
    """The tables as lists."""

    def __init__(self, requests, width, num_blocks, block_size):
        self.rows, self.lengths, self.width, self.bs = [[] for _ in range(requests)], [0] * requests, width, block_size
        self.free = list(range(num_blocks - 1, -1, -1))

    def extend(self, new, tokens):
        new = [max(0, n) for n in new]
        cu, pos, slots, granted, blocks, chunks, end, asked = [0], [], [], [], [0], [0], 0, 0
        count = len(self.free)
        for r, n in enumerate(new):
            have, end = self.lengths[r], end + n
            want = -(-(have + n) // self.bs)
            ok = n == 0
            if n and want <= self.width and end <= tokens:
                need = want - len(self.rows[r])
                asked += need
                ok = need == 0 or asked <= count
            if ok:
                while len(self.rows[r]) < want:
                    self.rows[r].append(self.free.pop())
                self.lengths[r] += n
            for i in range(n):
                if len(pos) < tokens:
                    p = have + i
                    pos.append(p)
                    slots.append(self.rows[r][p // self.bs] * self.bs + p % self.bs if ok else -1)
            active = ok and n > 0
            cu.append(min(end, tokens))
            granted.append(ok)
            blocks.append(blocks[-1] + (want - have // self.bs if active else 0))
            chunks.append(chunks[-1] + (-(-self.lengths[r] // 64) if active else 0))
        pad = tokens - len(pos)
        return dict(cu_seqlens=cu, positions=pos + [0] * pad, slots=slots + [-1] * pad, lengths=list(self.lengths), granted=granted,
                    cu_blocks=blocks, cu_chunks=chunks)

    def truncate(self, lengths):
        gone = []
        for r, n in enumerate(lengths):
            self.lengths[r] = min(self.lengths[r], max(0, n))
            keep = -(-self.lengths[r] // self.bs)
            gone += self.rows[r][keep:]
            self.rows[r] = self.rows[r][:keep]
        self.free += gone[::-1]

    def check(self, tables):
        assert tables.lengths.tolist() == self.lengths
        assert tables.table.tolist() == [row + [-1] * (self.width - len(row)) for row in self.rows]
        assert tables.free_count.tolist() == [len(self.free)] and tables.ticket.tolist() == [0]
        assert tables.free[:len(self.free)].tolist() == self.free


@pytest.mark.parametrize("requests,width,num_blocks,bs,most", [(1, 3, 2, 16, 20), (7, 40, 90, 32, 300), (300, 12, 1500, 16, 40),
                                                              (1500, 4, 3000, 128, 200), (8192, 2, 9000, 16, 9)])
def test_tables(dev, requests, width, num_blocks, bs, most):
    g = torch.Generator().manual_seed(requests)
    tables = fsa.block_tables(requests, width, num_blocks, bs, device=dev)
    model = Model(requests, width, num_blocks, bs)
    model.check(tables)
    for i in range(8):
        new = torch.randint(-1, most, (requests,), generator=g)
        if i % 2:
            new[torch.rand(requests, generator=g) < 0.5] = 0
        tokens = int(new.clamp(min=0).sum()) + (0, 5, -3)[i % 3]
        tokens = max(tokens, 0)
        before = tables.lengths.clone()
        step = tables.extend(new.to(torch.int32).to(dev), tokens)
        for name, want in model.extend(new.tolist(), tokens).items():
            assert getattr(step, name).tolist() == want, (i, name)
        model.check(tables)
        if i % 4 == 1:  # as a rejected draft: everything is as it was
            free = (tables.free.clone(), tables.free_count.clone())
            tables.truncate(before)
            model.truncate(before.tolist())
        else:
            free = None
            back = (torch.rand(requests, generator=g) * 1.5 * tables.lengths.cpu()).to(torch.int32)
            tables.truncate(back.to(dev))
            model.truncate(back.tolist())
        model.check(tables)
    tables.truncate(torch.zeros_like(tables.lengths))
    assert tables.free_count.item() == num_blocks and sorted(tables.free.tolist()) == list(range(num_blocks))


def test_tables_without_tokens(dev):
    tables = fsa.block_tables(3, 2, 4, 16, device=dev)
    step = tables.extend(ints([0, 0, 0], dev), 0)
    assert step.slots.numel() == 0 and step.granted.tolist() == [True] * 3 and tables.free_count.item() == 4
    step = tables.extend(ints([2 ** 31 - 1, 1, 1], dev), 2)  # far too many tokens: refused, and with it what ends behind them
    assert step.granted.tolist() == [False] * 3 and step.slots.tolist() == [-1, -1] and tables.lengths.tolist() == [0, 0, 0]


def test_tables_refusals(dev):
    t = fsa.block_tables(2, 2, 4, 16, device=dev)
    good = ints([1, 1], dev)
    for bad in (good.cpu(), good.long(), good[:1], ints([[1, 1]], dev), ints([1, 9, 1, 9], dev)[::2]):
        with pytest.raises(RuntimeError):
            t.extend(bad, 2)
        with pytest.raises(RuntimeError):
            t.truncate(bad)
    for wrong in (t._replace(block_size=24), t._replace(table=t.table.cpu()), t._replace(free=t.free.long()), t._replace(lengths=t.lengths[:1]),
                  t._replace(ticket=t.ticket[:0])):
        with pytest.raises(RuntimeError):
            wrong.extend(good, 2)
    with pytest.raises(RuntimeError):
        t.extend(good, -1)
    t.extend(good, 2)


# ---- the writer --------------------------------------------------------------------------------------------------------
def exponent(x):
    """The smallest e from -100 on with x <= 448 * 2^e."""
    if x == 0:
        return -100
    m, e = math.frexp(x)
    return max(-100, e - 9 + (m > 0.875))


def filled(dev, requests, cached, new, Hk, d, bs, seed, spare=2):
    """Tables and a cache of random contents with `cached` tokens per request, and the step of `new` more; the cache's unused places
    are NaN."""
    g = torch.Generator(device=dev).manual_seed(seed)
    R = len(cached)
    blocks = sum(-(-(a + b) // bs) for a, b in zip(cached, new)) + spare
    width = max(1, max(-(-(a + b) // bs) for a, b in zip(cached, new)))
    tables = fsa.block_tables(R, width, blocks, bs, device=dev)
    tables.free.copy_(torch.randperm(blocks, generator=g, device=dev).to(torch.int32))
    tables.extend(ints(cached, dev), sum(cached))
    cache = fsa.quantized_cache(blocks, Hk, d, bs, device=dev)
    for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        x.copy_((torch.randn(x.shape, generator=g, device=dev) * 60).clamp(-448, 448).to(E4M3))
        s.copy_(torch.exp2(torch.randint(-9, -3, s.shape, generator=g, device=dev).float()))
        used = torch.zeros(blocks, bs, dtype=torch.bool, device=dev)
        for r, n in enumerate(cached):
            for p in range(0, n, bs):
                used[tables.table[r, p // bs], :min(bs, n - p)] = True
        x.view(torch.uint8).masked_fill_(~used[:, None, :, None], 0x7F)
    total = sum(new)
    step = tables.extend(ints(new, dev), total)
    return tables, cache, step, g


def written(cache, tables, step, key, value):
    """(values, scales) of k and v after the write of key and value (64 bits, on the CPU)."""
    out = []
    cu, length, table, bs = step.cu_seqlens.tolist(), step.lengths.tolist(), tables.table.tolist(), tables.block_size
    for x, old, scale in ((key, cache.k, cache.k_scale), (value, cache.v, cache.v_scale)):
        values, scales, x = old.cpu().double() , scale.cpu().double(), x.cpu().double()
        for r, granted in enumerate(step.granted.tolist()):
            n = cu[r + 1] - cu[r]
            if not granted or n == 0:
                continue
            start = length[r] - n
            for page in range(start // bs, -(-length[r] // bs)):
                b, lo, hi = table[r][page], max(start - page * bs, 0), min(length[r] - page * bs, bs)
                for h in range(x.shape[1]):
                    rows = x[cu[r] + page * bs + lo - start:cu[r] + page * bs + hi - start, h]
                    finite = rows[rows.isfinite()].abs()
                    e = 2.0 ** exponent(finite.max().item() if finite.numel() else 0.0)
                    if lo > 0:
                        e = max(e, scales[b, h].item())
                        values[b, h, :lo] = (values[b, h, :lo] * scales[b, h] / e).to(E4M3).double()
                    values[b, h, lo:hi] = (rows / e).clamp(-448, 448).to(E4M3).double()
                    scales[b, h] = e
        out.append((values, scales))
    return out


SHAPES = [  # cached, new, kv heads, head dim, block size
    ([0], [1], 1, 64, 16), ([0, 5, 16, 31], [1, 1, 1, 1], 2, 128, 16), ([0, 63, 64, 100], [130, 1, 64, 29], 3, 96, 64),
    ([7, 0, 128], [300, 0, 5], 1, 256, 128), ([33] * 9, [4] * 9, 8, 16, 32), ([1], [500], 2, 80, 16)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cached,new,Hk,d,bs", SHAPES)
def test_append_without_rotation_is_bit_exact(dev, dtype, cached, new, Hk, d, bs):
    """Scales are powers of two, so every number has one correct value: bytes are equal."""
    tables, cache, step, g = filled(dev, len(cached), cached, new, Hk, d, bs, 3)
    T = sum(new)
    size = torch.exp2(torch.randint(-8, 9, (T, Hk, 1), generator=g, device=dev).float())  # some blocks' scales grow, some do not
    key = (torch.randn((T, Hk, d), generator=g, device=dev) * size).to(dtype)
    value = (torch.randn((T, Hk, d), generator=g, device=dev)).to(dtype)
    want = written(cache, tables, step, key, value)
    assert fsa.cache_append(cache, tables, step, key, value) is None
    for (values, scales), x, s in zip(want, (cache.k, cache.v), (cache.k_scale, cache.v_scale)):
        assert torch.equal(s.cpu().double(), scales)
        got = x.cpu().double()
        assert torch.equal(got.isnan(), values.isnan()) and torch.equal(got.nan_to_num(), values.nan_to_num())
    again = [t.clone().view(torch.uint8) if t.dtype == E4M3 else t.clone() for t in cache]
    fsa.cache_append(cache, tables, step, key, value)  # the same step once more changes nothing
    for a, b in zip(again, cache):
        assert torch.equal(a, b.view(torch.uint8) if b.dtype == E4M3 else b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rd,inter", [(0, False), (0, True), (32, False), (10, True)])
@pytest.mark.parametrize("cached,new,Hk,d,bs", SHAPES)
def test_append_with_rotation(dev, dtype, cached, new, Hk, d, bs, rd, inter):
    """A turned key is off by 2^-20 of its terms before it is rounded to four bits (2^-4 of itself, or 2^-10 scales among the smallest
    numbers); the scale of its block is one of the two powers of two where the largest is that near to the border."""
    rd = min(rd or d, d)
    tables, cache, step, g = filled(dev, len(cached), cached, new, Hk, d, bs, 4)
    T, H = sum(new), 2 * Hk
    key, value = (torch.randn((T, Hk, d), generator=g, device=dev).to(dtype) for _ in range(2))
    query = torch.randn((T, H, d), generator=g, device=dev).to(dtype)
    f = fsa.rotary_frequencies(rd, interleaved=inter, amplitude=1.5, device=dev)
    inv = inv_freq(rd, dev)
    turned, size = turn(key, step.positions, inv, 1.5, inter)
    (_, k_scale), (v_values, v_scale) = written(cache, tables, step, turned, value)
    q = fsa.cache_append(cache, tables, step, key, value, query=query, frequencies=f)
    both = fsa.apply_rotary(query, key, f, step.positions)
    assert torch.equal(q, both[0])
    assert torch.equal(cache.v_scale.cpu().double(), v_scale)
    assert torch.equal(cache.v.cpu().double().nan_to_num(), v_values.nan_to_num())
    assert bool(((cache.k_scale.cpu().double() / k_scale).log2().abs() <= 1).all())
    near = (cache.k_scale.cpu().double() != k_scale)
    assert near.float().mean() <= 0.01
    slots = step.slots
    rows = cache.k[slots // bs, :, slots % bs].double() * cache.k_scale[slots // bs].double()[..., None]
    step_size = cache.k_scale[slots // bs].double()[..., None]
    tol = 2.0 ** -4 * turned.abs() + 2.0 ** -10 * step_size + 2.0 ** -19 * size
    assert bool(((rows - turned).abs() <= tol).all())


def test_append_special_values(dev):
    tables, cache, step, g = filled(dev, 3, [0, 3, 0], [5, 2, 1], 1, 32, 16, 5)
    key = torch.randn((8, 1, 32), generator=g, device=dev, dtype=torch.bfloat16)
    value = torch.zeros_like(key)
    key[0, 0, 3], key[1, 0, 4], key[2, 0, 5], key[5, 0, 6] = math.inf, -math.inf, math.nan, math.nan
    value[7, 0, 0] = 3.0e38
    want = written(cache, tables, step, key, value)
    fsa.cache_append(cache, tables, step, key, value)
    for (values, scales), x, s in zip(want, (cache.k, cache.v), (cache.k_scale, cache.v_scale)):
        assert torch.equal(s.cpu().double(), scales)
        got = x.cpu().double()
        assert torch.equal(got.isnan(), values.isnan()) and torch.equal(got.nan_to_num(), values.nan_to_num())
    b = step.slots[0].item() // 16
    assert cache.k[b, 0, 0, 3].item() == 448 and cache.k[b, 0, 1, 4].item() == -448 and math.isnan(cache.k[b, 0, 2, 5].item())
    assert cache.v_scale[b, 0].item() == 2.0 ** -100  # nothing but zeros


def test_append_layouts_and_refused_tokens(dev):
    """Slices of a fused projection, an odd offset; tokens of a refused request and behind the last one are written nowhere."""
    tables = fsa.block_tables(3, 2, 2, 16, device=dev)
    cache = fsa.quantized_cache(2, 2, 64, 16, device=dev)
    step = tables.extend(ints([16, 40, 3], dev), 64)
    assert step.granted.tolist() == [True, False, True]
    fused = torch.randn((64, 6, 64), device=dev, dtype=torch.float16)
    f = fsa.rotary_frequencies(64, device=dev)
    q = fsa.cache_append(cache, tables, step, fused[:, 2:4], fused[:, 4:6], query=fused[:, :2], frequencies=f)
    assert torch.equal(q, fsa.apply_rotary(fused[:, :2], None, f, step.positions)[0])
    want = [t.clone() for t in cache]
    odd = torch.empty(64 * 6 * 64 + 1, device=dev, dtype=torch.float16)[1:].view(64, 6, 64).copy_(fused)
    other = fsa.quantized_cache(2, 2, 64, 16, device=dev)
    fsa.cache_append(other, tables, step, odd[:, 2:4], odd[:, 4:6], query=odd[:, :2], frequencies=f)
    for a, b in zip(want, other):
        assert torch.equal(a.float(), b.float())
    third = step.slots[56].item() // 16
    assert not bool(cache.k[third, :, 3:].float().any())


# ---- attention ---------------------------------------------------------------------------------------------------------
def attend(query, cache, tables, step, kept=None, bias=None, scale=None, causal=True):
    """(result, tolerance) in 64 bits, request by request.

    Scores are sums of d exact products in 32 bits, at worst 2^-23 of their magnitudes per addition, times two factors and plus a bias
    (2^-22 of what they are added to): that makes an error of the score, and so of a probability relative to itself, twice (numerator
    and sum). Probabilities are rounded to fp16, 2^-11 of themselves, or 2^-38 of the largest times a value; for requests with 32 or more
    new tokens to the type of the queries, eps / 2. One rounding to the type."""
    T, H, d = query.shape
    Hk, bs = cache.k.shape[1], tables.block_size
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros((T, H, d), dtype=torch.float64, device=query.device)
    tol = torch.zeros_like(out)
    cu, length = step.cu_seqlens.tolist(), step.lengths.tolist()
    for r, granted in enumerate(step.granted.tolist()):
        n = cu[r + 1] - cu[r]
        if not granted or n == 0:
            continue
        blocks = tables.table[r, :-(-length[r] // bs)].long()
        for h in range(H):
            hk = h // (H // Hk)
            k, v = ((x[blocks, hk].double() * s[blocks, hk].double()[:, None, None]).reshape(-1, d)[:length[r]]
                    for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
            pos = torch.arange(length[r], device=query.device)
            b = torch.zeros(length[r], dtype=torch.float64, device=query.device)
            if bias is not None:
                row = bias[r if bias.shape[0] > 1 else 0, 0 if bias.shape[1] == 1 else hk if bias.shape[1] == Hk else h, 0].double()
                m = min(length[r], row.shape[0])
                b[:m] = row[:m]
            if kept is not None:
                i, j = (r if kept.key_pos.shape[0] > 1 else 0), (hk if kept.key_pos.shape[1] > 1 else 0)
                pos = kept.key_pos[i, j, :int(kept.count[i, j])].long()
                pos = pos[pos < length[r]]
                k, v, b = k[pos], v[pos], b[pos]
            q = query[cu[r]:cu[r + 1], h].double()
            s = scale * (q @ k.T)
            x = s + b
            err = abs(scale) * d * 2.0 ** -23 * (q.abs() @ k.abs().T) + 2.0 ** -22 * (s.abs() + b.abs())
            if causal:
                hide = pos[None, :] > length[r] - n + torch.arange(n, device=query.device)[:, None]
                x, err = x.masked_fill(hide, -math.inf), err.masked_fill(hide, 0.0)
            err = err.masked_fill(x == -math.inf, 0.0)
            top = x.amax(-1, keepdim=True) if x.shape[1] else torch.full((n, 1), -math.inf, dtype=torch.float64, device=query.device)
            p = (x - top.masked_fill(top == -math.inf, 0.0)).exp()
            l = p.sum(-1, keepdim=True)
            p = p / l.masked_fill(l == 0, 1.0)
            vv = torch.where(p.amax(0)[:, None] > 0, v, torch.zeros_like(v))  # (0 * NaN of a hidden key)
            y = p @ vv
            worst = (2 * err + 2.0 ** -22 * (x - top).abs().nan_to_num(0, 0, 0).clamp(max=1e4)).amax(-1, keepdim=True) if x.shape[1] else 0.0
            worst = torch.as_tensor(worst)
            out[cu[r]:cu[r + 1], h] = y
            rounding = 2.0 ** -11 if n < 32 else torch.finfo(query.dtype).eps / 2
            tol[cu[r]:cu[r + 1], h] = ((rounding + 2 * worst.expm1()) * (p @ vv.abs()) + torch.finfo(query.dtype).eps / 2 * y.abs() +
                                       2.0 ** -30 * vv.abs().amax().item() if v.numel() else 0.0)
    return out, tol + torch.finfo(query.dtype).tiny


def check(got, want, tol):
    assert torch.equal(got.isnan(), want.isnan())
    ratio = ((got.double() - want).abs() / tol).nan_to_num(0.0)
    assert ratio.max().item() <= 1.0, ratio.max().item()


ATTEND = [  # cached, new, heads, kv heads, head dim, block size
    ([0], [1], 1, 1, 64, 16), ([4096], [1], 8, 2, 128, 64), ([1000, 0, 63, 64, 4099], [1] * 5, 8, 8, 128, 16),
    ([130, 3], [1, 1], 32, 2, 96, 32), ([500, 777], [1, 1], 20, 1, 256, 128), ([127, 129, 90], [1, 5, 3], 8, 2, 64, 64),
    ([700, 0, 12], [5, 9, 1], 12, 4, 128, 16), ([300], [40], 6, 2, 128, 64), ([65, 40], [33, 0], 2, 1, 256, 32), ([0, 10], [130, 70], 4, 4, 64, 128),
    ([40] * 300, [1] * 300, 2, 1, 16, 16), ([0, 500, 31, 7, 900], [31, 32, 1, 300, 65], 8, 2, 128, 16), ([1000, 64], [257, 2], 4, 1, 64, 32),
    ([20] * 140, [1, 40] * 70, 4, 2, 64, 16), ([33] * 200, [2, 30, 1, 5] * 50, 4, 4, 32, 16), ([100, 0], [33, 31], 32, 4, 64, 16),
    ([50] * 100, [31] * 99 + [45], 2, 1, 16, 32), ([9] * 150, [31] * 149 + [40], 4, 4, 16, 16), ([300, 64], [128, 129], 3, 1, 96, 64), ([2000, 100], [2, 1], 9, 3, 80, 64), ([513, 60], [1, 7], 4, 2, 192, 64), ([5000], [1], 4, 4, 48, 128)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cached,new,H,Hk,d,bs", ATTEND)
def test_attention(dev, dtype, cached, new, H, Hk, d, bs):
    tables, cache, step, g = filled(dev, len(cached), cached, new, Hk, d, bs, 6)
    T = sum(new)
    kv = torch.randn((2, T, Hk, d), generator=g, device=dev).to(dtype)
    fsa.cache_append(cache, tables, step, kv[0], kv[1])
    q = torch.randn((T, H, d), generator=g, device=dev).to(dtype)
    want = attend(q, cache, tables, step)
    check(fsa.flash_sparse_attn_cache_func(q, cache, tables, step), *want)
    got = fsa.flash_sparse_attn_cache_func(q, cache, tables, step, max_seqlen_q=max(new), max_seqlen_k=max(step.lengths.tolist()))
    check(got, *want)
    check(fsa.flash_sparse_attn_cache_func(q, cache, tables, step, is_causal=False, softmax_scale=0.3, max_seqlen_q=max(new)),
          *attend(q, cache, tables, step, scale=0.3, causal=False))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bias_heads", ["one", "kv", "all"])
@pytest.mark.parametrize("cached,new,H,Hk,d,bs", [([500, 70, 0], [1, 1, 1], 8, 2, 128, 16), ([300, 90], [3, 6], 12, 4, 64, 64),
                                                 ([200, 333], [1, 20], 16, 4, 256, 32)])
def test_attention_with_bias_and_kept_keys(dev, dtype, bias_heads, cached, new, H, Hk, d, bs):
    from flash_sparse_attn.utils.mask import create_kept_keys, create_mask

    R, keys = len(cached), 600
    tables, cache, step, g = filled(dev, R, cached, new, Hk, d, bs, 7)
    T = sum(new)
    kv = torch.randn((2, T, Hk, d), generator=g, device=dev).to(dtype)
    fsa.cache_append(cache, tables, step, kv[0], kv[1])
    q = torch.randn((T, H, d), generator=g, device=dev).to(dtype)
    bias = torch.randn((R, {"one": 1, "kv": Hk, "all": H}[bias_heads], 1, keys), generator=g, device=dev).to(dtype)
    args = dict(attn_bias=bias, max_seqlen_q=max(new))
    check(fsa.flash_sparse_attn_cache_func(q, cache, tables, step, **args), *attend(q, cache, tables, step, bias=bias))
    short = bias[:1, :, :, :77]
    check(fsa.flash_sparse_attn_cache_func(q, cache, tables, step, attn_bias=short), *attend(q, cache, tables, step, bias=short))
    rows = torch.randn((R, Hk, 1, keys), generator=g, device=dev).to(dtype)
    valid = torch.arange(keys, device=dev)[None] < step.lengths[:, None]
    kept = create_kept_keys(rows, valid, R, 1, keys, 90, torch.finfo(dtype).min)
    check(fsa.flash_sparse_attn_cache_func(q, cache, tables, step, attn_mask=kept, **args), *attend(q, cache, tables, step, kept, bias))
    check(fsa.flash_sparse_attn_cache_func(q, cache, tables, step, attn_mask=kept), *attend(q, cache, tables, step, kept))
    mask = create_mask(rows, valid, R, 1, keys, 90, torch.finfo(dtype).min)
    got = fsa.flash_sparse_attn_cache_func(q, cache, tables, step, attn_mask=mask, **args)
    check(got, *attend(q, cache, tables, step, kept, bias))
    del mask._fdma_kept  # a mask of the caller's own
    assert torch.equal(fsa.flash_sparse_attn_cache_func(q, cache, tables, step, attn_mask=mask, **args), got)
    shared = fsa.KeptKeys(kept.key_pos[:1, :1].contiguous(), kept.count[:1, :1].contiguous(), kept.slot_mask[:1, :1], keys)
    check(fsa.flash_sparse_attn_cache_func(q, cache, tables, step, attn_mask=shared, **args), *attend(q, cache, tables, step, shared, bias))


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_masked_rows(dev, dtype, kept):
    """Biases of -inf and of the type's lowest number: a row of nothing but -inf is 0, one of nothing but the lowest an average."""
    cached, H, Hk, d = [200, 130, 64], 4, 2, 64
    tables, cache, step, g = filled(dev, 3, cached, [1, 1, 1], Hk, d, 32, 8)
    kv = torch.randn((2, 3, Hk, d), generator=g, device=dev).to(dtype)
    fsa.cache_append(cache, tables, step, kv[0], kv[1])
    q = torch.randn((3, H, d), generator=g, device=dev).to(dtype)
    bias = torch.zeros((3, Hk, 1, 256), device=dev, dtype=dtype)
    bias[0] = -math.inf
    bias[0, 1, 0, 100] = 0
    bias[1] = torch.finfo(dtype).min
    bias[2, 0, 0, ::2] = -math.inf
    bias[2, 1, 0, 1::2] = torch.finfo(dtype).min
    keep = None
    if kept:
        pos = torch.arange(256, dtype=torch.int32, device=dev).expand(3, Hk, 256).contiguous()
        count = ints([[256, 256], [40, 0], [65, 3]], dev)
        keep = fsa.KeptKeys(pos, count, pos[:, :, None] < count[..., None, None], 256)
    got = fsa.flash_sparse_attn_cache_func(q, cache, tables, step, attn_mask=keep, attn_bias=bias, max_seqlen_q=1)
    check(got, *attend(q, cache, tables, step, keep, bias))
    assert not bool(got[0, :2].any()) and bool(got[0, 2:].any())
    if kept:
        assert not bool(got[1, 2:].any())


def test_not_a_number_stays_in_its_request(dev):
    tables, cache, step, g = filled(dev, 3, [70, 90, 66], [1, 2, 1], 2, 128, 64, 9)
    kv = torch.randn((2, 4, 2, 128), generator=g, device=dev, dtype=torch.bfloat16)
    fsa.cache_append(cache, tables, step, kv[0], kv[1])
    q = torch.randn((4, 4, 128), generator=g, device=dev, dtype=torch.bfloat16)
    want = fsa.flash_sparse_attn_cache_func(q, cache, tables, step)
    cache.v.view(torch.uint8)[tables.table[1, 0].item(), 0, 5, 7] = 0x7F
    cache.k.view(torch.uint8)[tables.table[2, 0].item(), 1, 9, 3] = 0x7F
    got = fsa.flash_sparse_attn_cache_func(q, cache, tables, step)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1:3, 2:], want[1:3, 2:]) and torch.equal(got[3, :2], want[3, :2])
    assert bool(got[1:3, :2, 7].isnan().all()) and bool(got[3, 2:].isnan().all())
    others = [i for i in range(128) if i != 7]
    assert torch.equal(got[1:3, :2, others], want[1:3, :2, others])


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("H,n,d,bs", [(2, 3, 64, 16), (8, 6, 128, 64), (16, 5, 256, 32)])
def test_not_a_number_is_not_seen_through_a_mask(dev, kept, H, n, d, bs):
    """Values and keys that are NaN at a later token of a draft, or behind a bias of -inf, leave the queries that do not see them as
    they are; those that do become NaN."""
    tables, cache, step, g = filled(dev, 2, [100, 61], [n, n], 2, d, bs, 19)
    kv = torch.randn((2, 2 * n, 2, d), generator=g, device=dev, dtype=torch.bfloat16)
    fsa.cache_append(cache, tables, step, kv[0], kv[1])
    q = torch.randn((2 * n, H, d), generator=g, device=dev, dtype=torch.bfloat16)
    bias = torch.zeros((2, 2, 1, 128), device=dev, dtype=torch.bfloat16)
    bias[0, :, :, 40:60] = -math.inf
    keep = None
    if kept:
        keep = fsa.KeptKeys(torch.arange(128, dtype=torch.int32, device=dev).expand(2, 2, 128).contiguous(), ints([[128, 128]] * 2, dev), None, 128)
    args = dict(attn_mask=keep, attn_bias=bias, max_seqlen_q=n)
    want = fsa.flash_sparse_attn_cache_func(q, cache, tables, step, **args)
    at = step.slots[[n - 1, 2 * n - 2]].tolist()  # the last token of one request, the last but one of the other
    for slot, x in zip(at, (cache.v, cache.k)):
        x.view(torch.uint8)[slot // bs, 0, slot % bs, 5] = 0xFF
    hidden = tables.table[0, 40 // bs:60 // bs + 1].tolist()
    for pos in range(40, 60):
        cache.v.view(torch.uint8)[hidden[pos // bs - 40 // bs], :, pos % bs] = 0x7F
    got = fsa.flash_sparse_attn_cache_func(q, cache, tables, step, **args)
    G = H // 2
    assert torch.equal(got[:n - 1], want[:n - 1]) and torch.equal(got[n:2 * n - 2], want[n:2 * n - 2])
    assert torch.equal(got[n - 1, G:], want[n - 1, G:]) and torch.equal(got[2 * n - 2:, G:], want[2 * n - 2:, G:])
    assert bool(got[n - 1, :G, 5].isnan().all()) and bool(got[2 * n - 2:, :G].isnan().all())


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("heads", [1, 2, 4])
def test_not_a_number_in_a_key_is_not_seen_through_a_bias(dev, kept, heads):
    tables, cache, step, g = filled(dev, 2, [100, 61], [1, 1], 2, 64, 16, 23)
    kv = torch.randn((2, 2, 2, 64), generator=g, device=dev, dtype=torch.bfloat16)
    fsa.cache_append(cache, tables, step, kv[0], kv[1])
    q = torch.randn((2, 4, 64), generator=g, device=dev, dtype=torch.bfloat16)
    bias = torch.randn((2, heads, 1, 128), generator=g, device=dev, dtype=torch.bfloat16)
    bias[:, :, :, 16:48] = -math.inf
    keep = None
    if kept:
        keep = fsa.KeptKeys(torch.arange(128, dtype=torch.int32, device=dev).expand(2, 2, 128).contiguous(), ints([[128, 128]] * 2, dev), None, 128)
    want = fsa.flash_sparse_attn_cache_func(q, cache, tables, step, keep, bias)
    for block in tables.table[:, 1:3].flatten().tolist():
        cache.k.view(torch.uint8)[block] = 0x7F
        cache.v.view(torch.uint8)[block] = 0xFF
    got = fsa.flash_sparse_attn_cache_func(q, cache, tables, step, keep, bias)
    assert bool(want.isfinite().all()) and torch.equal(got, want)


@pytest.mark.parametrize("bound", [0, 1])
def test_a_bound_of_no_tokens_is_one_of_one(dev, bound):
    """More requests than a CTA holds, and more heads per kv head than a tile has rows."""
    requests, H, d = 130, 16, 64
    tables, cache, step, g = filled(dev, requests, [(37 * r) % 150 for r in range(requests)], [1] * requests, 1, d, 16, 24)
    kv = torch.randn((2, requests, 1, d), generator=g, device=dev, dtype=torch.float16)
    fsa.cache_append(cache, tables, step, kv[0], kv[1])
    q = torch.randn((requests, H, d), generator=g, device=dev, dtype=torch.float16)
    check(fsa.flash_sparse_attn_cache_func(q, cache, tables, step, max_seqlen_q=bound), *attend(q, cache, tables, step))


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("lengths,d,bs", [([1, 17, 100], 48, 16), ([3, 129, 64], 128, 64), ([33, 40, 65], 256, 128)])
def test_what_was_in_a_block_before_does_not_matter(dev, kept, lengths, d, bs):
    tables = fsa.block_tables(3, 9, 30, bs, device=dev)
    cache = fsa.quantized_cache(30, 2, d, bs, device=dev)
    for x, byte in ((cache.k, 0x7F), (cache.v, 0xFF)):
        x.view(torch.uint8).fill_(byte)
    cache.k_scale.fill_(math.nan)
    cache.v_scale.fill_(math.nan)
    g = torch.Generator(device=dev).manual_seed(26)
    for new in (lengths, [2, 1, 3]):
        T = sum(new)
        step = tables.extend(ints(new, dev), T)
        kv = torch.randn((2, T, 2, d), generator=g, device=dev, dtype=torch.float16)
        fsa.cache_append(cache, tables, step, kv[0], kv[1])
        q = torch.randn((T, 4, d), generator=g, device=dev, dtype=torch.float16)
        keep = None
        if kept:
            keep = fsa.KeptKeys(torch.arange(0, 256, 2, dtype=torch.int32, device=dev).expand(3, 2, 128).contiguous(), ints([[128, 90]] * 3, dev), None, 256)
        check(fsa.flash_sparse_attn_cache_func(q, cache, tables, step, keep), *attend(q, cache, tables, step, keep))


def widen(tables):
    """The same requests with rows for 40000 tokens: the work is then split for long requests, whatever their lengths are."""
    more = 40000 // tables.block_size - tables.table.shape[1]
    return tables._replace(table=torch.nn.functional.pad(tables.table, (0, more), value=-1))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cached,new,H,Hk,d,bs", ATTEND)
def test_attention_under_wide_bounds(dev, dtype, cached, new, H, Hk, d, bs):
    tables, cache, step, g = filled(dev, len(cached), cached, new, Hk, d, bs, 27)
    T = sum(new)
    kv = torch.randn((2, T, Hk, d), generator=g, device=dev).to(dtype)
    fsa.cache_append(cache, tables, step, kv[0], kv[1])
    q = torch.randn((T, H, d), generator=g, device=dev).to(dtype)
    tables = widen(tables)
    check(fsa.flash_sparse_attn_cache_func(q, cache, tables, step), *attend(q, cache, tables, step))
    most = max(step.lengths.tolist())
    pos = torch.arange(40000, dtype=torch.int32, device=dev) * 2
    kept = fsa.KeptKeys(pos.expand(1, Hk, -1).contiguous(), torch.full((1, Hk), most // 2, dtype=torch.int32, device=dev), None, 80000)
    bias = torch.randn((1, H, 1, most), generator=g, device=dev).to(dtype)
    check(fsa.flash_sparse_attn_cache_func(q, cache, tables, step, kept, bias, max_seqlen_q=max(new)), *attend(q, cache, tables, step, kept, bias))


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("requests,length,Hk", [(1, 1, 1), (1, 70, 2), (2, 200, 1), (1, 1200, 1), (1, 20000, 1), (3, 5000, 8), (40, 600, 1),
                                                (100, 130, 1), (210, 100, 1), (300, 100, 1)])
def test_shared_units(dev, kept, requests, length, Hk):
    """Units of one to sixteen CTAs and more, requests of one token and of the full length, refused ones, and tokens behind the last."""
    d, bs = 64, 64
    lengths = [1 + (length - 1) * (i % 3) // 2 for i in range(requests)]
    lengths[-1] = length
    tables, cache, _, g = filled(dev, requests, [n - 1 for n in lengths], [1] * requests, Hk, d, bs, 28)
    tables.truncate(ints([n - 1 for n in lengths], dev))
    new = [1] * requests
    if requests > 1:
        new[0] = tables.table.shape[1] * bs + 1  # is refused
    T = sum(new) + 3
    step = tables.extend(ints(new, dev), T)
    assert step.granted.tolist() == [n == 1 for n in new]
    kv = torch.randn((2, T, Hk, d), generator=g, device=dev, dtype=torch.bfloat16)
    fsa.cache_append(cache, tables, step, kv[0], kv[1])
    q = torch.randn((T, 4 * Hk, d), generator=g, device=dev, dtype=torch.bfloat16)
    keep = None
    if kept:
        n = (length + 2) // 3
        count = torch.randint(0, n + 1, (requests, Hk), generator=g, device=dev, dtype=torch.int32)
        keep = fsa.KeptKeys((3 * torch.arange(n, dtype=torch.int32, device=dev)).expand(requests, Hk, n).contiguous(), count, None, 3 * n)
    out = fsa.flash_sparse_attn_cache_func(q, cache, tables, step, keep, max_seqlen_q=1, max_seqlen_k=length)
    check(out, *attend(q, cache, tables, step, keep))
    assert not out[-3:].any() and (requests == 1 or not out[:new[0]].any())


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("wide", [False, True])
def test_not_a_number_in_every_key(dev, kept, wide):
    """Scores that are all NaN are larger than no maximum; the result is NaN all the same, and only there."""
    tables, cache, step, g = filled(dev, 3, [300, 90, 500], [1, 3, 2], 2, 128, 32, 29)
    kv = torch.randn((2, 6, 2, 128), generator=g, device=dev, dtype=torch.bfloat16)
    fsa.cache_append(cache, tables, step, kv[0], kv[1])
    q = torch.randn((6, 8, 128), generator=g, device=dev, dtype=torch.bfloat16)
    keep = None
    if kept:
        keep = fsa.KeptKeys(torch.arange(512, dtype=torch.int32, device=dev).expand(1, 1, 512).contiguous(), ints([[512]], dev), None, 512)
    if wide:
        tables = widen(tables)
        if kept:
            keep = keep._replace(key_pos=torch.nn.functional.pad(keep.key_pos, (0, 40000)))
    want = fsa.flash_sparse_attn_cache_func(q, cache, tables, step, keep)
    cache.k.view(torch.uint8)[tables.table[1, :3].long(), 1] = 0x7F
    got = fsa.flash_sparse_attn_cache_func(q, cache, tables, step, keep)
    assert bool(got[1:4, 4:].isnan().all())
    assert torch.equal(got[1:4, :4], want[1:4, :4]) and torch.equal(got[[0, 4, 5]], want[[0, 4, 5]])


def test_refused_and_padded_tokens_are_zero(dev):
    tables = fsa.block_tables(4, 3, 4, 16, device=dev)
    cache = fsa.quantized_cache(4, 1, 64, 16, device=dev)
    step = tables.extend(ints([20, 33, 0, 4], dev), 70)  # the second needs three blocks of the two that are left; none behind it gets any
    assert step.granted.tolist() == [True, False, True, False]
    x = torch.randn((70, 1, 64), device=dev, dtype=torch.bfloat16)
    fsa.cache_append(cache, tables, step, x, x)
    for kept in (None, fsa.KeptKeys(torch.arange(128, dtype=torch.int32, device=dev).expand(4, 1, 128).contiguous(), ints([[128]] * 4, dev), None, 128)):
        for bound in (None, 33, 20):
            got = fsa.flash_sparse_attn_cache_func(x, cache, tables, step, attn_mask=kept, max_seqlen_q=bound)
            want, tol = attend(x, cache, tables, step, kept)
            check(got, want, tol)
            assert not bool(got[20:].any())
    assert not bool(fsa.flash_sparse_attn_cache_func(x, cache, tables, step, max_seqlen_q=3)[3:20].any())


@pytest.mark.parametrize("scale", [2.0 ** -90, 2.0 ** -20, 2.0 ** 60])
def test_scales_far_apart(dev, scale):
    """Blocks whose values differ by many powers of two: the larger ones rule the output, the smaller ones the sum where their scores
    are as high."""
    tables, cache, step, g = filled(dev, 1, [300], [1], 1, 64, 16, 10)
    kv = torch.randn((2, 1, 1, 64), generator=g, device=dev, dtype=torch.bfloat16)
    fsa.cache_append(cache, tables, step, kv[0], kv[1])
    cache.v_scale[tables.table[0, ::2].long()] *= scale
    q = torch.randn((1, 2, 64), generator=g, device=dev, dtype=torch.bfloat16)
    check(fsa.flash_sparse_attn_cache_func(q, cache, tables, step), *attend(q, cache, tables, step))
    cache.v_scale.mul_(scale)
    check(fsa.flash_sparse_attn_cache_func(q, cache, tables, step), *attend(q, cache, tables, step))


@pytest.mark.parametrize("size", [2.0 ** -60, 2.0 ** 60])
def test_queries_of_any_size(dev, size):
    """bf16 queries go through fp16 by a power of two per row."""
    tables, cache, step, g = filled(dev, 1, [100], [1], 2, 128, 64, 11)
    kv = torch.randn((2, 1, 2, 128), generator=g, device=dev, dtype=torch.bfloat16)
    fsa.cache_append(cache, tables, step, kv[0], kv[1])
    q = (torch.randn((1, 4, 128), generator=g, device=dev) * size).to(torch.bfloat16)
    args = dict(scale=128 ** -0.5 / size)
    check(fsa.flash_sparse_attn_cache_func(q, cache, tables, step, softmax_scale=args["scale"]), *attend(q, cache, tables, step, **args))


def test_query_layouts(dev):
    tables, cache, step, g = filled(dev, 2, [90, 20], [1, 3], 2, 64, 16, 12)
    fused = torch.randn((4, 8, 64), generator=g, device=dev, dtype=torch.float16)
    fsa.cache_append(cache, tables, step, fused[:, 4:6], fused[:, 6:])
    want = fsa.flash_sparse_attn_cache_func(fused[:, :4].contiguous(), cache, tables, step)
    assert torch.equal(fsa.flash_sparse_attn_cache_func(fused[:, :4], cache, tables, step), want)
    odd = torch.empty(4 * 4 * 64 + 1, device=dev, dtype=torch.float16)[1:].view(4, 4, 64).copy_(fused[:, :4])
    assert torch.equal(fsa.flash_sparse_attn_cache_func(odd, cache, tables, step), want)
    strided = fused[:, :4].transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(fsa.flash_sparse_attn_cache_func(strided, cache, tables, step), want)


def test_no_tokens(dev):
    tables, cache, step, g = filled(dev, 2, [90, 20], [0, 0], 2, 64, 16, 12)
    x = torch.empty((0, 2, 64), device=dev, dtype=torch.bfloat16)
    assert fsa.cache_append(cache, tables, step, x, x) is None
    assert fsa.flash_sparse_attn_cache_func(x, cache, tables, step).shape == (0, 2, 64)


def test_attention_refusals(dev):
    tables, cache, step, g = filled(dev, 2, [20, 5], [1, 1], 2, 64, 16, 13)
    q = torch.zeros((2, 4, 64), device=dev, dtype=torch.bfloat16)
    k = q[:, :2]
    kept = fsa.KeptKeys(torch.zeros((2, 2, 128), dtype=torch.int32, device=dev), ints([[1, 1]] * 2, dev), None, 21)
    for args in [(q.cpu(), cache, tables, step), (q.float(), cache, tables, step), (q[:1], cache, tables, step), (q[:, :3], cache, tables, step),
                 (q[..., :32], cache, tables, step), (q[None], cache, tables, step), (q, cache._replace(k=cache.k.view(torch.uint8)), tables, step),
                 (q, cache._replace(v=cache.v[:, :1]), tables, step), (q, cache._replace(k_scale=cache.k_scale.half()), tables, step),
                 (q, cache, tables._replace(block_size=32), step), (q, cache, tables, step._replace(lengths=step.lengths.long())),
                 (q, cache, tables, step._replace(cu_chunks=step.cu_chunks[:2])), (q, cache, tables._replace(table=tables.table[:1]), step),
                 (q.clone().requires_grad_(True), cache, tables, step)]:
        with pytest.raises(RuntimeError):
            fsa.flash_sparse_attn_cache_func(*args)
    bias = torch.zeros((2, 2, 1, 30), device=dev, dtype=torch.bfloat16)
    for kw in [dict(attn_bias=bias.float()), dict(attn_bias=bias[0]), dict(attn_bias=bias.expand(2, 2, 2, 30)), dict(attn_bias=bias[:, :, :, :0]),
               dict(attn_bias=torch.zeros((3, 2, 1, 30), device=dev, dtype=torch.bfloat16)), dict(attn_bias=bias.cpu()),
               dict(attn_bias=bias.clone().requires_grad_(True)),
               dict(attn_mask=kept._replace(key_pos=kept.key_pos.long())), dict(attn_mask=kept._replace(count=kept.count[:1])),
               dict(attn_mask=kept._replace(key_pos=torch.zeros((3, 2, 128), dtype=torch.int32, device=dev))),
               dict(attn_mask=bias), dict(attn_mask=torch.ones((2, 2, 2, 30), dtype=torch.bool, device=dev)), dict(max_seqlen_q=-1)]:
        with pytest.raises(RuntimeError):
            fsa.flash_sparse_attn_cache_func(q, cache, tables, step, **kw)
    f = fsa.rotary_frequencies(64, device=dev)
    for args in [(k, k[:1]), (k.float(), k.float()), (k, k.half()), (k[:, :1], k[:, :1]), (k.cpu(), k.cpu()), (k, k, q), (k, k, q[:1], f),
                 (k, k, q.half(), f), (k, k, q, fsa.rotary_frequencies(66, device=dev)), (k, k, q, fsa.rotary_frequencies(64, device="cpu")),
                 (k.clone().requires_grad_(True), k)]:
        with pytest.raises(RuntimeError):
            fsa.cache_append(cache, tables, step, *args)


# ---- all of it, as it is used ------------------------------------------------------------------------------------------
def serving_step(state, x, new):
    """One step of a model with one layer; x: its fused projection."""
    cache, tables, f, H, Hk = state
    step = tables.extend(new, x.shape[0])
    q = fsa.cache_append(cache, tables, step, x[:, H:H + Hk], x[:, H + Hk:], query=x[:, :H], frequencies=f)
    return step, q, fsa.flash_sparse_attn_cache_func(q, cache, tables, step, max_seqlen_q=x.shape[0])


def test_serving_matches_attention_without_a_cache(dev):
    """Prompts, then tokens one by one, then a draft of which part is rejected: every output equals attention in 64 bits over the
    turned keys and values, to within what eight bits hold: 2^-4 of each key and value (a block's scale may grow once more: 2^-3)."""
    H, Hk, d, R, dtype = 4, 2, 64, 3, torch.bfloat16
    g = torch.Generator(device=dev).manual_seed(14)
    f, inv = fsa.rotary_frequencies(d, device=dev), inv_freq(d, dev)
    tables, cache = fsa.block_tables(R, 8, 24, 16, device=dev), fsa.quantized_cache(24, Hk, d, 16, device=dev)
    state = (cache, tables, f, H, Hk)
    seen = [torch.empty((0, H + 2 * Hk, d), device=dev, dtype=dtype) for _ in range(R)]
    plan = [[30, 0, 17], [1, 9, 1], [1, 1, 1], [1, 0, 1], [4, 4, 4]]
    for i, new in enumerate(plan + [[1, 1, 1]]):
        x = torch.randn((sum(new) + i % 2, H + 2 * Hk, d), generator=g, device=dev).to(dtype)
        step, q, out = serving_step(state, x, ints(new, dev))
        at = 0
        for r, n in enumerate(new):
            seen[r] = torch.cat((seen[r], x[at:at + n]))
            pos = torch.arange(seen[r].shape[0], device=dev)
            turned, _ = turn(seen[r][:, :H + Hk], pos, inv)
            for h in range(H):
                hk = h // (H // Hk)
                k, v, qq = turned[:, H + hk], seen[r][:, H + Hk + hk].double(), turned[-n:, h] if n else turned[:0, h]
                s = d ** -0.5 * qq @ k.T
                slack = 2 * d ** -0.5 * (2.0 ** -3 + 2.0 ** -8) * (qq.abs() @ k.abs().T).amax() if n else 0.0
                hide = pos[None] > pos[-n:, None] if n else torch.zeros((0, pos.numel()), dtype=torch.bool, device=dev)
                p = s.masked_fill(hide, -math.inf).softmax(-1)
                got = out[at:at + n, h].double()
                if n:
                    tol = (2.0 ** -3 + 2.0 ** -7) * (p @ v.abs()) + (math.exp(float(slack)) - 1) * (p @ v.abs()) + 2.0 ** -8 * v.abs().amax()
                    assert bool(((got - p @ v).abs() <= tol).all())
            at += n
        check(out, *attend(q, cache, tables, step))
        if new == [4, 4, 4]:
            keep = [tables.lengths[0].item() - 1, tables.lengths[1].item() - 4, tables.lengths[2].item()]
            tables.truncate(ints(keep, dev))
            seen = [t[:n] for t, n in zip(seen, keep)]
    tables.truncate(ints([0, 0, 0], dev))
    assert tables.free_count.item() == 24


def test_captured_steps(dev):
    """A whole step in a CUDA graph, replayed with other activations and lengths, equals the eager steps."""
    H, Hk, d, dtype = 8, 2, 128, torch.bfloat16
    f = fsa.rotary_frequencies(d, device=dev)
    g = torch.Generator(device=dev).manual_seed(15)
    xs = [torch.randn((6, H + 2 * Hk, d), generator=g, device=dev).to(dtype) for _ in range(6)]
    news = [ints(n, dev) for n in ([3, 1, 2], [1, 1, 1], [0, 4, 2], [2, 0, 0], [1, 5, 0], [1, 1, 4])]

    def fresh():
        return fsa.quantized_cache(12, Hk, d, 16, device=dev), fsa.block_tables(3, 4, 12, 16, device=dev), f, H, Hk

    eager = fresh()
    want = [serving_step(eager, x, n)[2].clone() for x, n in zip(xs, news)]
    state, x, new = fresh(), xs[0].clone(), news[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        serving_step(fresh(), x, new)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = serving_step(state, x, new)[2]
    for i in range(6):
        x.copy_(xs[i]), new.copy_(news[i])
        graph.replay()
        assert torch.equal(out, want[i]), i
    assert torch.equal(state[1].table, eager[1].table) and torch.equal(state[0].k.float(), eager[0].k.float())


def test_two_graphs_and_two_streams(dev):
    """Two calls at once have scratch of their own."""
    calls = []
    for seed in (16, 17):
        tables, cache, step, g = filled(dev, 2, [3000, 2000], [1, 1], 2, 128, 64, seed)
        x = torch.randn((2, 2, 128), generator=g, device=dev, dtype=torch.bfloat16)
        fsa.cache_append(cache, tables, step, x, x)
        q = torch.randn((2, 8, 128), generator=g, device=dev, dtype=torch.bfloat16)
        calls.append((q, cache, tables, step))
    want = [fsa.flash_sparse_attn_cache_func(*c, max_seqlen_q=1) for c in calls]
    torch.cuda.synchronize()
    streams, graphs, outs = [torch.cuda.Stream() for _ in calls], [], []
    for c, s in zip(calls, streams):
        with torch.cuda.stream(s):
            fsa.flash_sparse_attn_cache_func(*c, max_seqlen_q=1)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(fsa.flash_sparse_attn_cache_func(*c, max_seqlen_q=1))
        graphs.append(graph)
    for _ in range(20):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(outs, want):
        assert torch.equal(a, b)
    for _ in range(20):
        got = []
        for c, s in zip(calls, streams):
            with torch.cuda.stream(s):
                got.append(fsa.flash_sparse_attn_cache_func(*c, max_seqlen_q=1))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_repeated_calls_are_equal(dev):
    tables, cache, step, g = filled(dev, 4, [5000, 1, 700, 64], [1] * 4, 2, 64, 16, 18)
    x = torch.randn((4, 2, 64), generator=g, device=dev, dtype=torch.float16)
    fsa.cache_append(cache, tables, step, x, x)
    q = torch.randn((4, 16, 64), generator=g, device=dev, dtype=torch.float16)
    first = fsa.flash_sparse_attn_cache_func(q, cache, tables, step)
    for _ in range(10):
        assert torch.equal(fsa.flash_sparse_attn_cache_func(q, cache, tables, step), first)


def test_inference_mode(dev):
    with torch.inference_mode():
        cache, tables = fsa.quantized_cache(4, 1, 64, 16, device=dev), fsa.block_tables(1, 4, 4, 16, device=dev)
        x = torch.randn((5, 1, 64), device=dev, dtype=torch.bfloat16)
        step = tables.extend(ints([5], dev), 5)
        fsa.cache_append(cache, tables, step, x, x)
        check(fsa.flash_sparse_attn_cache_func(x, cache, tables, step), *attend(x, cache, tables, step))
        tables.truncate(ints([0], dev))
    assert tables.free_count.item() == 4


def test_bool_masks_in_inference_mode(dev):
    from flash_sparse_attn.utils.mask import create_kept_keys, create_mask

    tables, cache, step, g = filled(dev, 2, [90, 40], [1, 1], 2, 64, 16, 25)
    x = torch.randn((2, 4, 64), generator=g, device=dev, dtype=torch.bfloat16)
    bias = torch.randn((2, 2, 1, 96), generator=g, device=dev, dtype=torch.bfloat16)
    low = torch.finfo(bias.dtype).min
    mask = create_mask(bias, None, 2, 1, 96, 32, low)
    with torch.inference_mode():
        kept = create_kept_keys(bias, None, 2, 1, 96, 32, low)
        fsa.cache_append(cache, tables, step, x[:, :2], x[:, 2:])
        got = [fsa.flash_sparse_attn_cache_func(x, cache, tables, step, m, bias) for m in (kept, mask, mask & True)]
        check(got[0], *attend(x, cache, tables, step, kept, bias))
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


def test_compiled_step(dev):
    H, Hk, d = 4, 2, 64
    f = fsa.rotary_frequencies(d, device=dev)
    x = torch.randn((5, H + 2 * Hk, d), device=dev, dtype=torch.bfloat16)
    new = ints([3, 2], dev)

    def fresh():
        return fsa.quantized_cache(4, Hk, d, 16, device=dev), fsa.block_tables(2, 2, 4, 16, device=dev)

    def fn(x, new, k, v, ks, vs, table, lengths, free, count, ticket):
        tables = fsa.BlockTables(table, lengths, free, count, ticket, 16)
        step, q, out = serving_step((fsa.QuantizedCache(k, v, ks, vs), tables, f, H, Hk), x, new)
        tables.truncate(new - 1)
        return out

    a, b = fresh(), fresh()
    want = fn(x, new, *a[0], *a[1][:5])
    got = torch.compile(fn, backend="aot_eager", fullgraph=True)(x, new, *b[0], *b[1][:5])
    assert torch.equal(got, want)
    for s, t in zip((*a[0], *a[1][:5]), (*b[0], *b[1][:5])):
        assert torch.equal(s.float(), t.float())
