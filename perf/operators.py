"""The operators around attention that a model needs to be trained on long contexts and served from a cache: rotary positions,
block tables and slot maps, the 8-bit cache's writer, and attention over that cache. Each case is a dict of plain values:

  op        "rotary"  apply_rotary; train: with the gradients        "tables"  BlockTables.extend, then .truncate back
            "append"  cache_append, queries rotated beside           "attend"  flash_sparse_attn_cache_func
  heads, kv_heads, head_dim, dtype; block_size (tokens of a block)
  batch, seqlen, rotary_dim, interleaved, scaling, factor, offset (first position)                         rotary
  requests, cached, new, mixed   requests with up to `cached` tokens in the cache and up to `new` more; mixed: of all lengths, else
            all with the most; requests draw theirs from the seed of the case, so that states of one case have the same sizes
  kept      attend: 0, or the kept keys of each (request, kv head), with a bias for each key

`run` computes the same in its plain form and through the framework.
"""
import math
import os
import random
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_E4M3 = torch.float8_e4m3fn
_CHUNK = 64      # tokens of a unit of attention's work
_BASE = 500000.0  # rotary base
_ORIGINAL = 4096  # context that a scaled model was trained at

# (query heads, kv heads): multi-query, grouped and plain multi-head layouts
_HEADS = ((2, 1), (8, 2), (8, 8), (12, 4), (16, 4), (16, 1), (32, 8))


def _package():
    path = os.path.join(os.getcwd(), "flash-dmattn_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import flash_sparse_attn

    return flash_sparse_attn


def _rotary(batch, seqlen, heads, head_dim, dtype="bf16", rotary_dim=0, interleaved=False, scaling="none", offset=0,
            train=True, name=None):
    c = {} if name is None else {"name": name}
    c.update(op="rotary", batch=batch, seqlen=seqlen, heads=heads[0], kv_heads=heads[1], head_dim=head_dim, dtype=dtype,
             rotary_dim=rotary_dim or head_dim, interleaved=interleaved, scaling=scaling, factor=8.0, offset=offset, train=train)
    return c


def _cached(op, requests, cached, new, heads, head_dim, dtype="bf16", block_size=64, mixed=True, kept=0, sizes=1, name=None):
    c = {} if name is None else {"name": name}
    c.update(op=op, requests=requests, cached=cached, new=new, heads=heads[0], kv_heads=heads[1], head_dim=head_dim, dtype=dtype,
             block_size=block_size, mixed=mixed, kept=kept, sizes=sizes)
    return c


def listed():
    return [
        # One token of one sequence in a small model: the smallest call there is.
        _rotary(1, 1, (2, 1), 64, "fp16", interleaved=True, offset=4095, train=False, name="rotary_one_token"),
        # A training step's layer at the usual context: forward and backward.
        _rotary(2, 4096, (32, 8), 128, name="rotary_train_4k"),
        # One very long sequence, wide heads of which half are rotated, scaled beyond the trained context; an odd length.
        _rotary(1, 65537, (16, 1), 256, rotary_dim=128, scaling="yarn", name="rotary_long_partial"),
        # Serving, token phase: every request takes one token, some a new block.
        _cached("tables", 256, 65536, 1, (1, 1), 64, name="tables_decode_256"),
        # Serving, prompt phase: requests with prompts of any length enter together.
        _cached("tables", 48, 4096, 700, (1, 1), 64, block_size=16, name="tables_prompts_48"),
        # Serving, token phase: a layer's new keys and values, queries and keys rotated.
        _cached("append", 64, 4096, 1, (32, 8), 128, name="append_decode_64"),
        # Serving, prompt phase: prompts and parts of prompts, beginning and ending inside blocks.
        _cached("append", 6, 3000, 2700, (32, 8), 128, name="append_prompts_6"),
        # Serving, token phase, one user: latency of a step.
        _cached("attend", 1, 4096, 1, (32, 8), 128, mixed=False, name="attend_one"),
        # Serving, token phase, many users with caches of all lengths: memory traffic counts.
        _cached("attend", 32, 65536, 1, (32, 8), 128, name="attend_32_mixed"),
        # The same with a dynamic mask: 4096 kept keys of 65536 for each request and kv head.
        _cached("attend", 32, 65535, 1, (32, 8), 128, mixed=False, kept=4096, name="attend_32_kept"),
        # Drafts of one to five tokens that are verified at once, fp16, small heads.
        _cached("attend", 16, 8192, 5, (8, 2), 64, "fp16", block_size=16, name="attend_drafts_16"),
        # Parts of long prompts over what is cached of them already.
        _cached("attend", 2, 14000, 2048, (32, 8), 128, mixed=False, name="attend_prompt_parts"),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    """One more case of the ranges above: rotary up to 65536 tokens, tables of up to 512 requests, caches up to 65536 tokens a
    request, up to five new tokens (drafts) or prompt parts up to 2048."""
    heads = rng.choice(_HEADS)
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    head_dim = rng.choice((64, 64, 128, 128, 128, 96, 256))
    block = rng.choice((16, 32, 64, 64, 128))
    sizes = rng.randint(1, 10 ** 6)
    op = rng.choice(("rotary", "tables", "append", "attend", "attend", "attend"))
    if op == "rotary":
        s = _log(rng, 1, 65536)
        batch = _log(rng, 1, max(1, min(64, 65536 // s)))
        part = rng.choice((1, 1, 2, 4)) if head_dim != 96 else 1
        return _rotary(batch, s, heads, head_dim, rng.choice((dtype, dtype, "fp32")), head_dim // part, rng.random() < 0.5,
                       rng.choice(("none", "linear", "ntk", "yarn")), rng.choice((0, 0, 1000, 1000003)), rng.random() < 0.6)
    if op == "tables":
        r = _log(rng, 1, 512)
        new = rng.choice((1, 5, _log(rng, 16, max(16, 65536 // r))))
        return _cached(op, r, _log(rng, 1, 65536), new, (1, 1), 64, block_size=block, sizes=sizes)
    if op == "append":
        r = _log(rng, 1, 128)
        new = rng.choice((1, 5, _log(rng, 16, max(16, 8192 // r))))
        return _cached(op, r, _log(rng, 1, 8192), new, heads, head_dim, dtype, block, sizes=sizes)
    kind = rng.choice(("token", "token", "kept", "draft", "prompt"))
    if kind == "prompt":
        new = _log(rng, 64, 2048)
        r = _log(rng, 1, max(1, min(8, 4096 // new)))
        return _cached(op, r, _log(rng, 1, 16384), new, heads, head_dim, dtype, block, sizes=sizes)
    r, cached = _log(rng, 1, 32), _log(rng, 64, 65536)
    if kind == "draft":
        return _cached(op, min(r, 16), min(cached, 16384), rng.randint(2, 8), heads, head_dim, dtype, block, sizes=sizes)
    if head_dim == 256:
        r = min(r, 16)
    kept = _log(rng, 64, 4096) if kind == "kept" else 0
    return _cached(op, r, max(cached, kept), 1, heads, head_dim, dtype, block, rng.random() < 0.75, kept, sizes)


# ---- sizes of the requests ------------------------------------------------------------------------------------------
def _sizes(c):
    """(cached tokens, new tokens) of each request; the same for every state of the case."""
    rng = random.Random(c["sizes"])
    r, cached, new = c["requests"], c["cached"], c["new"]
    if not c["mixed"]:
        return [cached] * r, [new] * r
    have, more = [], []
    for i in range(r):
        # prompt phase: every third request is new, with nothing cached yet
        have.append(0 if new > 8 and i % 3 == 0 else rng.randint(max(min(1, cached), cached // 16, min(cached, c["kept"])), cached))
        more.append(rng.randint(max(1, new // 16), new))
    return have, more


def _blocks(n, size):
    return -(-n // size)


def _inv_freq(c):
    """(inverse frequencies in 64 bits, factor on cos and sin) of the case, as the methods define them."""
    r, base, factor = c["rotary_dim"], _BASE, c["factor"]
    if c["scaling"] == "ntk":
        base = base * factor ** (r / (r - 2))
    i = torch.arange(0, r, 2, dtype=torch.float64)
    inv = base ** (-i / r)
    if c["scaling"] == "linear":
        inv = inv / factor
    if c["scaling"] == "yarn":
        dim = [r * math.log(_ORIGINAL / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32.0, 1.0)]
        low, high = max(math.floor(dim[0]), 0), min(math.ceil(dim[1]), r - 1)
        ramp = ((i / 2 - low) / max(high - low, 0.001)).clamp(0, 1)
        inv = inv / factor * ramp + inv * (1 - ramp)
        return inv, 0.1 * math.log(factor) + 1.0
    return inv, 1.0


# ---- what a program has in hand ---------------------------------------------------------------------------------------
def prepare(case, seed):
    """Activations ~ N(0,1), as after a normalisation layer; blocks of the cache handed out in the order in which requests came
    and went, that is, in none."""
    c, dev = case, torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype, H, Hk, d = _DTYPES[c.get("dtype", "bf16")], c["heads"], c["kv_heads"], c["head_dim"]

    def rnd(*shape, grad=False):
        return torch.randn(shape, generator=g, device=dev, dtype=dtype).requires_grad_(grad)

    if c["op"] == "rotary":
        B, S, train = c["batch"], c["seqlen"], c["train"]
        inv, amplitude = _inv_freq(c)
        s = {"case": c, "q": rnd(B, S, H, d, grad=train), "k": rnd(B, S, Hk, d, grad=train), "inv": inv.to(dev), "amplitude": amplitude,
             "positions": (torch.arange(S, device=dev) + c["offset"]).expand(B, S).contiguous()}
        if train:
            s["dq"], s["dk"] = rnd(B, S, H, d), rnd(B, S, Hk, d)
        if own:
            s["frequencies"] = _package().rotary_frequencies(
                c["rotary_dim"], base=_BASE, scaling=c["scaling"], factor=c["factor"], original_length=_ORIGINAL,
                interleaved=c["interleaved"], device=dev)
        return s

    have, more = _sizes(c)
    R, bs = c["requests"], c["block_size"]
    used = [_blocks(n, bs) for n in have]
    after = [_blocks(n + m, bs) for n, m in zip(have, more)]
    width = max(after)
    total = sum(after) + 3
    order = torch.randperm(total, generator=g, device=dev).to(torch.int32)  # blocks, in the order of their use
    n_used = torch.tensor(used, device=dev)
    first = n_used.cumsum(0) - n_used
    at = torch.arange(width, device=dev)[None, :]
    held = at < n_used[:, None]
    table = torch.where(held, order[(first[:, None] + at).clamp(max=total - 1)], torch.full((), -1, dtype=torch.int32, device=dev))
    left = total - sum(used)
    free = torch.zeros(total, dtype=torch.int32, device=dev)
    free[:left] = order[sum(used):].flip(0)
    s = {"case": c, "table": table, "lengths": torch.tensor(have, dtype=torch.int32, device=dev), "free": free,
         "free_count": torch.tensor([left], dtype=torch.int32, device=dev), "ticket": torch.zeros(1, dtype=torch.int32, device=dev),
         "new": torch.tensor(more, dtype=torch.int32, device=dev), "tokens": sum(more), "longest": max(more)}
    s["base"] = s["lengths"].clone()
    if c["op"] == "tables":
        return s

    s["step"] = _extend(s)  # the plan of this step, the same for all layers
    step_lengths = s["step"]["lengths"]
    T = s["tokens"]
    s["q"] = rnd(T, H, d)
    s["k_scale"] = torch.exp2(torch.randint(-8, -4, (total, Hk), generator=g, device=dev).float())
    s["v_scale"] = torch.exp2(torch.randint(-8, -4, (total, Hk), generator=g, device=dev).float())
    for name in ("cache_k", "cache_v"):
        s[name] = torch.empty((total, Hk, bs, d), dtype=_E4M3, device=dev)
        flat = s[name].view(torch.uint8).view(-1)
        for i in range(0, flat.numel(), 1 << 28):
            n = min(1 << 28, flat.numel() - i)
            x = torch.randn(n, generator=g, device=dev, dtype=torch.bfloat16).mul_(80.0).clamp_(-448.0, 448.0)
            flat[i:i + n] = x.to(_E4M3).view(torch.uint8)
    if c["op"] == "append":
        s["k"], s["v"] = rnd(T, Hk, d), rnd(T, Hk, d)
        inv, _ = _inv_freq({"rotary_dim": d, "scaling": "none", "factor": 1.0})
        s["inv"], s["amplitude"] = inv.to(dev), 1.0
        if own:
            s["frequencies"] = _package().rotary_frequencies(d, base=_BASE, device=dev)
    elif c["kept"]:
        W, keys = c["kept"], max(n + m for n, m in zip(have, more))
        s["bias"] = rnd(R, Hk, 1, keys)
        masked = torch.where(torch.arange(keys, device=dev) < step_lengths[:, None, None], s["bias"][:, :, 0].float(), -math.inf)
        pos = masked.topk(min(W, keys), dim=-1).indices.sort(dim=-1).values.to(torch.int32)
        count = step_lengths.clamp(max=W)[:, None].expand(R, Hk).contiguous()
        cap = max(128, _blocks(W, 128) * 128)
        s["key_pos"] = torch.full((R, Hk, cap), 2 ** 31 - 1, dtype=torch.int32, device=dev)
        s["key_pos"][..., :pos.shape[-1]] = pos
        in_use = torch.arange(cap, device=dev) < count[..., None]
        s["key_pos"].masked_fill_(~in_use, 2 ** 31 - 1)
        s["count"], s["slot_mask"], s["keys"] = count, in_use[:, :, None], keys
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------------
def _angles(positions, inv, amplitude):
    a = positions.double()[..., None] * inv
    return (a.cos() * amplitude).float(), (a.sin() * amplitude).float()


def _rotate(x, cos, sin, interleaved):
    """x (..., heads, d), cos and sin (..., rotary_dim / 2), all in 32 bits."""
    half = cos.shape[-1]
    cos, sin = cos[..., None, :], sin[..., None, :]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        x1, x2 = turned[..., 0::2], turned[..., 1::2]
        return torch.cat((torch.stack((x1 * cos - x2 * sin, x2 * cos + x1 * sin), -1).flatten(-2), rest), -1)
    x1, x2 = turned[..., :half], turned[..., half:]
    return torch.cat((x1 * cos - x2 * sin, x2 * cos + x1 * sin, rest), -1)


def _plain_rotary(s):
    c = s["case"]
    cos, sin = _angles(s["positions"], s["inv"], s["amplitude"])
    out = [_rotate(s[n].detach().float(), cos, sin, c["interleaved"]).to(s[n].dtype) for n in ("q", "k")]
    if c["train"]:
        out += [_rotate(s[n].float(), cos, -sin, c["interleaved"]).to(s[n].dtype) for n in ("dq", "dk")]
    return out


def _extend(s):
    """Blocks for the new tokens: the table, the lengths and the free list are brought up to date; returns the step's plan. A request
    takes all its blocks or none."""
    bs, T, dev = s["case"]["block_size"], s["tokens"], s["table"].device
    R, width = s["table"].shape
    have, n = s["lengths"].long(), s["new"].long()
    old, want = (have + bs - 1) // bs, (have + n + bs - 1) // bs
    end = n.cumsum(0)
    may = (n > 0) & (want <= width) & (end <= T)
    need = torch.where(may, want - old, 0)
    taken = need.cumsum(0)
    granted = (n == 0) | (may & ((need == 0) | (taken <= s["free_count"])))
    need = torch.where(granted, need, 0)
    at = torch.arange(width, device=dev)[None, :]
    mine = (at >= old[:, None]) & (at < (old + need)[:, None])
    nth = (taken - need)[:, None] + at - old[:, None]
    s["table"].copy_(torch.where(mine, s["free"][(s["free_count"] - 1 - nth).clamp(0, s["free"].numel() - 1).long()], s["table"]))
    after = torch.where(granted, have + n, have)
    s["lengths"].copy_(after)
    s["free_count"].sub_(torch.where(need > 0, taken, 0).amax(0, keepdim=True).to(torch.int32))
    t = torch.arange(T, device=dev)
    r = torch.searchsorted(end, t, right=True).clamp(max=R - 1)
    inside = t < end[-1]
    pos = torch.where(inside, have[r] + t - (end - n)[r], 0)
    slot = s["table"][r, (pos // bs).clamp(max=width - 1)].long() * bs + pos % bs
    zero = torch.zeros(1, dtype=torch.long, device=dev)
    active = granted & (n > 0)
    whole = lambda x: torch.cat((zero, x.cumsum(0))).to(torch.int32)  # noqa: E731
    return {"cu_seqlens": torch.cat((zero, end)).clamp(max=T).to(torch.int32), "positions": pos.to(torch.int32),
            "slots": torch.where(inside & granted[r], slot, -1), "lengths": after.to(torch.int32), "granted": granted,
            "cu_blocks": whole(torch.where(active, want - have // bs, 0)),
            "cu_chunks": whole(torch.where(active, (have + n + _CHUNK - 1) // _CHUNK, 0))}


def _truncate(s, lengths):
    """Requests go back to the given lengths; the blocks they no longer need return to the free list, the last one taken first."""
    bs, width = s["case"]["block_size"], s["table"].shape[1]
    have = s["lengths"].long()
    keep = torch.minimum(lengths.long().clamp(min=0), have)
    old, new = (have + bs - 1) // bs, (keep + bs - 1) // bs
    gone = old - new
    first = gone.cumsum(0) - gone
    total = gone.sum()
    at = torch.arange(width, device=have.device)[None, :]
    mine = (at >= new[:, None]) & (at < old[:, None])
    place = (s["free_count"] + total - 1 - (first[:, None] + at - new[:, None])).clamp(0, s["free"].numel() - 1)
    count = s["free_count"] + total
    # the same the other way round: which entry of the table each free place gets
    spot = torch.full((s["free"].numel() + 1,), -1, dtype=torch.long, device=have.device)
    flat = torch.arange(s["table"].numel(), device=have.device).view_as(s["table"])
    spot.scatter_(0, torch.where(mine, place, s["free"].numel()).flatten(), torch.where(mine, flat, -1).flatten())
    spot = spot[:-1]
    s["free"].copy_(torch.where(spot >= 0, s["table"].flatten()[spot.clamp(min=0)], s["free"]))
    s["table"].masked_fill_(mine, -1)
    s["lengths"].copy_(keep)
    s["free_count"].copy_(count)


def _plain_tables(s):
    step = _extend(s)
    _truncate(s, s["base"])
    return {**step, "table": s["table"], "left": s["free"], "left_count": s["free_count"], "after": s["lengths"]}


def _exponent(amax):
    """The smallest e with amax <= 448 * 2^e (at least -100)."""
    m, e = torch.frexp(amax)  # amax = m * 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    return torch.where(amax > 0, (e - 9 + (m > 0.875)).clamp(min=-100), -100)


def _units(s):
    """Blocks that the new tokens go to: (request, block, first and last + 1 new token's place in the block, tokens there); as many
    as there can be, those past the last repeat it."""
    c, st = s["case"], s["step"]
    bs, T, R = c["block_size"], s["tokens"], c["requests"]
    most = min(T, T // bs + 2 * R)
    u = torch.minimum(torch.arange(most, device=st["lengths"].device), st["cu_blocks"][-1].long() - 1)
    r = torch.searchsorted(st["cu_blocks"].long(), u, right=True) - 1
    n = (st["cu_seqlens"][1:] - st["cu_seqlens"][:-1]).long()[r]
    before = st["lengths"].long()[r] - n
    nth = before // bs + u - st["cu_blocks"].long()[r]
    block = s["table"][r, nth].long()
    lo = (before - nth * bs).clamp(min=0)
    hi = (before + n - nth * bs).clamp(max=bs)
    place = torch.arange(bs, device=u.device)[None, :]
    token = st["cu_seqlens"].long()[r][:, None] + nth[:, None] * bs + place - before[:, None]
    new = (place >= lo[:, None]) & (place < hi[:, None])
    return block, lo, place, token.clamp(0, T - 1), new


def _write(s, x, name, units):
    """x (tokens, kv heads, d) in 32 bits into the 8-bit cache `name` and its scales."""
    block, lo, place, token, new = units
    cache, scale = s["cache_" + name], s[name + "_scale"]
    rows = x[token].transpose(1, 2)                                   # (units, kv heads, block, d)
    fresh = new[:, None, :, None]
    size = torch.where(fresh & rows.isfinite(), rows.abs(), 0).amax((2, 3))
    e = torch.exp2(_exponent(size).float())
    begun = (lo > 0)[:, None]
    e = torch.where(begun, torch.maximum(e, scale[block]), e)
    old = cache.view(torch.uint8)[block]
    held = (old.view(_E4M3).float() * (scale[block] / e)[..., None, None]).to(_E4M3).view(torch.uint8)
    put = (rows / e[..., None, None]).clamp(-448.0, 448.0).to(_E4M3).view(torch.uint8)
    kept = (place < lo[:, None])[:, None, :, None]
    cache.view(torch.uint8)[block] = torch.where(fresh, put, torch.where(kept, held, old))
    scale[block] = e


def _plain_append(s):
    cos, sin = _angles(s["step"]["positions"], s["inv"], s["amplitude"])
    q = _rotate(s["q"].float(), cos, sin, False).to(s["q"].dtype)
    k = _rotate(s["k"].float(), cos, sin, False)
    units = _units(s)
    _write(s, k, "k", units)
    _write(s, s["v"].float(), "v", units)
    return {"q": q, "k": s["cache_k"], "v": s["cache_v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _cached_rows(s, name, pos):
    """Rows of the 8-bit cache in 32 bits: (requests, kv heads, keys, d). pos: the positions, or the number of the first ones."""
    c = s["case"]
    R, Hk, d, bs = c["requests"], c["kv_heads"], c["head_dim"], c["block_size"]
    cache, scale = s["cache_" + name], s[name + "_scale"]
    if isinstance(pos, int):
        block = s["table"][:, :_blocks(pos, bs)].long().clamp(min=0)
        x = cache.view(torch.uint8)[block].view(_E4M3).float() * scale[block][..., None, None]
        return x.transpose(1, 2).reshape(R, Hk, -1, d)[:, :, :pos]
    r, h = torch.arange(R, device=pos.device)[:, None, None], torch.arange(Hk, device=pos.device)[None, :, None]
    block = s["table"][r, pos // bs].long()
    return cache.view(torch.uint8)[block, h, pos % bs].view(_E4M3).float() * scale[block, h][..., None]


def _plain_attend(s):
    c, st = s["case"], s["step"]
    R, H, Hk, d = c["requests"], c["heads"], c["kv_heads"], c["head_dim"]
    G, N, T, dev = H // Hk, s["longest"], s["tokens"], s["q"].device
    length, first = st["lengths"].long(), st["cu_seqlens"].long()
    n = first[1:] - first[:-1]
    i = torch.arange(N, device=dev)
    q = s["q"][(first[:-1, None] + i).clamp(max=T - 1)].float()        # (R, N, H, d)
    q = q.view(R, N, Hk, G, d).permute(0, 2, 1, 3, 4).reshape(R, Hk, N * G, d)
    if c["kept"]:
        pos = s["key_pos"].long()
        there = pos < length[:, None, None]
        pos = torch.where(there, pos, 0)
        bias = torch.where(there, s["bias"][:, :, 0].float().gather(-1, pos), -math.inf)[:, :, None]
        k, v = _cached_rows(s, "k", pos), _cached_rows(s, "v", pos)
        pos = pos[:, :, None]
    else:
        most = max(a + b for a, b in zip(*_sizes(c)))
        k, v = _cached_rows(s, "k", most), _cached_rows(s, "v", most)
        pos, bias = torch.arange(most, device=dev)[None, None, None], None
    last = (length - n)[:, None] + i                                   # the newest key that each query sees
    seen = pos <= last.repeat_interleave(G, 1)[:, None, :, None]
    x = (q @ k.transpose(-1, -2)) * d ** -0.5
    if bias is not None:
        x = x + bias
    x = x.masked_fill_(~seen, -math.inf)
    del seen, k
    top = x.amax(-1, keepdim=True)
    x = x.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = x.sum(-1, keepdim=True)
    out = (x @ v) / total.masked_fill(total == 0, 1.0)
    out = out.view(R, Hk, N, G, d).permute(0, 2, 1, 3, 4).reshape(R, N, H, d)
    t = torch.arange(T, device=dev)
    r = torch.searchsorted(first[1:], t, right=True).clamp(max=R - 1)
    return out[r, (t - first[r]).clamp(0, N - 1)].to(s["q"].dtype)


# ---- the framework's calls ----------------------------------------------------------------------------------------------
def _own(s):
    fsa, c = _package(), s["case"]
    if c["op"] == "rotary":
        out = fsa.apply_rotary(s["q"], s["k"], s["frequencies"], s["positions"])
        return [*out, *torch.autograd.grad(out, (s["q"], s["k"]), (s["dq"], s["dk"]))] if c["train"] else list(out)
    tables = fsa.BlockTables(s["table"], s["lengths"], s["free"], s["free_count"], s["ticket"], c["block_size"])
    if c["op"] == "tables":
        step = tables.extend(s["new"], s["tokens"])
        tables.truncate(s["base"])
        return {**step._asdict(), "table": s["table"], "left": s["free"], "left_count": s["free_count"], "after": s["lengths"]}
    cache = fsa.QuantizedCache(s["cache_k"], s["cache_v"], s["k_scale"], s["v_scale"])
    step = fsa.CacheStep(**s["step"])
    if c["op"] == "append":
        q = fsa.cache_append(cache, tables, step, s["k"], s["v"], query=s["q"], frequencies=s["frequencies"])
        return {"q": q, "k": s["cache_k"], "v": s["cache_v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    mask = fsa.KeptKeys(s["key_pos"], s["count"], s["slot_mask"], s["keys"]) if c["kept"] else None
    return fsa.flash_sparse_attn_cache_func(s["q"], cache, tables, step, attn_mask=mask, attn_bias=s.get("bias"),
                                            max_seqlen_q=s["longest"], max_seqlen_k=c["cached"] + c["new"])


def run(s):
    if own:
        return _own(s)
    return {"rotary": _plain_rotary, "tables": _plain_tables, "append": _plain_append, "attend": _plain_attend}[s["case"]["op"]](s)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------
def work(case):
    c = case
    size = 4.0 if c.get("dtype") == "fp32" else 2.0
    H, Hk, d = c["heads"], c["kv_heads"], c["head_dim"]
    if c["op"] == "rotary":
        elems = c["batch"] * c["seqlen"] * (H + Hk) * d * (2.0 if c["train"] else 1.0)
        return {"bytes": 2 * size * elems, "flops": 3.0 * elems * c["rotary_dim"] / d}
    have, more = _sizes(c)
    R, T, bs = c["requests"], sum(more), c["block_size"]
    if c["op"] == "tables":
        fresh = sum(_blocks(a + b, bs) - _blocks(a, bs) for a, b in zip(have, more))
        # lengths read and written twice, the plan, the slot (8 bytes) and position of each token, blocks into the table and back
        return {"bytes": R * 4.0 * 8 + T * 12.0 + fresh * 4.0 * 4, "flops": 4.0 * T + 16.0 * R}
    if c["op"] == "append":
        return {"bytes": T * d * (2 * size * H + (size + 1) * 2 * Hk), "flops": 3.0 * T * d * (H + Hk) + 4.0 * T * d * Hk}
    pairs, rows = 0.0, 0.0
    for a, b in zip(have, more):
        if c["kept"]:
            pairs += min(c["kept"], a + b)
            rows += min(c["kept"], a + b)
        else:
            pairs += b * a + b * (b + 1) / 2
            rows += a + b
    lists = rows * Hk * (4.0 + size) if c["kept"] else 0.0
    return {"bytes": 2 * size * T * H * d + rows * Hk * 2 * d + rows / bs * (4 + 8 * Hk) + lists, "flops": 4.0 * pairs * H * d}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------
def _turn(x, positions, inv, amplitude, interleaved, sign=1.0):
    """Pairs of x as complex numbers, times amplitude * exp(i angle)."""
    half = inv.numel()
    x = x.detach().double()
    pair = x[..., :2 * half].unflatten(-1, (half, 2)) if interleaved else x[..., :2 * half].unflatten(-1, (2, half)).transpose(-1, -2)
    z = torch.view_as_complex(pair.contiguous()) * torch.polar(torch.full((), amplitude, dtype=torch.float64, device=x.device),
                                                              sign * positions.double()[..., None, None] * inv)
    y = torch.view_as_real(z)
    y = y.flatten(-2) if interleaved else y.transpose(-1, -2).flatten(-2)
    return torch.cat((y, x[..., 2 * half:]), -1)


def exact(case, seed):
    c = case
    if c["op"] == "tables":  # whole numbers
        return None
    s = prepare(case, seed)
    if c["op"] == "rotary":
        args = (s["positions"], s["inv"], s["amplitude"], c["interleaved"])
        out = [_turn(s["q"], *args), _turn(s["k"], *args)]
        if c["train"]:
            out += [_turn(s["dq"], *args, sign=-1.0), _turn(s["dk"], *args, sign=-1.0)]
        return out
    st, bs, table = s["step"], c["block_size"], s["table"].tolist()
    first, length = st["cu_seqlens"].tolist(), st["lengths"].tolist()
    if c["op"] == "append":
        q, k = (_turn(s[n], st["positions"], s["inv"], 1.0, False) for n in ("q", "k"))
        for name, x in (("k", k), ("v", s["v"].double())):
            values, scales = s["cache_" + name], s[name + "_scale"]
            for r in range(c["requests"]):
                n = first[r + 1] - first[r]
                start = length[r] - n
                for b in range(start // bs, _blocks(length[r], bs)):
                    lo, hi = max(start, b * bs), min(length[r], (b + 1) * bs)
                    rows = x[first[r] + lo - start:first[r] + hi - start].transpose(0, 1)
                    e = torch.ceil(torch.log2(rows.abs().amax((1, 2)) / 448.0))
                    at = table[r][b]
                    if lo > b * bs:
                        before = torch.log2(scales[at].double())
                        e = torch.maximum(e, before)
                        held = values[at, :, :lo - b * bs].double() * torch.exp2(before - e)[:, None, None]
                        values[at, :, :lo - b * bs] = held.to(_E4M3)
                    values[at, :, lo - b * bs:hi - b * bs] = (rows / torch.exp2(e)[:, None, None]).to(_E4M3)
                    scales[at] = torch.exp2(e).float()
        return {"q": q, "k": s["cache_k"], "v": s["cache_v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    H, Hk, d = c["heads"], c["kv_heads"], c["head_dim"]
    out = torch.zeros((s["tokens"], H, d), dtype=torch.float64, device=s["q"].device)
    for r in range(c["requests"]):
        blocks = s["table"][r, :_blocks(length[r], bs)].long()
        for h in range(Hk):
            k = (s["cache_k"][blocks, h].double() * s["k_scale"][blocks, h].double()[:, None, None]).reshape(-1, d)[:length[r]]
            v = (s["cache_v"][blocks, h].double() * s["v_scale"][blocks, h].double()[:, None, None]).reshape(-1, d)[:length[r]]
            keys = torch.arange(length[r], device=k.device)
            if c["kept"]:
                keys = s["key_pos"][r, h, :int(s["count"][r, h])].long()
                k, v = k[keys], v[keys]
            for g in range(H // Hk):
                head = h * (H // Hk) + g
                x = s["q"][first[r]:first[r + 1], head].double() @ k.T / math.sqrt(d)
                if c["kept"]:
                    x = x + s["bias"][r, h, 0, keys].double()
                n = first[r + 1] - first[r]
                newest = length[r] - n + torch.arange(n, device=k.device)
                x = x.masked_fill(keys[None, :] > newest[:, None], -math.inf)
                out[first[r]:first[r + 1], head] = torch.softmax(x, -1) @ v
    return out
