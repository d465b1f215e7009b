"""Attention with a sliding window and sink tokens, in training, on packed sequences and over the paged 8-bit cache, and the verification
of drafted tokens. Each case is a dict of plain values:

  op        "window"  flash_sparse_attn_window_func    "packed"  flash_sparse_attn_window_varlen_func
            "cache"   flash_sparse_attn_cache_func     "verify"  verify_drafts
  heads, kv_heads, head_dim, dtype; window (keys that a query sees, its own among them), sinks (first keys that stay visible)
  batch, seqlen, past (keys before the first query), padded (a mask of the keys that are there), train: with the gradients     window
  tokens, sequences, train                                                                                              packed
  requests, cached, new, mixed, block_size    requests with up to `cached` tokens in the cache and up to `new` more      cache
  requests, new, mixed, vocab, dtype (of the logits), probs (the drafter's probabilities are given), temperature
            (-1: one for each request, some of them 0)                                                                  verify
  sizes     where sizes differ within a case, they are drawn from this seed: states of one case have the same ones

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
_CHUNK = 64  # tokens of a unit of the cache attention's work

# (query heads, kv heads): multi-query, grouped and plain multi-head layouts
_HEADS = ((2, 1), (8, 2), (8, 8), (12, 4), (16, 4), (16, 1), (32, 8))


def _package():
    path = os.path.join(os.getcwd(), "flash-dmattn_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import flash_sparse_attn

    return flash_sparse_attn


def _case(op, name, **more):
    c = {} if name is None else {"name": name}
    c.update(op=op, **more)
    return c


def _window(batch, seqlen, heads, head_dim, window, sinks, dtype="bf16", past=0, padded=False, train=True, sizes=1, name=None):
    return _case("window", name, batch=batch, seqlen=seqlen, heads=heads[0], kv_heads=heads[1], head_dim=head_dim, window=window,
                 sinks=sinks, dtype=dtype, past=past, padded=padded, train=train, sizes=sizes)


def _packed(tokens, sequences, heads, head_dim, window, sinks, dtype="bf16", train=True, sizes=1, name=None):
    return _case("packed", name, tokens=tokens, sequences=sequences, heads=heads[0], kv_heads=heads[1], head_dim=head_dim,
                 window=window, sinks=sinks, dtype=dtype, train=train, sizes=sizes)


def _cache(requests, cached, new, heads, head_dim, window, sinks, dtype="bf16", block_size=64, mixed=True, sizes=1, name=None):
    return _case("cache", name, requests=requests, cached=cached, new=new, heads=heads[0], kv_heads=heads[1], head_dim=head_dim,
                 window=window, sinks=sinks, dtype=dtype, block_size=block_size, mixed=mixed, sizes=sizes)


def _verify(requests, new, vocab, dtype="bf16", mixed=True, probs=True, temperature=1.0, sizes=1, name=None):
    return _case("verify", name, requests=requests, new=new, vocab=vocab, dtype=dtype, mixed=mixed, probs=probs,
                 temperature=temperature, sizes=sizes)


def listed():
    return [
        # A layer of a long-context training step: forward and backward, the largest case.
        _window(1, 32768, (32, 8), 128, 2048, 4, name="window_train_32k"),
        # A batch of padded sequences, small heads, many sinks.
        _window(4, 2048, (16, 4), 64, 256, 64, padded=True, name="window_train_padded"),
        # Short odd sequences, fp16, a window without sinks: launches and the host path count.
        _window(2, 301, (12, 4), 96, 64, 0, "fp16", name="window_train_short"),
        # Prompt phase with wide heads that share one kv head, behind keys that are there already; forward alone.
        _window(1, 8191, (16, 1), 256, 1024, 128, past=1000, train=False, name="window_prefill_wide"),
        # Packed training: a few sequences of any length.
        _packed(8192, 5, (16, 4), 128, 512, 4, name="packed_train_5"),
        # Packed training: many short sequences, some shorter than the window.
        _packed(3001, 40, (8, 8), 64, 48, 1, "fp16", name="packed_train_40"),
        # Serving, token phase, one user far beyond the window: latency of a step.
        _cache(1, 40000, 1, (32, 8), 128, 4096, 4, mixed=False, name="cache_one"),
        # Serving, drafts of up to five tokens for many users, caches of all lengths.
        _cache(64, 32768, 5, (32, 8), 128, 2048, 64, name="cache_drafts_64"),
        # Parts of long prompts over what is cached of them.
        _cache(4, 14000, 2048, (32, 8), 128, 2048, 4, mixed=False, name="cache_prompt_parts"),
        # One user's three drafts, made by a look-up (no probabilities): latency of a step.
        _verify(1, 4, 32000, mixed=False, probs=False, name="verify_one"),
        # Many users' drafts from a smaller model with its probabilities, a large vocabulary: memory traffic counts.
        _verify(64, 9, 131072, mixed=False, name="verify_64"),
        # Users with and without drafts, fp32 logits, an odd vocabulary, some of them greedy.
        _verify(200, 6, 50257, "fp32", temperature=-1.0, name="verify_mixed"),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    """One more case of the ranges above: up to 32768 queries, windows of 1 to 4096 keys, up to 256 sinks, caches up to 65536 tokens a
    request, up to eight new tokens (drafts) or prompt parts up to 2048, vocabularies of 1000 to 131072."""
    heads = rng.choice(_HEADS)
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    head_dim = rng.choice((64, 64, 128, 128, 128, 96, 256))
    window, sinks = _log(rng, 1, 4096), rng.choice((0, 1, 4, 4, 64, rng.randint(2, 256)))
    sizes = rng.randint(1, 10 ** 6)
    op = rng.choice(("window", "window", "packed", "cache", "cache", "verify", "verify"))
    if op == "window":
        # queries x heads x window: no more than the largest listed case
        s = _log(rng, 1, 32768)
        window = min(window, max(64, 2 ** 26 // s))
        batch = _log(rng, 1, max(1, min(16, 2 ** 31 // (s * (window + 512) * heads[0]))))
        train = rng.random() < 0.75
        return _window(batch, s, heads, min(head_dim, 128) if train else head_dim, window, sinks, dtype,
                       rng.choice((0, 0, rng.randint(1, 2000))), rng.random() < 0.4, train, sizes)
    if op == "packed":
        n = _log(rng, 1, 64)
        return _packed(max(n, _log(rng, 64, 8192)), n, heads, min(head_dim, 128), min(window, 1024), sinks, dtype, rng.random() < 0.75, sizes)
    if op == "verify":
        vocab = _log(rng, 1000, 131072)
        return _verify(_log(rng, 1, max(1, min(256, 2 ** 23 // vocab))), rng.randint(1, 9), vocab, rng.choice(("bf16", "fp16", "fp32")),
                       rng.random() < 0.7, rng.random() < 0.6, rng.choice((1.0, 0.7, -1.0, 0.0)), sizes)
    block = rng.choice((16, 32, 64, 64, 128))
    if rng.random() < 0.35:
        new = _log(rng, 64, 2048)
        return _cache(_log(rng, 1, max(1, min(8, 4096 // new))), _log(rng, 1, 16384), new, heads, head_dim, window, sinks, dtype, block, sizes=sizes)
    return _cache(_log(rng, 1, 64), _log(rng, 1, 32768), rng.choice((1, 1, rng.randint(2, 8))), heads, min(head_dim, 128), window, sinks,
                  dtype, block, rng.random() < 0.75, sizes)


# ---- sizes within a case ----------------------------------------------------------------------------------------------
def _lengths(c):
    """Keys that are there in each row of a padded batch; tokens of each packed sequence."""
    rng = random.Random(c["sizes"])
    if c["op"] == "window":
        keys = c["seqlen"] + c["past"]
        return [rng.randint(max(1, keys // 3), keys) if c["padded"] else keys for _ in range(c["batch"])]
    cuts = sorted(rng.sample(range(1, c["tokens"]), c["sequences"] - 1)) if c["sequences"] > 1 else []
    return [b - a for a, b in zip([0] + cuts, cuts + [c["tokens"]])]


def _requests(c):
    """(cached tokens, new tokens) of each request."""
    rng = random.Random(c["sizes"])
    r, new, cached = c["requests"], c["new"], c.get("cached", 0)
    if not c["mixed"]:
        return [cached] * r, [new] * r
    # prompt phase: every third request is new, with nothing cached yet
    have = [0 if new > 8 and i % 3 == 0 else rng.randint(max(min(1, cached), cached // 16), cached) for i in range(r)]
    return have, [rng.randint(max(1, new // 16), new) for _ in range(r)]


def _blocks(n, size):
    return -(-n // size)


# ---- what a program has in hand ---------------------------------------------------------------------------------------
def prepare(case, seed):
    """Activations ~ N(0,1), as after a normalisation layer; blocks of the cache handed out in the order in which requests came and
    went, that is, in none; logits of a model that is sure of some tokens, drafts from one that resembles it."""
    c, dev = case, torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = _DTYPES[c["dtype"]]

    def rnd(*shape, grad=False):
        return torch.randn(shape, generator=g, device=dev, dtype=dtype).requires_grad_(grad)

    def ints(x, kind=torch.int32):
        return torch.tensor(x, dtype=kind, device=dev)

    s = {"case": c}
    if c["op"] in ("window", "packed"):
        H, Hk, d, train = c["heads"], c["kv_heads"], c["head_dim"], c["train"]
        if c["op"] == "window":
            rows, keys = (c["batch"], c["seqlen"]), (c["batch"], c["seqlen"] + c["past"])
            if c["padded"]:
                s["mask"] = (torch.arange(keys[1], device=dev) < ints(_lengths(c))[:, None])[:, None, None, :].contiguous()
        else:
            rows = keys = (c["tokens"],)
            lengths = _lengths(c)
            s["cu"], s["longest"] = ints([sum(lengths[:i]) for i in range(len(lengths) + 1)]), max(lengths)
        s["q"], s["k"], s["v"] = rnd(*rows, H, d, grad=train), rnd(*keys, Hk, d, grad=train), rnd(*keys, Hk, d, grad=train)
        if train:
            s["dout"] = rnd(*rows, H, d)
        return s

    have, more = _requests(c)
    R, T = c["requests"], sum(more)
    s["tokens"], s["longest"] = T, max(more)
    cu = [sum(more[:i]) for i in range(R + 1)]
    bs = c.get("block_size", 64)
    if c["op"] == "verify":
        have = [17 + 5 * i for i in range(R)]
    after = [_blocks(a + b, bs) for a, b in zip(have, more)]
    width, total = max(after), sum(after) + 3
    # the plan of the step, as the block tables leave it
    order = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    n_after = ints(after, torch.long)
    at = torch.arange(width, device=dev)[None, :]
    s["table"] = torch.where(at < n_after[:, None], order[((n_after.cumsum(0) - n_after)[:, None] + at).clamp(max=total - 1)],
                             torch.full((), -1, dtype=torch.int32, device=dev))
    s["lengths"] = ints([a + b for a, b in zip(have, more)])
    positions = torch.cat([torch.arange(a, a + b) for a, b in zip(have, more)]).to(dev)
    request = torch.repeat_interleave(torch.arange(R, device=dev), ints(more, torch.long))
    s["step"] = {"cu_seqlens": ints(cu), "positions": positions.to(torch.int32),
                 "slots": s["table"][request, positions // bs].long() * bs + positions % bs, "lengths": s["lengths"].clone(),
                 "granted": torch.ones(R, dtype=torch.bool, device=dev),
                 "cu_blocks": ints([sum(after[j] - have[j] // bs for j in range(i)) for i in range(R + 1)]),
                 "cu_chunks": ints([sum(_blocks(have[j] + more[j], _CHUNK) for j in range(i)) for i in range(R + 1)])}
    if c["op"] == "cache":
        H, Hk, d = c["heads"], c["kv_heads"], c["head_dim"]
        s["free"], s["free_count"] = order[-3:].contiguous(), ints([3])
        s["ticket"] = ints([0])
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
        return s

    V = c["vocab"]
    logits = torch.randn((T, V), generator=g, device=dev) * 3.0
    s["logits"] = logits.to(dtype)
    s["uniforms"] = torch.rand(T, generator=g, device=dev)
    if c["temperature"] < 0:
        t = torch.rand(R, generator=g, device=dev) + 0.5
        s["temperature"] = torch.where(torch.arange(R, device=dev) % 3 == 1, 0.0, t)
    else:
        s["temperature"] = c["temperature"]
    # the drafter's token after each token: drawn from its probabilities, or its likeliest
    guess = logits.add_(torch.randn((T, V), generator=g, device=dev), alpha=0.5)
    if c["probs"]:
        s["probs"] = torch.softmax(guess, -1)
        guess = guess - torch.log(-torch.log(torch.rand((T, V), generator=g, device=dev).clamp_(1e-20, 1.0 - 1e-7)))
    drafts = guess.argmax(-1)
    first = torch.randint(0, V, (T,), generator=g, device=dev)
    begins = torch.zeros(T, dtype=torch.bool, device=dev)
    begins[s["step"]["cu_seqlens"][:-1].long()] = True
    s["ids"] = torch.where(begins, first, drafts.roll(1))
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------------
def _blocked(q, k, v, keep, window, sinks, dout=None):
    """Attention of q (B, Sq, H, d) over k, v (B, Sk, Hk, d) in 32 bits, keep (B, Sk): a block of queries at a time, over the keys that
    some of them see. Returns out, and with dout (out, dq, dk, dv)."""
    B, Sq, H, d = q.shape
    Sk, Hk = k.shape[1:3]
    G, off, dev = H // Hk, Sk - Sq, q.device
    window, sinks = min(window, Sk), min(sinks, Sk)
    bq = min(max(window // 8, 32), 256)
    nb = _blocks(Sq, bq)
    width = window - 1 + bq
    block = torch.arange(nb, device=dev)[:, None] * bq
    qpos = off + block + torch.arange(bq, device=dev)                         # (nb, bq)
    kpos = off + block + torch.arange(width, device=dev) - (window - 1)       # (nb, width)
    sink = torch.arange(sinks, device=dev).expand(nb, sinks)
    kpos = torch.cat((kpos, sink), 1)                                         # sinks once more, where the window does not reach
    there = (kpos >= 0) & (kpos < Sk)
    at = kpos.clamp(0, Sk - 1)
    behind = kpos[:, None, :] <= qpos[:, :, None] - window
    is_sink = torch.arange(width + sinks, device=dev) >= width
    seen = torch.where(is_sink, behind, ~behind & (kpos[:, None, :] <= qpos[:, :, None])) & there[:, None, :]
    seen = seen[None] & keep[:, at][:, :, None, :]                            # (B, nb, bq, keys)
    seen = seen[:, None, :, None]                                             # (B, 1, nb, 1, bq, keys)

    def rows(x):  # (B, Sq, H, d) -> (B, Hk, nb, G, bq, d)
        x = torch.cat((x, x.new_zeros(B, nb * bq - Sq, H, d)), 1)
        return x.view(B, nb, bq, Hk, G, d).permute(0, 3, 1, 4, 2, 5)

    def back(x):
        return x.permute(0, 2, 4, 1, 3, 5).reshape(B, nb * bq, H, d)[:, :Sq]

    n = at.shape[1]
    kb, vb = (x[:, at].permute(0, 3, 1, 2, 4) for x in (k, v))                # (B, Hk, nb, keys, d)
    qb = rows(q).reshape(B, Hk, nb, G * bq, d)
    p = (qb @ kb.transpose(-1, -2)).mul_(d ** -0.5).view(B, Hk, nb, G, bq, n).masked_fill_(~seen, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(top.masked_fill_(top == -math.inf, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(total.masked_fill_(total == 0, 1.0)).view(B, Hk, nb, G * bq, n)
    out = p @ vb
    result = back(out.view(B, Hk, nb, G, bq, d))
    if dout is None:
        return result
    do = rows(dout).reshape(B, Hk, nb, G * bq, d)
    grads = torch.zeros((2, B, Sk, Hk, d), dtype=q.dtype, device=dev)
    grads[1].index_add_(1, at.flatten(), (p.transpose(-1, -2) @ do).permute(0, 2, 3, 1, 4).reshape(B, nb * n, Hk, d))
    ds = (do @ vb.transpose(-1, -2)).sub_((do * out).sum(-1, keepdim=True)).mul_(p).mul_(d ** -0.5)
    del p
    dq = back((ds @ kb).view(B, Hk, nb, G, bq, d))
    grads[0].index_add_(1, at.flatten(), (ds.transpose(-1, -2) @ qb).permute(0, 2, 3, 1, 4).reshape(B, nb * n, Hk, d))
    return [result, dq, grads[0], grads[1]]


def _plain_window(s):
    c = s["case"]
    keys = c["seqlen"] + c["past"]
    keep = s["mask"][:, 0, 0] if c["padded"] else torch.ones((c["batch"], keys), dtype=torch.bool, device=s["q"].device)
    args = [s[n].detach().float() for n in ("q", "k", "v")]
    out = _blocked(*args, keep, c["window"], c["sinks"], s["dout"].float() if c["train"] else None)
    return [x.to(s["q"].dtype) for x in out] if c["train"] else [out.to(s["q"].dtype)]


def _plain_packed(s):
    """The sequences as rows of a padded batch."""
    c, first = s["case"], s["cu"].long()
    dev, T = first.device, c["tokens"]
    place = torch.arange(s["longest"], device=dev)
    token = (first[:-1, None] + place).clamp(max=T - 1)
    keep = place < (first[1:] - first[:-1])[:, None]
    r = torch.searchsorted(first[1:], torch.arange(T, device=dev), right=True)
    mine = torch.arange(T, device=dev) - first[r]
    args = [s[n].detach().float()[token] for n in ("q", "k", "v")]
    dout = s["dout"].float()[token] * keep[..., None, None] if c["train"] else None
    out = _blocked(*args, keep, c["window"], c["sinks"], dout)
    return [x[r, mine].to(s["q"].dtype) for x in (out if c["train"] else [out])]


def _plain_cache(s):
    c, st = s["case"], s["step"]
    R, H, Hk, d, bs, W = c["requests"], c["heads"], c["kv_heads"], c["head_dim"], c["block_size"], c["window"]
    G, N, T, dev = H // Hk, s["longest"], s["tokens"], s["q"].device
    length, first = st["lengths"].long(), st["cu_seqlens"].long()
    n = first[1:] - first[:-1]
    i = torch.arange(N, device=dev)
    q = s["q"][(first[:-1, None] + i).clamp(max=T - 1)].float()
    q = q.view(R, N, Hk, G, d).permute(0, 2, 1, 3, 4).reshape(R, Hk, N * G, d)
    # the keys that some query of the request sees: the sinks, and the last ones
    most = max(a + b for a, b in zip(*_requests(c)))
    near = min(W + N - 1, most)
    pos = torch.cat((torch.arange(min(c["sinks"], most), device=dev).expand(R, -1),
                     length[:, None] - near + torch.arange(near, device=dev)), 1)     # (R, keys)
    is_sink = torch.arange(pos.shape[1], device=dev) < min(c["sinks"], most)
    there = torch.where(is_sink, pos < length[:, None], pos >= c["sinks"])
    at = pos.clamp(0, most - 1)
    block = torch.take_along_dim(s["table"], at // bs, 1).long().clamp(min=0)[:, None, :]
    h = torch.arange(Hk, device=dev)[None, :, None]

    def cached(name):
        x = s["cache_" + name].view(torch.uint8)[block, h, (at % bs)[:, None, :]].view(_E4M3).float()
        return x * s[name + "_scale"][block, h][..., None]

    x = (q @ cached("k").transpose(-1, -2)).mul_(d ** -0.5)
    last = ((length - n)[:, None] + i).repeat_interleave(G, 1)[:, None, :, None]
    key = pos[:, None, None, :]
    x = x.masked_fill_(~(there[:, None, None, :] & (key <= last) & (is_sink | (key > last - W))), -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(top.masked_fill_(top == -math.inf, 0.0)).exp_()
    total = x.sum(-1, keepdim=True)
    out = (x @ cached("v")) / total.masked_fill_(total == 0, 1.0)
    out = out.view(R, Hk, N, G, d).permute(0, 2, 1, 3, 4).reshape(R, N, H, d)
    t = torch.arange(T, device=dev)
    r = torch.searchsorted(first[1:], t, right=True).clamp(max=R - 1)
    return out[r, (t - first[r]).clamp(0, N - 1)].to(s["q"].dtype)


def _plain_verify(s):
    """In 64 bits: a random number beside a border decides between two tokens."""
    c, st = s["case"], s["step"]
    R, V, T, dev = c["requests"], c["vocab"], s["tokens"], s["ids"].device
    first = st["cu_seqlens"].long()
    n = first[1:] - first[:-1]
    i = torch.arange(s["longest"], device=dev)
    row = (first[:-1, None] + i).clamp(max=T - 1)                             # (R, rows)
    request = torch.searchsorted(first[1:], torch.arange(T, device=dev), right=True)
    temperature = torch.as_tensor(s["temperature"], dtype=torch.float32, device=dev).double().expand(R)
    greedy = temperature == 0
    x = s["logits"].double()
    best = x.argmax(-1)
    x = x.div_(temperature.masked_fill(greedy, 1.0)[request][:, None])
    x = x.sub_(x.amax(-1, keepdim=True)).exp_()
    x = x.div_(x.sum(-1, keepdim=True))                                       # the target's probabilities
    token = s["ids"].long().roll(-1)                                          # of each row: the draft behind it
    p = x.gather(1, token[:, None])[:, 0]
    q = s["probs"].gather(1, token[:, None])[:, 0].double() if c["probs"] else torch.ones_like(p)
    passed = torch.where(greedy[request], token == best, s["uniforms"].double() * q < p)
    accepted = (passed[row] & (i < n[:, None] - 1)).long().cumprod(1).sum(1)
    at = first[:-1] + accepted                                                # the row that the next token comes from
    rest = x[at]
    everything = accepted == n - 1
    if c["probs"]:
        left = (rest - s["probs"][at].double()).clamp_(min=0.0)
    else:
        left = rest.scatter(1, token[at][:, None], 0.0)
    left = torch.where(everything[:, None] | (left.sum(-1, keepdim=True) == 0), rest, left)
    edges = left.cumsum(-1)
    next_token = (edges <= s["uniforms"].double()[first[1:] - 1][:, None] * edges[:, -1:]).sum(-1).clamp(max=V - 1)
    return {"accepted": accepted.to(torch.int32), "next_tokens": torch.where(greedy, best[at], next_token),
            "lengths": (st["lengths"].long() - (n - 1 - accepted)).to(torch.int32)}


# ---- the framework's calls ----------------------------------------------------------------------------------------------
def _own(s):
    fsa, c = _package(), s["case"]
    if c["op"] in ("window", "packed"):
        if c["op"] == "window":
            out = fsa.flash_sparse_attn_window_func(s["q"], s["k"], s["v"], c["window"], c["sinks"], attn_mask=s.get("mask"))
        else:
            out = fsa.flash_sparse_attn_window_varlen_func(s["q"], s["k"], s["v"], s["cu"], s["cu"], s["longest"], s["longest"],
                                                           c["window"], c["sinks"])
        return [out, *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])] if c["train"] else [out]
    step = fsa.CacheStep(**s["step"])
    if c["op"] == "verify":
        res = fsa.verify_drafts(step, s["ids"], s["logits"], s["uniforms"], draft_probs=s.get("probs"), temperature=s["temperature"])
        return {"accepted": res.accepted, "next_tokens": res.next_tokens, "lengths": res.lengths}
    tables = fsa.BlockTables(s["table"], s["lengths"], s["free"], s["free_count"], s["ticket"], c["block_size"])
    cache = fsa.QuantizedCache(s["cache_k"], s["cache_v"], s["k_scale"], s["v_scale"])
    return fsa.flash_sparse_attn_cache_func(s["q"], cache, tables, step, max_seqlen_q=s["longest"], max_seqlen_k=c["cached"] + c["new"],
                                            sliding_window=c["window"], sink_tokens=c["sinks"])


def run(s):
    if own:
        return _own(s)
    return {"window": _plain_window, "packed": _plain_packed, "cache": _plain_cache, "verify": _plain_verify}[s["case"]["op"]](s)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------
def _pairs(first, n, window, sinks):
    """Keys that queries at positions first .. first + n - 1 see, summed up, and how many different ones."""
    pairs = keys = 0
    for p in range(first, first + n):
        near = min(window, p + 1)
        pairs += near + min(sinks, p + 1 - near)
    if n > 0:
        oldest = max(0, first - window + 1)
        keys = first + n - oldest + min(sinks, oldest)
    return pairs, keys


def work(case):
    c = case
    if c["op"] == "verify":
        _, more = _requests(c)
        T, V, R = sum(more), c["vocab"], c["requests"]
        size = 4.0 if c["dtype"] == "fp32" else 2.0
        # the logits once; of the drafter's probabilities those of the drafts, and a row for each request's next token
        probs = 4.0 * (T - R + R * V) if c["probs"] and max(more) > 1 else 0.0
        return {"bytes": T * V * size + probs + T * 12.0 + R * 24.0, "flops": 4.0 * T * V}
    H, Hk, d, W, S = c["heads"], c["kv_heads"], c["head_dim"], c["window"], c["sinks"]
    if c["op"] == "cache":
        seen = [_pairs(a, b, W, S) for a, b in zip(*_requests(c))]
        T, rows = sum(_requests(c)[1]), sum(x[1] for x in seen)
        return {"bytes": 4.0 * T * H * d + rows * Hk * 2.0 * d + rows / c["block_size"] * (4.0 + 8.0 * Hk),
                "flops": 4.0 * sum(x[0] for x in seen) * H * d}
    if c["op"] == "window":
        # (padding leaves keys out and queries in)
        pairs = c["batch"] * _pairs(c["past"], c["seqlen"], W, S)[0]
        rows, keys = c["batch"] * c["seqlen"], c["batch"] * (c["seqlen"] + c["past"])
    else:
        pairs, rows = sum(_pairs(0, n, W, S)[0] for n in _lengths(c)), c["tokens"]
        keys = rows
    size = 2.0 * d
    # forward: q, k, v in, out out; backward: those, dout in and the gradients out
    forward, backward = rows * H * 2 + keys * Hk * 2, rows * H * 2 + keys * Hk * 2
    return {"bytes": size * (forward + (backward if c["train"] else 0)), "flops": (14.0 if c["train"] else 4.0) * pairs * H * d}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------
def _definition(q, k, v, first, window, sinks, there, dout=None):
    """One head: queries q (n, d) at positions first, first + 1, ... over keys k, v (m, d) at positions 0, 1, ... of which `there` are
    there. All in 64 bits, a part of the queries at a time."""
    n, d = q.shape
    m, step = k.shape[0], 2048
    out = torch.zeros_like(q)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for a in range(0, n, step):
        b = min(n, a + step)
        lo = max(0, first + a - window + 1) if first + a - window + 1 > sinks else 0
        hi = min(m, first + b)
        if hi <= 0:
            continue
        keys = torch.arange(lo, hi, device=q.device)
        if lo:
            keys = torch.cat((torch.arange(sinks, device=q.device), keys))
        t = torch.arange(first + a, first + b, device=q.device)[:, None]
        visible = (keys <= t) & ((t - keys < window) | (keys < sinks)) & there[keys]
        x = q[a:b] @ k[keys].T / math.sqrt(d)
        x = torch.where(visible, x, torch.full((), -math.inf, dtype=x.dtype, device=x.device))
        p = torch.nan_to_num(torch.softmax(x, -1), nan=0.0)
        out[a:b] = p @ v[keys]
        if dout is not None:
            g = dout[a:b]
            dp = g @ v[keys].T
            dx = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(d)
            dq[a:b] = dx @ k[keys]
            dk.index_add_(0, keys, dx.T @ q[a:b])
            dv.index_add_(0, keys, p.T @ g)
    return out, dq, dk, dv


def exact(case, seed):
    c = case
    if c["op"] == "verify":  # whole numbers, whose plain form is in 64 bits
        return None
    s = prepare(case, seed)
    H, Hk, d, W, S = c["heads"], c["kv_heads"], c["head_dim"], c["window"], c["sinks"]
    q = s["q"].detach().double()
    if c["op"] == "cache":
        out, bs = torch.zeros_like(q), c["block_size"]
        first, length = s["step"]["cu_seqlens"].tolist(), s["step"]["lengths"].tolist()
        for r in range(c["requests"]):
            blocks, rows = s["table"][r, :_blocks(length[r], bs)].long(), slice(first[r], first[r + 1])
            for h in range(H):
                kv = h // (H // Hk)
                k, v = ((s["cache_" + x][blocks, kv].double() * s[x + "_scale"][blocks, kv].double()[:, None, None]).reshape(-1, d)[:length[r]]
                        for x in ("k", "v"))
                there = torch.ones(length[r], dtype=torch.bool, device=q.device)
                out[rows, h] = _definition(q[rows, h], k, v, length[r] - (first[r + 1] - first[r]), W, S, there)[0]
        return out
    k, v = s["k"].detach().double(), s["v"].detach().double()
    dout = s["dout"].double() if c["train"] else None
    res = [torch.zeros_like(x) for x in (q, q, k, v)]
    if c["op"] == "window":
        parts = [((b, slice(None)), (b, slice(None)), c["past"], n) for b, n in enumerate(_lengths(c))]
    else:
        cu = s["cu"].tolist()
        parts = [((slice(a, b),), (slice(a, b),), 0, b - a) for a, b in zip(cu, cu[1:])]
    for rows, keys, first, n in parts:
        for h in range(H):
            kv = h // (H // Hk)
            kh = k[keys + (kv,)]
            there = torch.arange(kh.shape[0], device=q.device) < n
            got = _definition(q[rows + (h,)], kh, v[keys + (kv,)], first, W, S, there, None if dout is None else dout[rows + (h,)])
            res[0][rows + (h,)] = got[0]
            res[1][rows + (h,)] = got[1]
            res[2][keys + (kv,)] += got[2]
            res[3][keys + (kv,)] += got[3]
    return res if c["train"] else res[:1]
