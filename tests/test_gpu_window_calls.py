"""Attention with a sliding window and sinks: how it is called. Layouts, head dims between the kernels' own, streams, captures, tracing,
repeated runs, lengths of zero, refusals, and gradients against differences of the definition. Bounds are those of test_gpu_window.py."""
import pytest
import torch

import flash_sparse_attn as fsa
from flash_sparse_attn.flash_sparse_attn_interface import set_kernel_path
from test_gpu_window import check, padding, packed_reference, reference, tensors

pytestmark = pytest.mark.gpu
window_func, varlen_func = fsa.flash_sparse_attn_window_func, fsa.flash_sparse_attn_window_varlen_func


def step(q, k, v, dout, *args, **kw):
    out = window_func(q, k, v, *args, **kw)
    return [out, *torch.autograd.grad(out, (q, k, v), dout)]


@pytest.mark.parametrize("layout", ["heads first", "part of a row", "expanded batch", "odd base", "odd stride", "expanded gradient"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_layouts(layout, d):
    B, S, H, Hk, window, sinks = 2, 333, 4, 2, 50, 3
    q, k, v, dout = (x.detach() for x in tensors(B, S, S, H, Hk, d, torch.bfloat16))

    def lay(x):
        if layout == "heads first":
            return x.transpose(1, 2).contiguous().transpose(1, 2)
        if layout == "part of a row":
            return torch.cat([x, x], -1)[..., d:]
        if layout == "expanded batch":
            return x[:1].expand_as(x)
        if layout == "odd base":
            return torch.cat([x.flatten()[:1], x.flatten()])[1:].view(x.shape)
        if layout == "odd stride":
            return torch.cat([x, x[..., :3]], -1)[..., :d]
        return x

    leaves = [lay(x).detach().requires_grad_() for x in (q, k, v)]
    g = dout[:, :1, :, :1].expand_as(dout) if layout == "expanded gradient" else lay(dout)
    out = window_func(*leaves, window, sinks)
    check([out, *torch.autograd.grad(out, leaves, g)], *reference(*leaves, window, sinks, dout=g))


@pytest.mark.parametrize("d", [4, 20, 100, 129, 250])
@pytest.mark.parametrize("masked", [False, True])
def test_other_head_dims_and_lse(d, masked):
    q, k, v, dout = tensors(2, 150, 190, 4, 2, d, torch.float16)
    mask = padding(2, 190) if masked else None
    check(step(q, k, v, dout, 40, 2, attn_mask=mask), *reference(q, k, v, 40, 2, mask, dout=dout))
    out, lse, none = window_func(q, k, v, 40, 2, attn_mask=mask, return_attn_probs=True)
    x = torch.einsum("bqhd,bkhd->bhqk", q.double(), k.double().repeat_interleave(2, 2)) * d ** -0.5
    t, j = torch.arange(150, device="cuda")[:, None] + 40, torch.arange(190, device="cuda")
    seen = ((j <= t) & ((t - j < 40) | (j < 2)))[None, None] & (mask if masked else True)
    want = x.masked_fill(~seen, -torch.inf).logsumexp(-1)
    rows = seen.any(-1).expand_as(want)
    assert lse.shape == (2, 4, 150) and none.numel() == 0
    # scores are exact products summed up in 32 bits, the sum of exponentials has 2^-17 relative
    assert (lse.double() - want)[rows].abs().max() <= 3e-5
    assert bool((lse[~rows] == torch.inf).all()) or bool((lse[~rows] == -torch.inf).all())
    check([out, *torch.autograd.grad(out, (q, k, v), dout)], *reference(q, k, v, 40, 2, mask, dout=dout))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("heads", [None, "one", "kv", "query"])
@pytest.mark.parametrize("B,Sk,H,Hk,d,window,sinks", [(1, 1, 2, 1, 64, 1, 0), (2, 700, 4, 2, 128, 1, 0), (3, 700, 4, 2, 128, 300, 4), (1, 9000, 16, 1, 64, 4096, 130),
                                                     (2, 20000, 2, 2, 96, 15000, 3), (2, 300, 2, 1, 256, 20, 270), (3, 333, 6, 2, 72, 40, 293), (1, 500, 2, 1, 128, 499, 0)])
def test_single_tokens(B, Sk, H, Hk, d, window, sinks, heads, dtype):
    """One query of each head, at the last position, from training and while serving."""
    q, k, v, dout = tensors(B, 1, Sk, H, Hk, d, dtype)
    mask = None if heads is None else padding(B, Sk, {"one": 1, "kv": Hk, "query": H}[heads])
    if d > 128 and heads == "query":
        q, k, v = (x.detach() for x in (q, k, v))
        want, off = reference(q, k, v, window, sinks, mask)
        check([window_func(q, k, v, window, sinks, attn_mask=mask)], want, off)
        return
    check(step(q, k, v, dout, window, sinks, attn_mask=mask), *reference(q, k, v, window, sinks, mask, dout=dout))
    with torch.no_grad():
        out, lse, _ = window_func(q, k, v, window, sinks, attn_mask=mask, return_attn_probs=True)
        assert torch.equal(out, window_func(q, k, v, window, sinks, attn_mask=mask))
        j = torch.arange(Sk, device="cuda")
        seen = ((Sk - 1 - j < window) | (j < sinks))[None, None]
        if mask is not None:
            seen = seen & mask[:, :, 0].repeat_interleave(H // mask.shape[1], 1)
        x = torch.einsum("bhd,bkhd->bhk", q[:, 0].double(), k.double().repeat_interleave(H // Hk, 2)) * d ** -0.5
        want = x.masked_fill(~seen, -torch.inf).logsumexp(-1)
        some = seen.any(-1).expand_as(want)
        assert (lse[:, :, 0].double() - want)[some].abs().max() <= 3e-5 and bool((lse[:, :, 0][~some] == torch.inf).all())


@pytest.mark.parametrize("scale", [0.0, 0.3, 3.0])
def test_scales(scale):
    q, k, v, dout = tensors(1, 200, 200, 2, 1, 64, torch.bfloat16)
    check(step(q, k, v, dout, 30, 4, softmax_scale=scale), *reference(q, k, v, 30, 4, scale=scale, dout=dout))


def test_masks_that_are_broadcast_and_the_same_tensor_three_times():
    B, S, window, sinks = 3, 260, 33, 5
    q, k, v, dout = tensors(B, S, S, 4, 2, 64, torch.bfloat16)
    one = padding(1, S)
    for mask in (one, one.expand(B, 1, 1, S), one[..., :1], torch.ones((B, 1, 1, 1), dtype=torch.bool, device="cuda"), one.expand(B, 4, 1, S)):
        check(step(q, k, v, dout, window, sinks, attn_mask=mask), *reference(q, k, v, window, sinks, mask.expand(B, mask.shape[1], 1, S), dout=dout))
    x = q.detach()[:, :, :2].contiguous().requires_grad_()
    dx = dout[:, :, :2]
    (got,) = torch.autograd.grad(window_func(x, x, x, window, sinks), x, dx)
    parts, off = reference(x, x, x, window, sinks, dout=dx)
    u = torch.finfo(torch.bfloat16).eps / 2
    want = parts[1] + parts[2] + parts[3]
    # the three are added in the type, one after the other
    assert bool(((got.double() - want).abs() <= off[1] + off[2] + off[3] + 2 * u * (parts[1].abs() + parts[2].abs() + parts[3].abs()) + 1e-6).all())


def test_some_of_the_gradients():
    q, k, v, dout = tensors(1, 300, 300, 4, 2, 128, torch.bfloat16)
    want, off = reference(q, k, v, 64, 4, dout=dout)
    for i in range(3):
        leaves = [x.detach().requires_grad_(j == i) for j, x in enumerate((q, k, v))]
        out = window_func(*leaves, 64, 4)
        check([out, torch.autograd.grad(out, leaves[i], dout)[0]], [want[0], want[i + 1]], [off[0], off[i + 1]])
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            out = window_func(q, k, v, 64, 4)
            assert not out.requires_grad
            check([out], want, off)


@pytest.mark.parametrize("shape,window,sinks", [((1, 600, 600, 4, 2, 64), 100, 4), ((1, 300, 300, 2, 1, 256), 40, 3)], ids=str)
def test_gradients_against_differences(shape, window, sinks):
    """Along a direction e the gradients' product with e is the derivative of sum(out * dout), which the definition's central difference is
    off by less than 1e-6 from at this step."""
    q, k, v, dout = tensors(*shape, torch.bfloat16)
    got = step(q, k, v, dout, window, sinks)[1:]
    _, off = reference(q, k, v, window, sinks, dout=dout)
    h, g = 1e-4, torch.Generator(device="cuda").manual_seed(5)
    for i in range(3):
        e = torch.randn(got[i].shape, generator=g, device="cuda", dtype=torch.float64) * (torch.rand(got[i].shape, generator=g, device="cuda") < 0.01)
        moved = [[x.detach().double() + (sign * h * e if j == i else 0) for j, x in enumerate((q, k, v))] for sign in (1, -1)]
        outs = [definition(*x, window, sinks) for x in moved]
        difference = ((outs[0] - outs[1]) * dout.double()).sum() / (2 * h)
        assert (got[i].double() * e).sum().sub(difference).abs() <= (off[i + 1] * e.abs()).sum() + 1e-4


def definition(q, k, v, window, sinks):
    Sq, Sk = q.shape[1], k.shape[1]
    t, j = torch.arange(Sq, device="cuda")[:, None] + Sk - Sq, torch.arange(Sk, device="cuda")
    k, v = (x.repeat_interleave(q.shape[2] // x.shape[2], 2) for x in (k, v))
    x = torch.einsum("bqhd,bkhd->bhqk", q, k) * q.shape[-1] ** -0.5
    x = x.masked_fill(~((j <= t) & ((t - j < window) | (j < sinks))), -torch.inf)
    return torch.einsum("bhqk,bkhd->bqhd", x.softmax(-1), v)


def test_a_window_is_part_of_the_plain_call():
    """A window that covers all keys is causal attention; one that does so but for its last key is that in all rows but the last ones."""
    q, k, v, dout = tensors(2, 400, 400, 4, 2, 64, torch.bfloat16)
    out = fsa.flash_sparse_attn_func(q, k, v, is_causal=True)
    plain = [out, *torch.autograd.grad(out, (q, k, v), dout)]
    for args in ((400, 0), (2 ** 31 - 1, 2 ** 31 - 1), (1, 399)):
        for x, y in zip(step(q, k, v, dout, *args), plain):
            assert torch.equal(x, y)
    assert torch.equal(window_func(q, k, v, 399, 0)[:, :256], plain[0][:, :256])


def test_same_bits_every_time():
    """Sums are formed in a fixed order: dense and packed, alone and beside other launches."""
    q, k, v, dout = tensors(1, 5000, 5000, 8, 2, 64, torch.bfloat16)
    cu = torch.tensor([0, 4000, 4001, 5000], dtype=torch.int32, device="cuda")
    qp, kp, vp = (x[0].detach().requires_grad_() for x in (q, k, v))

    def run():
        out = varlen_func(qp, kp, vp, cu, cu, 4000, 4000, 130, 4)
        return step(q, k, v, dout, 300, 140) + [out, *torch.autograd.grad(out, (qp, kp, vp), dout[0])]

    want = run()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    runs = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                runs.append(run())
    torch.cuda.synchronize()
    for r in runs:
        for x, y in zip(r, want):
            assert torch.equal(x, y)


@pytest.mark.parametrize("d,masked", [(64, False), (128, True), (256, True)])
def test_captured_beside_an_eager_graph_of_the_same_leaves(d, masked):
    # (autograd joins a leaf's gradient with the stream on which the leaf was first used, so that is the stream to capture on)
    q, k, v, dout = tensors(2, 500, 500, 4, 2, d, torch.bfloat16)
    mask = padding(2, 500) if masked else None
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = window_func(q, k, v, 70, 4, attn_mask=mask)  # an eager graph that stays
        step(q, k, v, dout, 70, 4, attn_mask=mask)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            got = step(q, k, v, dout, 70, 4, attn_mask=mask)
    for seed in (7, 8):
        fresh = tensors(2, 500, 500, 4, 2, d, torch.bfloat16, seed=seed)
        with torch.no_grad():
            for x, y in zip((q, k, v, dout), fresh):
                x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        check(got, *reference(*fresh[:3], 70, 4, mask, dout=fresh[3]))
    del alive


@pytest.mark.parametrize("masked", [False, True])
def test_compiled(masked):
    q, k, v, dout = tensors(2, 200, 200, 4, 2, 64, torch.bfloat16)
    mask = padding(2, 200) if masked else None
    want = step(q, k, v, dout, 40, 3, attn_mask=mask)
    torch._dynamo.reset()
    fn = torch.compile(lambda q, k, v: window_func(q, k, v, 40, 3, attn_mask=mask), backend="aot_eager", fullgraph=True)
    out = fn(q, k, v)
    for x, y in zip([out, *torch.autograd.grad(out, (q, k, v), dout)], want):
        assert torch.equal(x, y)


def test_custom_operators():
    q, k, v, dout = (x.detach() for x in tensors(2, 64, 64, 4, 2, 64, torch.bfloat16))
    mask = torch.nn.functional.pad(padding(2, 64), [0, 64])  # as the operators take it
    ops = torch.ops.flash_sparse_attn
    out, lse = ops._window_forward(q, k, v, mask, 0.125, 9, 2)
    torch.library.opcheck(ops._window_forward, (q, k, v, mask, 0.125, 9, 2))
    torch.library.opcheck(ops._window_backward, (dout, q, k, v, mask, out, lse, 0.125, 9, 2))


@pytest.mark.parametrize("masked", [False, True])
def test_nothing_to_do(masked):
    for B, Sq, Sk in ((0, 5, 5), (2, 0, 5), (2, 5, 0), (1, 0, 0)):
        q, k, v, dout = tensors(B, Sq, Sk, 4, 2, 64, torch.bfloat16)
        mask = torch.ones((1, 1, 1, Sk), dtype=torch.bool, device="cuda") if masked else None
        with pytest.raises(RuntimeError):  # as the call without a window
            step(q, k, v, dout, 3, 1, attn_mask=mask)
    cu = torch.zeros(3, dtype=torch.int32, device="cuda")
    q, k, v, dout = (x[0].detach().requires_grad_(i < 3) for i, x in enumerate(tensors(1, 0, 0, 4, 2, 64, torch.bfloat16)))
    out = varlen_func(q, k, v, cu, cu, 0, 0, 3, 1)
    assert out.shape == (0, 4, 64) and torch.autograd.grad(out, q, dout)[0].shape == q.shape


def test_not_a_number_in_hidden_rows_of_the_mask():
    """What the mask and the window hide adds nothing, whatever finite numbers it holds."""
    q, k, v, dout = tensors(1, 400, 400, 4, 2, 64, torch.bfloat16)
    mask = padding(1, 400)
    with torch.no_grad():
        hidden = ~mask[0, 0, 0]
        k[:, hidden], v[:, hidden] = 1e30, -1e30
    got = step(q, k, v, dout, 60, 4, attn_mask=mask)
    with torch.no_grad():
        k[:, hidden], v[:, hidden] = 0, 0
    want = step(q, k, v, dout, 60, 4, attn_mask=mask)
    for x, y in zip(got, want):
        assert bool(x.isfinite().all())
    check(got, *reference(q, k, v, 60, 4, mask, dout=dout))
    assert torch.equal(got[0], want[0])


@pytest.mark.parametrize("d,H,Hk,S,window,sinks", [(64, 64, 64, 4500, 40, 4200), (256, 24, 24, 4500, 40, 4200), (64, 4, 2, 2700, 5, 2600)])
def test_many_sinks(d, H, Hk, S, window, sinks):
    """So many that the parts of the queries beyond the window are larger ones; compared head by head."""
    q, k, v, dout = tensors(1, S, S, H, Hk, d, torch.bfloat16)
    got = step(q, k, v, dout, window, sinks)
    G = H // Hk
    for hk in range(0, Hk, max(1, Hk // 5)):
        a, b = slice(hk * G, hk * G + G), slice(hk, hk + 1)
        check([got[0][:, :, a], got[1][:, :, a], got[2][:, :, b], got[3][:, :, b]],
              *reference(q[:, :, a], k[:, :, b], v[:, :, b], window, sinks, dout=dout[:, :, a]))


@pytest.mark.parametrize("what", ["lse", "d 256", "d 20", "another path"])
def test_packed_sequences_one_by_one(what):
    """Calls that the launch for all sequences does not take."""
    d = {"d 256": 256, "d 20": 20}.get(what, 64)
    lengths, window, sinks = [130, 0, 1, 300], 50, 3
    cu_list = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    cu = torch.tensor(cu_list, dtype=torch.int32, device="cuda")
    q, k, v, dout = (x[0].detach().requires_grad_(i < 3) for i, x in enumerate(tensors(1, cu_list[-1], cu_list[-1], 4, 2, d, torch.bfloat16)))
    try:
        if what == "another path":
            set_kernel_path("tcgen05")
        out = varlen_func(q, k, v, cu, cu, 300, 300, window, sinks, return_attn_probs=what == "lse")
    finally:
        set_kernel_path("auto")
    if what == "lse":
        out = out[0]
    check([out, *torch.autograd.grad(out, (q, k, v), dout)], *packed_reference(q, k, v, cu_list, cu_list, window, sinks, dout))


def test_boundaries_that_do_not_ascend_stay_within_the_tensors():
    T = 900
    q, k, v, dout = (x[0].detach().requires_grad_(i < 3) for i, x in enumerate(tensors(1, T, T, 4, 2, 64, torch.bfloat16)))

    def run(bounds):
        cu = torch.tensor(bounds, dtype=torch.int32, device="cuda")
        out = varlen_func(q, k, v, cu, cu, T, T, 60, 70)
        return [out, *torch.autograd.grad(out, (q, k, v), dout)]

    want = run([0, 400, 410, T])
    for bad in ([0, 500, 100, T], [T, 0, 500, 20], [-5, 700, 2 ** 31 - 1, 3], [300, 200, 100, 0], [0, 0, 0, -7]):
        run(bad)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(run([0, 400, 410, T]), want))


def test_refusals():
    q, k, v, dout = (x.detach() for x in tensors(2, 40, 40, 4, 2, 64, torch.bfloat16))
    mask = torch.ones((2, 1, 1, 40), dtype=torch.bool, device="cuda")
    window_func(q, k, v, 8, 1, attn_mask=mask)
    errors = (RuntimeError, ValueError, NotImplementedError, IndexError, AssertionError, TypeError)
    for bad in (dict(query=q.float()), dict(query=q.half()), dict(key=k.cpu()), dict(query=q[0]), dict(key=k[:1]), dict(value=v[:, :39]),
                dict(value=v[..., :32]), dict(query=q[:, :, :3]), dict(attn_mask=mask.cpu()), dict(attn_mask=mask[:, :, 0]),
                dict(attn_mask=mask.expand(2, 3, 1, 40)), dict(attn_mask=mask[..., :30]), dict(attn_mask=mask.expand(2, 1, 40, 40)),
                dict(attn_mask=mask.float()), dict(sliding_window=0), dict(sink_tokens=-1), dict(softmax_scale=-0.1),
                dict(softmax_scale=float("nan")), dict(query=q[:0], key=k[:0], value=v[:0]), dict(query=q[:, :0]),
                dict(value=v.cpu())):
        with pytest.raises(errors):
            print({n: getattr(x, "shape", x) for n, x in bad.items()})
            window_func(**{**dict(query=q, key=k, value=v, sliding_window=8, sink_tokens=1), **bad})
    wide = [torch.zeros((1, 20, h, 264), dtype=torch.bfloat16, device="cuda") for h in (2, 1, 1)]
    with pytest.raises(errors):
        window_func(*wide, 8)
    cu = torch.tensor([0, 30, 80], dtype=torch.int32, device="cuda")
    qp, kp, vp = q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1)
    varlen_func(qp, kp, vp, cu, cu, 50, 50, 8, 1)
    for bad in (dict(cu_seqlens_q=cu.float()), dict(cu_seqlens_k=cu[:2]), dict(query=qp.float()), dict(key=kp[:, :1].expand(80, 3, 64)),
                dict(query=q), dict(value=vp[:50]), dict(cu_seqlens_q=cu[:0], cu_seqlens_k=cu[:0]), dict(sliding_window=0),
                dict(softmax_scale=-1.0)):
        with pytest.raises(errors):
            print({n: getattr(x, "shape", x) for n, x in bad.items()})
            varlen_func(**{**dict(query=qp, key=kp, value=vp, cu_seqlens_q=cu, cu_seqlens_k=cu, max_seqlen_q=50, max_seqlen_k=50,
                                  sliding_window=8, sink_tokens=1), **bad})
    try:
        set_kernel_path("simt")
        with pytest.raises(errors):
            window_func(q, k, v, 8, 1)
    finally:
        set_kernel_path("auto")


def test_packed_single_tokens():
    """A batch of one query each, over keys of its own length."""
    keys, window, sinks = [500, 1, 90, 3000], 64, 3
    cu_q, cu_k = list(range(5)), [sum(keys[:i]) for i in range(5)]
    q, k, v, dout = (x[0].detach().requires_grad_(i < 3) for i, x in enumerate(tensors(1, 4, cu_k[-1], 4, 2, 64, torch.bfloat16)))
    cu = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (cu_q, cu_k)]
    out = varlen_func(q, k, v, *cu, 1, max(keys), window, sinks)
    check([out, *torch.autograd.grad(out, (q, k, v), dout)], *packed_reference(q, k, v, cu_q, cu_k, window, sinks, dout))
