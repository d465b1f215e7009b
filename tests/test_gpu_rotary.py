"""apply_rotary against the rotation in 64 bits: layouts, parts of the head, scalings, far positions, strides, gradients, refusals.

Tolerances. A result is y = a (x1 cos - x2 sin). Its factors are off by at most 4 ulp (2^-22) of sincospif and the products with the
amplitude, its argument by 2^-24 of half a turn, and the sum of two products of magnitude up to a |x| is rounded in 32 bits: 2^-20
of a (|x1| + |x2|) bounds all of it. Then comes one rounding to the type, finfo.eps / 2 of the result."""
import math

import pytest
import torch

import flash_sparse_attn as fsa

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda:0")


def turn(x, positions, inv, amplitude=1.0, interleaved=False, sign=1.0):
    """(result, bound on the magnitude of its terms) in 64 bits; x (..., S, heads, d), positions (..., S)."""
    half = inv.numel()
    x = x.detach().double()
    a = sign * positions.double()[..., None] * inv.double()
    cos, sin = (a.cos() * amplitude)[..., None, :], (a.sin() * amplitude)[..., None, :]
    y, size = x.clone(), x.abs()
    i1 = torch.arange(half, device=x.device) * 2 if interleaved else torch.arange(half, device=x.device)
    i2 = i1 + 1 if interleaved else i1 + half
    x1, x2 = x[..., i1], x[..., i2]
    y[..., i1], y[..., i2] = x1 * cos - x2 * sin, x2 * cos + x1 * sin
    size[..., i1] = size[..., i2] = amplitude * (x1.abs() + x2.abs())
    return y, size


def close(got, want, size):
    tol = torch.finfo(got.dtype).eps / 2 * want.abs() + 2.0 ** -20 * size + torch.finfo(got.dtype).tiny
    bad = (got.double() - want).abs() > tol
    assert not bool(bad.any()), ((got.double() - want).abs() / tol).max().item()


def inv_freq(dim, dev, base=10000.0):
    return base ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=dev) / dim)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,S,H,Hk,d,rd,inter", [
    (1, 1, 1, 1, 64, 64, False), (2, 129, 4, 2, 128, 128, False), (1, 257, 8, 1, 128, 64, True), (3, 33, 5, 5, 96, 32, False),
    (2, 17, 3, 1, 80, 80, True), (1, 65, 2, 2, 20, 6, False), (1, 65, 2, 1, 18, 18, True), (1, 9, 12, 4, 256, 128, False)])
def test_forward_and_gradients(dev, dtype, B, S, H, Hk, d, rd, inter):
    g = torch.Generator(device=dev).manual_seed(S)
    q, k, dq, dk = (torch.randn((B, S, h, d), generator=g, device=dev, dtype=torch.float32).to(dtype) for h in (H, Hk, H, Hk))
    q.requires_grad_(True), k.requires_grad_(True)
    f = fsa.rotary_frequencies(rd, interleaved=inter, device=dev, amplitude=1.25)
    pos = torch.randint(-5000, 100000, (B, S), generator=g, device=dev)
    inv = inv_freq(rd, dev)
    out = fsa.apply_rotary(q, k, f, pos)
    for y, x in zip(out, (q, k)):
        close(y, *turn(x, pos, inv, 1.25, inter))
    for y, x in zip(torch.autograd.grad(out, (q, k), (dq, dk)), (dq, dk)):
        close(y, *turn(x, pos, inv, 1.25, inter, sign=-1.0))


def test_gradient_against_differences(dev):
    g = torch.Generator(device=dev).manual_seed(1)
    q = torch.randn((2, 5, 3, 16), generator=g, device=dev, requires_grad=True)
    k = torch.randn((2, 5, 1, 16), generator=g, device=dev, requires_grad=True)
    wq, wk, vq, vk = (torch.randn(t.shape, generator=g, device=dev) for t in (q, k, q, k))
    f = fsa.rotary_frequencies(8, device=dev)

    def loss(a, b):
        x, y = fsa.apply_rotary(a, b, f)
        return ((x.double() * wq.double()).sum() + (y.double() * wk.double()).sum()).item()

    dq, dk = torch.autograd.grad(fsa.apply_rotary(q, k, f), (q, k), (wq, wk))
    with torch.no_grad():  # linear in (q, k): the difference quotient is exact but for rounding, 2^-20 of 480 terms of size ~ 4
        diff = (loss(q + vq, k + vk) - loss(q - vq, k - vk)) / 2
    slope = (dq.double() * vq.double()).sum().item() + (dk.double() * vk.double()).sum().item()
    assert abs(diff - slope) < 480 * 4 * 2.0 ** -20 * 4


@pytest.mark.parametrize("offset", [0, 10 ** 6 + 3, 2 ** 31 - 70, 2 ** 40])
def test_far_positions(dev, offset):
    """Angles in 64 bits are off by 2^-53 of the position; here positions up to 2^40 are reduced exactly in the oracle too."""
    q = torch.randn((1, 64, 2, 64), device=dev)
    f = fsa.rotary_frequencies(64, device=dev)
    pos = torch.arange(64, device=dev)[None] + offset
    got, none = fsa.apply_rotary(q, None, f, pos)
    assert none is None
    turns = [t % 2 ** 64 for t in f.turns.tolist()]
    frac = torch.tensor([[(p * t % 2 ** 64) / 2.0 ** 64 for t in turns] for p in pos[0].tolist()], dtype=torch.float64, device=dev)
    cos, sin = (2 * math.pi * frac).cos()[None, :, None], (2 * math.pi * frac).sin()[None, :, None]
    x = q.double()
    x1, x2 = x[..., :32], x[..., 32:]
    want = torch.cat((x1 * cos - x2 * sin, x2 * cos + x1 * sin), -1)
    close(got, want, torch.cat((x1.abs() + x2.abs(),) * 2, -1))
    if offset < 10 ** 7:  # and the frequencies are what they should be: 2^-53 of a frequency times the position
        close(got, *turn(q, pos, inv_freq(64, dev)))


@pytest.mark.parametrize("scaling", ["linear", "ntk", "yarn", "bands"])
def test_scaled_frequencies(scaling):
    dim, base, factor, original = 64, 10000.0, 4.0, 2048
    f = fsa.rotary_frequencies(dim, base, scaling, factor, original, device="cpu")
    inv = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    if scaling == "linear":
        want = inv / factor
    elif scaling == "ntk":
        want = (base * factor ** (dim / (dim - 2))) ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    elif scaling == "yarn":
        at = [dim * math.log(original / (n * 2 * math.pi)) / (2 * math.log(base)) for n in (32.0, 1.0)]
        low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), dim - 1)
        keep = torch.tensor([1 - min(max((i - low) / (high - low), 0.0), 1.0) for i in range(dim // 2)], dtype=torch.float64)
        want = inv / factor * (1 - keep) + inv * keep
        assert f.amplitude == pytest.approx(0.1 * math.log(factor) + 1)
    else:
        want = []
        for x in inv.tolist():
            wavelength = 2 * math.pi / x
            if wavelength < original / 4.0:
                want.append(x)
            elif wavelength > original / 1.0:
                want.append(x / factor)
            else:
                s = (original / wavelength - 1.0) / 3.0
                want.append((1 - s) * x / factor + s * x)
        want = torch.tensor(want, dtype=torch.float64)
    got = torch.tensor([t % 2 ** 64 for t in f.turns.tolist()], dtype=torch.float64) / 2.0 ** 64 * 2 * math.pi
    assert torch.allclose(got, want, rtol=1e-14, atol=1e-18)


def test_layouts(dev):
    """Slices of a fused projection, transposed heads, expanded heads, odd offsets, int32 and shared positions, packed tokens."""
    g = torch.Generator(device=dev).manual_seed(2)
    B, S, H, Hk, d = 2, 37, 4, 2, 64
    f, inv = fsa.rotary_frequencies(d, device=dev), inv_freq(d, dev)
    pos = torch.arange(S, device=dev).expand(B, S)
    fused = torch.randn((B, S, (H + 2 * Hk) * d), generator=g, device=dev, dtype=torch.bfloat16)
    odd = torch.randn((B * S * H * d + 1,), generator=g, device=dev, dtype=torch.bfloat16)
    cases = [
        (fused[..., :H * d].view(B, S, H, d), fused[..., H * d:(H + Hk) * d].view(B, S, Hk, d)),
        (torch.randn((B, H, S, d), generator=g, device=dev, dtype=torch.bfloat16).transpose(1, 2),
         torch.randn((B, Hk, S, d), generator=g, device=dev, dtype=torch.bfloat16).transpose(1, 2)),
        (odd[1:].view(B, S, H, d), torch.randn((B, S, 1, d), generator=g, device=dev, dtype=torch.bfloat16).expand(B, S, Hk, d)),
        (torch.randn((B, S, H, 2 * d), generator=g, device=dev, dtype=torch.bfloat16)[..., ::2],
         torch.randn((B, d, S, Hk), generator=g, device=dev, dtype=torch.bfloat16).permute(0, 2, 3, 1)),
    ]
    for q, k in cases:
        for p in (None, pos.to(torch.int32), pos[:1], torch.stack([pos[0], pos[0]], -1)[:, 0]):
            for y, x in zip(fsa.apply_rotary(q, k, f, p), (q, k)):
                assert y.shape == x.shape
                close(y, *turn(x, pos, inv))
        y, _ = fsa.apply_rotary(q[0], k[0], f, pos[0])
        close(y, *turn(q[0], pos[0], inv))


def test_gradients_of_expanded_and_single_inputs(dev):
    f, inv = fsa.rotary_frequencies(64, device=dev), inv_freq(64, dev)
    k = torch.randn((1, 19, 1, 64), device=dev, requires_grad=True)
    q = torch.randn((1, 19, 4, 64), device=dev)
    pos = torch.arange(19, device=dev)[None]
    _, y = fsa.apply_rotary(q, k.expand(1, 19, 4, 64), f)
    w = torch.randn_like(y)
    (dk,) = torch.autograd.grad(y, k, w)
    want, size = turn(w, pos, inv, sign=-1.0)
    tol = 2.0 ** -20 * size.sum(2, keepdim=True) + 4 * 2.0 ** -24 * want.abs().sum(2, keepdim=True)
    assert bool(((dk.double() - want.sum(2, keepdim=True)).abs() <= tol).all())
    # only the query's output is used
    q.requires_grad_(True)
    x, _ = fsa.apply_rotary(q, k, f)
    dq, dk = torch.autograd.grad(x, (q, k), w, allow_unused=True)
    close(dq, *turn(w, pos, inv, sign=-1.0))
    assert dk is None or not bool(dk.any())


def test_second_derivative(dev):
    f = fsa.rotary_frequencies(32, device=dev)
    q = torch.randn((1, 7, 2, 32), device=dev, requires_grad=True)
    w = torch.randn((1, 7, 2, 32), device=dev, requires_grad=True)
    (dq,) = torch.autograd.grad(fsa.apply_rotary(q, None, f)[0], q, w, create_graph=True)
    v = torch.randn_like(dq)
    (dw,) = torch.autograd.grad(dq, w, v)  # dq is the rotation by -angle of w: its gradient turns v forward
    want, size = turn(v, torch.arange(7, device=dev)[None], inv_freq(32, dev))
    close(dw, want, size)


def test_empty_and_infinite(dev):
    f = fsa.rotary_frequencies(64, device=dev)
    q, k = fsa.apply_rotary(torch.empty((2, 0, 3, 64), device=dev), torch.empty((2, 0, 1, 64), device=dev), f)
    assert q.shape == (2, 0, 3, 64) and k.shape == (2, 0, 1, 64)
    x = torch.zeros((1, 3, 1, 64), device=dev)
    x[0, 1, 0, 5], x[0, 2, 0, 40] = math.inf, math.nan
    y, _ = fsa.apply_rotary(x, None, f)
    assert bool(y[0, 0].isfinite().all()) and not bool(y[0, 1, 0, [5, 37]].isfinite().any()) and bool(y[0, 2, 0, [8, 40]].isnan().all())
    others = [i for i in range(64) if i not in (5, 37)]
    assert not bool(y[0, 1, 0, others].any())


def test_graph_of_a_training_step(dev):
    """Forward and backward captured and replayed with new inputs, while an eager graph of the same leaves is alive. (Autograd joins a
    leaf's gradient with the stream on which the leaf was first used, so that is the stream to capture on.)"""
    f = fsa.rotary_frequencies(64, device=dev)
    q = torch.randn((1, 40, 4, 64), device=dev, dtype=torch.bfloat16, requires_grad=True)
    k = torch.randn((1, 40, 2, 64), device=dev, dtype=torch.bfloat16, requires_grad=True)
    w = (torch.randn_like(q), torch.randn_like(k))

    def step():
        out = fsa.apply_rotary(q, k, f)
        return [*out, *torch.autograd.grad(out, (q, k), w)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = fsa.apply_rotary(q, k, f)
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step()
    with torch.no_grad():
        q.copy_(torch.randn_like(q))
        w[0].copy_(torch.randn_like(q))
    graph.replay()
    for a, b in zip(got, step()):
        assert torch.equal(a, b)
    del alive


def test_compiled(dev):
    f = fsa.rotary_frequencies(64, device=dev)
    q = torch.randn((2, 12, 4, 64), device=dev, requires_grad=True)
    k = torch.randn((2, 12, 2, 64), device=dev, requires_grad=True)
    w = (torch.randn_like(q), torch.randn_like(k))

    def fn(q, k):
        return fsa.apply_rotary(q, k, f)

    want = fn(q, k)
    got = torch.compile(fn, backend="aot_eager", fullgraph=True)(q, k)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    for a, b in zip(torch.autograd.grad(got, (q, k), w), torch.autograd.grad(want, (q, k), w)):
        assert torch.equal(a, b)


def test_other_stream(dev):
    f = fsa.rotary_frequencies(64, device=dev)
    q = torch.randn((4, 512, 8, 64), device=dev)
    want, _ = fsa.apply_rotary(q, None, f)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, _ = fsa.apply_rotary(q, None, f)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_refusals(dev):
    f = fsa.rotary_frequencies(64, device=dev)
    q = torch.zeros((2, 8, 4, 64), device=dev, dtype=torch.bfloat16)
    k = torch.zeros((2, 8, 2, 64), device=dev, dtype=torch.bfloat16)
    wrong = [
        (q.cpu(), None, f, None), (q.double(), None, f, None), (q, k.float(), f, None), (q, k[:, :4], f, None), (q, k[..., :32], f, None),
        (q, k.cpu(), f, None), (q[..., :32], None, f, None), (q[0, 0], None, f, None), (q, k, f, torch.zeros((2, 7), device=dev, dtype=torch.int64)),
        (q, k, f, torch.zeros((3, 8), device=dev, dtype=torch.int64)), (q, k, f, torch.zeros((2, 8), device=dev)),
        (q, k, f, torch.zeros((2, 8), dtype=torch.int64)), (q, k, f._replace(turns=f.turns.cpu()), None),
        (q, k, f._replace(turns=f.turns.to(torch.int32)), None)]
    for args in wrong:
        with pytest.raises(RuntimeError):
            fsa.apply_rotary(*args)
