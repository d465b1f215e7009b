"""Gradients of the window calls are the same bits every time, also where the window covers all keys and few queries see many."""
import pytest
import torch

import flash_sparse_attn as fsa
from test_gpu_window import check, reference, tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("deterministic", [None, False, True])
@pytest.mark.parametrize("Sq,Sk,window,sinks", [(512, 8192, 8192, 0), (1024, 16384, 16000, 400), (1024, 16384, 16384, 16384)])
@pytest.mark.parametrize("probs", [False, True])
def test_few_queries_over_many_keys(Sq, Sk, window, sinks, deterministic, probs):
    q, k, v, dout = tensors(1, Sq, Sk, 32, 8, 128, torch.bfloat16)

    def run():
        out = fsa.flash_sparse_attn_window_func(q, k, v, window, sinks, deterministic=deterministic, return_attn_probs=probs)
        out = out[0] if probs else out
        return [out, *torch.autograd.grad(out, (q, k, v), dout)]

    want = run()
    for _ in range(8):
        for x, y in zip(run(), want):
            assert torch.equal(x, y)


@pytest.mark.parametrize("d", [128, 256])
def test_sequence_by_sequence(d):
    """Packed calls that go sequence by sequence, of which some are covered by the window."""
    cu_q, cu_k = (torch.tensor(x, device="cuda") for x in ([0, 512, 700], [0, 8192, 9000]))
    q, k, v, dout = (x[0].detach().requires_grad_(i < 3) for i, x in enumerate(tensors(1, 700, 9000, 16, 4, d, torch.bfloat16)))

    def run():
        out = fsa.flash_sparse_attn_window_varlen_func(q, k, v, cu_q, cu_k, 512, 8192, 8192, 4)
        return [out, *torch.autograd.grad(out, (q, k, v), dout)]

    want = run()
    for _ in range(8):
        for x, y in zip(run(), want):
            assert torch.equal(x, y)


def test_numbers_where_the_window_covers_all_keys():
    q, k, v, dout = tensors(1, 300, 4100, 8, 2, 128, torch.bfloat16)
    out = fsa.flash_sparse_attn_window_func(q, k, v, 4100, 0)
    check([out, *torch.autograd.grad(out, (q, k, v), dout)], *reference(q, k, v, 4100, 0, dout=dout))


@pytest.mark.parametrize("Sq,Sk,window", [(300, 4100, 4100), (300, 4100, 500), (900, 900, 900)])
@pytest.mark.parametrize("power", [-40, 20])
def test_gradients_of_any_size(Sq, Sk, window, power):
    """Times a power of two every number that the backward forms is the same but for its exponent."""
    q, k, v, dout = tensors(1, Sq, Sk, 8, 2, 128, torch.bfloat16)
    want = torch.autograd.grad(fsa.flash_sparse_attn_window_func(q, k, v, window), (q, k, v), dout)
    got = torch.autograd.grad(fsa.flash_sparse_attn_window_func(q, k, v, window), (q, k, v), dout * 2.0 ** power)
    for x, y in zip(got, want):
        assert torch.equal(x, y * 2.0 ** power)


@pytest.mark.parametrize("Sq,Sk,H,Hk,d", [(1, 2048, 4, 1, 64), (256, 2048, 8, 8, 64), (257, 2100, 6, 2, 96), (3, 5000, 4, 2, 128), (130, 9001, 32, 8, 128)])
def test_few_queries(Sq, Sk, H, Hk, d):
    q, k, v, dout = tensors(2, Sq, Sk, H, Hk, d, torch.float16)
    out = fsa.flash_sparse_attn_window_func(q, k, v, Sk - 3, 3)
    check([out, *torch.autograd.grad(out, (q, k, v), dout)], *reference(q, k, v, Sk - 3, 3, dout=dout))
