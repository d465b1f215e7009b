"""Packed sequences with a window, of many and few, short and long ones beside one another: the sinks' gradients, which are summed up in parts of
the queries, and the scratch that takes. Bounds are those of test_gpu_window.py."""
import pytest
import torch

import flash_sparse_attn as fsa
from test_gpu_window import check, packed_reference, tensors

pytestmark = pytest.mark.gpu
varlen_func = fsa.flash_sparse_attn_window_varlen_func


@pytest.mark.parametrize("lengths_q,lengths_k,window,sinks,H,Hk,d", [
    ([30, 500, 7, 0, 260] * 6, None, 20, 300, 4, 2, 64),                # sinks longer than most sequences
    ([200, 300, 129, 130, 131, 1, 500], None, 1, 4096, 4, 2, 128),      # all of them
    ([2500, 5000, 20, 2049, 2048, 2047], None, 100, 140, 4, 1, 64),     # parts of several sequences, two tiles of sinks, sums that are moved
    ([2500, 4500], None, 64, 3, 8, 1, 128),
    ([2500, 300, 4200], [2600, 0, 6000], 200, 5, 2, 2, 64),             # more keys than queries, none
    ([2300, 900, 3000], [400, 900, 2500], 30, 70, 4, 2, 96),            # fewer
    ([300] * 40, None, 150, 2, 4, 2, 64),
    ([1, 2, 3] * 50 + [700], None, 500, 9, 2, 1, 64),
], ids=["many sinks", "all sinks", "parts", "few", "past", "fewer keys", "forty", "tokens"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_gradients(lengths_q, lengths_k, window, sinks, H, Hk, d, dtype):
    lengths_k = lengths_k or lengths_q
    cu_q, cu_k = ([sum(x[:i]) for i in range(len(x) + 1)] for x in (lengths_q, lengths_k))
    q, k, v, dout = (x[0].detach().requires_grad_(i < 3) for i, x in enumerate(tensors(1, cu_q[-1], cu_k[-1], H, Hk, d, dtype)))
    cu = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (cu_q, cu_k)]

    def run():
        out = varlen_func(q, k, v, *cu, max(lengths_q), max(lengths_k), window, sinks)
        return [out, *torch.autograd.grad(out, (q, k, v), dout)]

    got = run()
    check(got, *packed_reference(q, k, v, cu_q, cu_k, window, sinks, dout))
    assert all(torch.equal(x, y) for x, y in zip(got, run()))


def test_scratch():
    n, length, window, sinks = 200, 500, 100, 4096
    T = n * length
    q, k, v, dout = (x[0].detach().requires_grad_(i < 3) for i, x in enumerate(tensors(1, T, T, 16, 8, 128, torch.bfloat16)))
    cu = torch.arange(0, T + 1, length, dtype=torch.int32, device="cuda")
    out = varlen_func(q, k, v, cu, cu, length, length, window, sinks)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    got = torch.autograd.grad(out, (q, k, v), dout)
    assert torch.cuda.max_memory_allocated() - before < 3e9
    a, b = 77 * length, 78 * length  # one of the sequences
    check([x[a:b] for x in (out, *got)], *packed_reference(q[a:b], k[a:b], v[a:b], [0, length], [0, length], window, sinks, dout[a:b]))
