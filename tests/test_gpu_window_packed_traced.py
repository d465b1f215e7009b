"""Packed sequences with a window under torch.compile: one graph, the same bits as without it."""
import pytest
import torch

import flash_sparse_attn as fsa
from test_gpu_window import check, packed_reference, tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 100, 128])
@pytest.mark.parametrize("lengths_q,lengths_k", [([300, 1, 77], None), ([100, 50, 700], [30, 50, 900]), ([500], None)])
def test_compiled(lengths_q, lengths_k, d):
    lengths_k = lengths_k or lengths_q
    cu_q, cu_k = ([sum(x[:i]) for i in range(len(x) + 1)] for x in (lengths_q, lengths_k))
    q, k, v, dout = (x[0].detach().requires_grad_(i < 3) for i, x in enumerate(tensors(1, cu_q[-1], cu_k[-1], 4, 2, d, torch.bfloat16)))
    cu = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (cu_q, cu_k)]
    torch._dynamo.reset()

    def call(q, k, v, cu_q, cu_k):
        return fsa.flash_sparse_attn_window_varlen_func(q, k, v, cu_q, cu_k, max(lengths_q), max(lengths_k), 40, 3)

    fn = torch.compile(call, backend="aot_eager", fullgraph=True)
    out = fn(q, k, v, *cu)
    got = [out, *torch.autograd.grad(out, (q, k, v), dout)]
    check(got, *packed_reference(q, k, v, cu_q, cu_k, 40, 3, dout))
    if d % 8 == 0:
        out = call(q, k, v, *cu)
        for x, y in zip(got, [out, *torch.autograd.grad(out, (q, k, v), dout)]):
            assert torch.equal(x, y)
    with torch.no_grad():
        assert torch.equal(fn(q, k, v, *cu), got[0])


def test_boundaries_that_are_filled_again_before_the_backward():
    q, k, v, dout = (x[0].detach().requires_grad_(i < 3) for i, x in enumerate(tensors(1, 400, 400, 4, 2, 64, torch.bfloat16)))
    cu = torch.tensor([0, 150, 400], dtype=torch.int32, device="cuda")
    torch._dynamo.reset()
    fn = torch.compile(lambda q, k, v, cu: fsa.flash_sparse_attn_window_varlen_func(q, k, v, cu, cu, 250, 250, 30, 2), backend="aot_eager", fullgraph=True)
    out = fn(q, k, v, cu)
    cu.copy_(torch.tensor([0, 10, 20]))
    got = [out, *torch.autograd.grad(out, (q, k, v), dout)]
    check(got, *packed_reference(q, k, v, [0, 150, 400], [0, 150, 400], 30, 2, dout))


def test_custom_operators():
    q, k, v, dout = (x[0].detach() for x in tensors(1, 130, 130, 4, 2, 64, torch.bfloat16))
    cu = torch.tensor([0, 50, 130], dtype=torch.int32, device="cuda")
    ops = torch.ops.flash_sparse_attn
    out, lse, both = ops._window_varlen_forward(q, k, v, cu, cu, 0.125, 9, 2)
    torch.library.opcheck(ops._window_varlen_forward, (q, k, v, cu, cu, 0.125, 9, 2))
    torch.library.opcheck(ops._window_varlen_backward, (dout, q, k, v, both, out, lse, 0.125, 9, 2))
    for bad in (cu.long(), cu[None], cu[:1], cu.cpu()):
        with pytest.raises(RuntimeError):
            ops._window_varlen_forward(q, k, v, bad, bad, 0.125, 9, 2)
    with pytest.raises(RuntimeError):
        ops._window_varlen_forward(q, k[:, :, :32], v, cu, cu, 0.125, 9, 2)
