"""Verification steps in which every request is refused or has no tokens, while there are rows: nothing is accepted, and the call has ended when
what follows it runs, so that its scratch can be used again."""
import pytest
import torch

import flash_sparse_attn as fsa
from test_gpu_cache import dev, ints  # noqa: F401
from test_gpu_drafts import check, drafts, plan

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["refused", "no tokens"])
@pytest.mark.parametrize("T,R,V", [(1, 1, 7), (6, 2, 1000), (64, 8, 131072), (512, 64, 32000)])
def test_nobody(dev, T, R, V, kind):  # noqa: F811
    ids, logits, u, q = drafts(dev, [T], V, torch.bfloat16, torch.float32, 1)
    new = [T // R] * R if kind == "refused" else [0] * R
    step = plan(dev, new, granted=[kind != "refused"] * R)
    check(dev, step, ids, logits, u, q)
    check(dev, step, ids, logits, u, None, 0.0)


@pytest.mark.parametrize("captured", [False, True])
def test_scratch_used_again(dev, captured):  # noqa: F811
    """Work right behind the call fills blocks of every size that its scratch can have: what it writes stays."""
    T, R, V = 512, 64, 100000
    ids, logits, u, _ = drafts(dev, [T], V, torch.bfloat16, None, 2)
    step = plan(dev, [T // R] * R, granted=[False] * R)

    def work():
        done = fsa.verify_drafts(step, ids, logits, u)
        return done, [torch.full((n,), 77, dtype=torch.uint8, device=dev) for n in (1 << k for k in range(9, 25))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        if captured:
            work()
            graph = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(graph, stream=side):
                done, filled = work()
        for _ in range(3):
            if captured:
                graph.replay()
            else:
                done, filled = work()
            torch.cuda.synchronize()
            assert all(bool((x == 77).all()) for x in filled)
            assert done.next_tokens.tolist() == [-1] * R and done.accepted.tolist() == [0] * R and torch.equal(done.lengths, step.lengths)
    if captured:  # the same graph, once they are granted
        step.granted.fill_(True)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(done, fsa.verify_drafts(step, ids, logits, u)))
        assert all(bool((x == 77).all()) for x in filled)
