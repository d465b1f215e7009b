"""The documentation's examples of rotary positions and of serving from the 8-bit cache run as they are written."""
import glob
import os
import re

import pytest
import torch

import flash_sparse_attn as fsa

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def examples(call):
    """Python blocks of the documents that make a call."""
    texts = [open(f).read() for f in sorted(glob.glob(os.path.join(ROOT, "*.md")))]
    return [b for t in texts for b in re.findall(r"```python\n(.*?)```", t, flags=re.S) if call in b]


class Layer:
    def __init__(self, H, Hk, d, dev):
        self.H, self.Hk, self.d = H, Hk, d
        self.w = torch.randn((H * d, (H + 2 * Hk) * d), device=dev, dtype=torch.bfloat16) * (H * d) ** -0.5

    def project(self, x):
        y = (x @ self.w).view(x.shape[0], -1, self.d)
        return y[:, :self.H], y[:, self.H:self.H + self.Hk], y[:, self.H + self.Hk:]

    def rest(self, x, out):
        return x + out.reshape(x.shape)


def test_examples():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    dev, H, Hk, d = torch.device("cuda:0"), 4, 2, 64
    q, k = (torch.randn((2, 9, h, d), device=dev, dtype=torch.bfloat16, requires_grad=True) for h in (H, Hk))
    training = examples("fsa.apply_rotary(")
    assert training
    for text in training:
        names = dict(head_dim=d, q=q, k=k)
        exec(text, names)
        want = fsa.apply_rotary(q, k, fsa.rotary_frequencies(d, device=dev))
        assert torch.equal(names["q"], want[0]) and torch.equal(names["k"], want[1])
        names["q"].sum().backward()
    serving = examples("fsa.block_tables(")
    assert serving
    new = torch.tensor([5, 1, 0] + [0] * 60 + [9], dtype=torch.int32, device=dev)
    for text in serving:
        names = dict(head_dim=d, kv_heads=Hk, layers=[Layer(H, Hk, d, dev) for _ in range(2)], new_lengths=new, total_tokens=15, kept=None,
                     bias=None, n=9, lengths=torch.zeros_like(new), x=torch.randn((15, H * d), device=dev, dtype=torch.bfloat16))
        exec(text, names)
        assert names["out"].shape == (15, H, d) and bool(names["out"].isfinite().all()) and names["step"].granted.all()
        assert names["tables"].free_count.item() == names["tables"].free.numel()
