"""C entry points of sliding windows and of the verification of drafts: wrong parameters are refused with a status, and workspaces are
sized, before a device is touched (no GPU needed). The Python entry points refuse what is wrong in itself."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

import flash_sparse_attn as fsa
from flash_sparse_attn import _lib
from test_cabi_cache import ADDR, HEADER, ROOT, Attention, cache, call, fill, mirror

Verify = mirror("fdma_verify_params", {})
BAD, UNSUPPORTED, WORKSPACE = -1, -2, -3


def entry(name, result):
    fn = getattr(_lib.load(), name)
    fn.restype = result
    fn.argtypes = [ctypes.c_void_p, ctypes.c_int32, ctypes.c_int32] + ([ctypes.c_int32] if result is ctypes.c_size_t else
                                                                        [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int32, ctypes.c_void_p])
    return fn


def params(cls, **change):
    p = cls()
    f = p.f if cls is _lib.BwdParams else p
    for x in ("q", "k", "v", "out", "lse"):
        setattr(f, x, ADDR)
    f.b, f.seqlen_q, f.seqlen_k, f.h, f.h_k, f.d, f.is_causal, f.dtype, f.softmax_scale = 1, 500, 500, 4, 2, 64, 1, _lib.FDMA_BF16, 0.125
    for x, h in (("q", 4), ("k", 2), ("v", 2), ("o", 4)):
        setattr(f, f"{x}_row_stride", h * 64), setattr(f, f"{x}_head_stride", 64), setattr(f, f"{x}_batch_stride", 500 * h * 64)
    if cls is _lib.BwdParams:
        for x in ("dout", "dq", "dk", "dv"):
            setattr(p, x, ADDR)
        for x, h in (("do", 4), ("dq", 4), ("dk", 2), ("dv", 2)):
            setattr(p, f"{x}_row_stride", h * 64), setattr(p, f"{x}_head_stride", 64), setattr(p, f"{x}_batch_stride", 500 * h * 64)
    for k, v in change.items():
        setattr(f, k, v)
    return p


@pytest.mark.parametrize("cls,name", [(_lib.FwdParams, "fdma_fwd_window"), (_lib.BwdParams, "fdma_bwd_window")])
@pytest.mark.parametrize("args,change,status", [
    ((0, 0, None, None, 0), {}, BAD), ((-1, 0, None, None, 0), {}, BAD), ((8, -1, None, None, 0), {}, BAD), ((8, 0, None, None, -1), {}, BAD),
    ((8, 0, ADDR, None, 1), {}, BAD), ((8, 0, None, ADDR, 1), {}, BAD), ((8, 0, ADDR, ADDR, 0), {}, BAD), ((8, 0, None, None, 0), dict(is_causal=0), BAD),
    ((8, 0, None, None, 0), dict(q=None), BAD), ((8, 0, None, None, 0), dict(h=3), BAD), ((8, 0, None, None, 0), dict(d=60), UNSUPPORTED),
    ((8, 0, None, None, 0), dict(d=264), UNSUPPORTED), ((8, 0, None, None, 0), dict(dtype=2), UNSUPPORTED),
    ((8, 0, None, None, 0), dict(path=_lib.PATH_SIMT), UNSUPPORTED), ((8, 0, None, None, 0), dict(mask=ADDR, mask_row_stride=512, h_mask=1), UNSUPPORTED),
    ((8, 0, ADDR, ADDR, 2), dict(mask=ADDR, h_mask=1), UNSUPPORTED),
], ids=str)
def test_attention_refuses(cls, name, args, change, status):
    p = params(cls, **change)
    assert entry(name, ctypes.c_int)(ctypes.byref(p), *args, None) == status
    assert entry(name, ctypes.c_int)(None, 8, 0, None, None, 0, None) == BAD


def test_workspace_of_the_forward_pass():
    size = entry("fdma_fwd_window_workspace_bytes", ctypes.c_size_t)
    assert size(None, 8, 0, 0) == 0
    assert size(ctypes.byref(params(_lib.FwdParams)), 8, 4, 0) == 0  # several queries
    one = params(_lib.FwdParams, seqlen_q=1, seqlen_k=1 << 20)
    for window, sinks, n in ((0, 0, 0), (8, -1, 0), (8, 0, -1), (8, 4, 1)):
        assert size(ctypes.byref(one), window, sinks, n) == 0
    assert size(ctypes.byref(one), 1 << 20, 0, 0) > 0  # the keys are split over more CTAs than a cluster has


def test_workspace_of_the_backward_pass():
    size = entry("fdma_bwd_window_workspace_bytes", ctypes.c_size_t)
    assert size(None, 8, 0, 0) == 0
    p = params(_lib.BwdParams)
    for window, sinks, n in ((0, 0, 0), (8, -1, 0), (8, 0, -1)):
        assert size(ctypes.byref(p), window, sinks, n) == 0
    without, some = size(ctypes.byref(p), 8, 0, 0), size(ctypes.byref(p), 8, 5, 0)
    assert 0 < without < some  # the sinks' gradients are summed up from parts
    assert size(ctypes.byref(p), 8, 500, 0) == size(ctypes.byref(p), 8, 2 ** 31 - 1, 0)
    # a million keys that are all sinks: the parts' sums stay within a few times the gradients' own fp32
    p = params(_lib.BwdParams, seqlen_q=2 ** 20, seqlen_k=2 ** 20)
    rows = 2 ** 20 * 64 * 4
    assert size(ctypes.byref(p), 8, 2 ** 20, 0) < (3 * 4 + 2 * 2 * 18) * rows


@pytest.mark.parametrize("change,status", [
    (dict(logits=None), BAD), (dict(token_ids=None), BAD), (dict(uniforms=None), BAD), (dict(cu_seqlens=None), BAD), (dict(lengths=None), BAD),
    (dict(accepted=None), BAD), (dict(next_tokens=None), BAD), (dict(lengths_out=None), BAD), (dict(requests=-1), BAD),
    (dict(tokens=-1), BAD), (dict(vocab=0), BAD), (dict(id_bits=16), UNSUPPORTED), (dict(dtype=9), UNSUPPORTED), (dict(draft_probs=ADDR, probs_dtype=9), UNSUPPORTED),
    (dict(workspace=None), WORKSPACE), (dict(workspace_bytes=0), WORKSPACE)], ids=str)
def test_drafts_refuse(change, status):
    p = fill(Verify(), ["logits", "token_ids", "uniforms", "cu_seqlens", "lengths", "granted", "accepted", "next_tokens", "lengths_out", "workspace"],
             requests=2, tokens=5, vocab=1000, logits_row_stride=1000, probs_row_stride=1000, id_bits=64, temperature=1.0, workspace_bytes=1 << 40)
    for k, v in change.items():
        setattr(p, k, v)
    assert call("fdma_verify_drafts", p) == status
    assert call("fdma_verify_drafts", None) == BAD


def test_workspace_of_drafts():
    fn = _lib.load().fdma_verify_drafts_workspace_bytes
    fn.restype, fn.argtypes = ctypes.c_size_t, [ctypes.c_void_p]
    assert fn(None) == 0
    p = fill(Verify(), [], requests=2, tokens=5, vocab=1000, id_bits=64)
    assert 0 < fn(ctypes.byref(p)) < 1 << 20


@pytest.mark.parametrize("change,status", [(dict(window=-1), BAD), (dict(window=8, sinks=-1), BAD), (dict(window=0, sinks=2), BAD), (dict(window=8), BAD),
                                           (dict(window=8, is_causal=1), WORKSPACE)])
def test_cache_attention_refuses(change, status):
    p = fill(Attention(), ["query", "out"], c=cache(requests=500), h=1, max_seqlen_q=1, max_seqlen_k=1, softmax_scale=1.0, **change)
    assert call("fdma_cache_attention", p) == status


def test_layout_of_the_parameter_block(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no gcc")
    src = tmp_path / "size.c"
    src.write_text('#include <stdio.h>\n#include "fdma.h"\nint main(void) { printf("%zu", sizeof(fdma_verify_params)); return 0; }\n')
    subprocess.run([gcc, "-I", os.path.dirname(HEADER), str(src), "-o", str(tmp_path / "size")], check=True)
    assert ctypes.sizeof(Verify) == int(subprocess.run([str(tmp_path / "size")], check=True, capture_output=True, text=True).stdout)
    assert os.path.isdir(ROOT)


@pytest.mark.parametrize("error,window,sinks", [(TypeError, 4.0, 0), (TypeError, True, 0), (TypeError, None, 0), (TypeError, 4, 1.0), (TypeError, 4, None),
                                               (ValueError, 0, 0), (ValueError, -1, 0), (ValueError, 2 ** 31, 0), (ValueError, 4, -1), (ValueError, 4, 2 ** 31)])
def test_python_refuses_windows(error, window, sinks):
    q = torch.zeros((1, 8, 2, 64), dtype=torch.bfloat16)
    cu = torch.tensor([0, 8], dtype=torch.int32)
    with pytest.raises(error):
        fsa.flash_sparse_attn_window_func(q, q, q, window, sinks)
    with pytest.raises(error):
        fsa.flash_sparse_attn_window_varlen_func(q[0], q[0], q[0], cu, cu, 8, 8, window, sinks)


def test_python_refuses_masks():
    q = torch.zeros((1, 8, 4, 192), dtype=torch.bfloat16)
    k = q[:, :, :2]
    for mask in (torch.ones((1, 1, 1, 8)), torch.ones((8,), dtype=torch.bool), 3):
        with pytest.raises(RuntimeError):
            fsa.flash_sparse_attn_window_func(q, k, k, 4, attn_mask=mask)
    for mask, grad in ((torch.ones((1, 1, 8, 8), dtype=torch.bool), False), (torch.ones((1, 4, 1, 8), dtype=torch.bool), True)):
        with pytest.raises(NotImplementedError, match="mask"):
            fsa.flash_sparse_attn_window_func(q.clone().requires_grad_(grad), k, k, 4, attn_mask=mask)
