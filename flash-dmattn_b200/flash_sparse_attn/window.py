"""Attention with a sliding window and sink tokens, dense and on packed sequences. No counterpart in the reference, whose window is the
number of keys that a dynamic mask keeps. Over the paged 8-bit cache: `flash_sparse_attn_cache_func(..., sliding_window, sink_tokens)`.

    the query at position t sees the key at position k:  k <= t  and  (t - k < sliding_window or k < sink_tokens)  and  mask(k)

Key tiles that no query of a tile sees are neither loaded nor multiplied (csrc/fdma_fwd_sm100.cu, fdma_bwd_rows_sm100.cu,
fdma_bwd256_sm100.cu; a single query: fdma_decode.cu); the mask is one of the keys, for all queries. Probabilities and dS are rounded to the
inputs' type before they enter a product, as in the calls without a window, and the backward's rowsum(dout * out) is formed from the rounded out.
"""
import ctypes
import math
from typing import Optional, Tuple

import torch

from . import _lib, _native
from . import flash_sparse_attn_interface as _interface

__all__ = ["flash_sparse_attn_window_func", "flash_sparse_attn_window_varlen_func"]


def _check_scale(softmax_scale) -> None:
    if softmax_scale is not None and not 0 <= softmax_scale < math.inf:
        raise ValueError(f"softmax_scale must be a finite number of at least 0, got {softmax_scale}")


def check_window(sliding_window, sink_tokens) -> None:
    for name, x in (("sliding_window", sliding_window), ("sink_tokens", sink_tokens)):
        if not isinstance(x, (int, torch.SymInt)) or isinstance(x, bool):
            raise TypeError(f"{name} must be an int, got {type(x).__name__}")
    if not 1 <= sliding_window < 2 ** 31 or not 0 <= sink_tokens < 2 ** 31:
        raise ValueError("sliding_window must be at least 1 and sink_tokens at least 0, both below 2^31")


def _sums_without_order(query, key, value) -> bool:
    """Whether the backward of the call without a window may add up dQ in any order, as it does for few queries over many keys
    (bwd_rows_taken in csrc/fdma_bwd_rows_sm100.cu); with `deterministic` it has one, but adds up in fixed point, which rounds small gradients.
    (1024 queries over 16384 keys, 32 heads over 8, d = 128, backward: 670 us in any order, 842 in fixed point, 948 here.)"""
    Sq, Sk = query.shape[1], key.shape[1]
    if query.shape[-1] > 128 or not torch.is_grad_enabled() or not any(t.requires_grad for t in (query, key, value)):
        return False
    if _interface._kernel_path not in (_lib.PATH_AUTO, _lib.PATH_TCGEN05) or Sk > 2 ** 20:  # not the window's
        return False
    return Sk >= 2048 and Sk >= (4 if Sk >= 4096 else 8) * Sq


def flash_sparse_attn_window_func(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    sliding_window: int,
    sink_tokens: int = 0,
    attn_mask: Optional[torch.Tensor] = None,
    softmax_scale: Optional[float] = None,
    deterministic: Optional[bool] = None,
    return_attn_probs: Optional[bool] = None,
):
    """Causal attention in which a query sees the last `sliding_window` keys, its own among them, and the first `sink_tokens`.

    query (B, Sq, H, d); key, value (B, Sk, Hk, d) with H % Hk == 0; fp16 or bf16, head dims up to 256. Query i is at position
    i + Sk - Sq, as under `flash_sparse_attn_func(is_causal=True)`, which this equals where the window is as long as the keys.
    attn_mask: bool ({B|1}, {H|Hk|1}, 1, {Sk|1}), False = masked out, such as padding; masks per query are not built. Rows that see no key
    return 0. Keys and values are expected to be finite, also where the mask hides them. softmax_scale, 0 or above, defaults to d ** -0.5.
    B, Sq and Sk are at least 1 (packed sequences may be empty), Sk at most 2^20 where the window leaves keys out.
    return_attn_probs=True returns (out, softmax_lse (B, H, Sq) fp32, empty tensor).

    Time and traffic go with the window, not with Sk. Returns out (B, Sq, H, d); gradients flow to query, key and value, each a sum in
    a fixed order, with `deterministic` or without. Head dims above 128 have none with a mask of its own for each query
    head. Nothing synchronises: a step can be captured into a CUDA graph."""
    check_window(sliding_window, sink_tokens)
    _check_scale(softmax_scale)
    if attn_mask is not None:
        if not isinstance(attn_mask, torch.Tensor) or attn_mask.dtype != torch.bool or attn_mask.dim() != 4:
            raise RuntimeError("attn_mask must be a bool tensor ({B|1}, {H|Hk|1}, 1, {Sk|1})")
        if attn_mask.shape[2] != 1:
            raise NotImplementedError("masks per query are not built with a sliding window: attn_mask must be ({B|1}, {H|Hk|1}, 1, {Sk|1})")
        if key.dim() == 4 and attn_mask.shape[3] not in (1, key.shape[1], _interface.round_multiple(key.shape[1], _interface._KEY_PAD)):
            raise RuntimeError("attn_mask must be a bool tensor ({B|1}, {H|Hk|1}, 1, {Sk|1})")
        if query.dim() == key.dim() == 4 and query.shape[-1] > 128 and attn_mask.shape[1] not in (1, key.shape[2]) and torch.is_grad_enabled() \
                and any(t.requires_grad for t in (query, key, value)):
            raise NotImplementedError("head dims above 128 have no gradients with a mask of its own for each query head")
    elif key.dim() == query.dim() == 4 and sliding_window + sink_tokens >= key.shape[1] and not _sums_without_order(query, key, value):
        # every query sees all keys up to its own
        return _interface.flash_sparse_attn_func(query, key, value, None, None, softmax_scale, True, None, deterministic,
                                                 return_attn_probs)
    if not return_attn_probs and not torch.compiler.is_compiling() and _interface._kernel_path in (_lib.PATH_AUTO, _lib.PATH_TCGEN05):
        out = _native.load().attention(query, key, value, attn_mask, None, None, None, None, None, softmax_scale, True, bool(deterministic),
                                       _interface._kernel_path, sliding_window, sink_tokens)
        if out is not None:
            return out
    d = query.shape[-1]
    softmax_scale = d ** -0.5 if softmax_scale is None else softmax_scale
    if d % 8:  # 16-bit rows are kept 16-byte aligned
        query, key, value = (torch.nn.functional.pad(t, [0, 8 - d % 8]) for t in (query, key, value))
    if attn_mask is not None and key.dim() == 4:
        keys = _interface.round_multiple(key.shape[1], _interface._KEY_PAD)
        if attn_mask.shape[-1] == 1:
            attn_mask = attn_mask.expand(*attn_mask.shape[:-1], keys)
        elif attn_mask.shape[-1] != keys:
            attn_mask = torch.nn.functional.pad(attn_mask, [0, keys - attn_mask.shape[-1]])
    out, lse = _WindowAttnFunc.apply(query, key, value, attn_mask, softmax_scale, sliding_window, sink_tokens)
    out = out[..., :d]
    return (out, lse, torch.empty((0,), dtype=query.dtype, device=query.device)) if return_attn_probs else out


def flash_sparse_attn_window_varlen_func(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    cu_seqlens_k: torch.Tensor,
    max_seqlen_q: int,
    max_seqlen_k: int,
    sliding_window: int,
    sink_tokens: int = 0,
    softmax_scale: Optional[float] = None,
    deterministic: Optional[bool] = None,
    return_attn_probs: Optional[bool] = None,
):
    """`flash_sparse_attn_window_func` on packed sequences: arguments and results as of `flash_sparse_attn_varlen_func`, positions,
    window and sinks in each sequence. Up to head dim 128 the sequences run in one launch per direction and nothing synchronises: the boundaries stay
    on the GPU, where they must ascend from 0 or more (otherwise results are undefined, within the tensors); what they leave out, or what lies
    beyond the tensors, belongs to no sequence, whose rows are 0, gradients too. Other calls go sequence by sequence, their boundaries read on the host."""
    check_window(sliding_window, sink_tokens)
    _check_scale(softmax_scale)
    if not return_attn_probs and not torch.compiler.is_compiling() and _interface._kernel_path == _lib.PATH_AUTO and query.is_cuda:
        scale = query.shape[-1] ** -0.5 if softmax_scale is None else float(softmax_scale)
        res = _native.load().packed_attention(query, key, value, cu_seqlens_q, cu_seqlens_k, scale, True, bool(deterministic), sliding_window,
                                              sink_tokens)
        if res is not None:
            return res[0]
    if torch.compiler.is_compiling() and not return_attn_probs and _traces_packed(query, key, value, cu_seqlens_q, cu_seqlens_k):
        d = query.shape[-1]
        softmax_scale = d ** -0.5 if softmax_scale is None else softmax_scale
        if d % 8:  # 16-bit rows are kept 16-byte aligned
            query, key, value = (torch.nn.functional.pad(t, [0, 8 - d % 8]) for t in (query, key, value))
        return _PackedWindowAttnFunc.apply(query, key, value, cu_seqlens_q, cu_seqlens_k, softmax_scale, sliding_window, sink_tokens)[0][..., :d]
    return _interface._varlen(query, key, value, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, softmax_scale, True, None,
                              deterministic, return_attn_probs, sliding_window, sink_tokens)


def _traces_packed(q, k, v, cu_q, cu_k) -> bool:
    """Whether a call that is traced is one operator, as it is one launch without tracing; others read the boundaries."""
    return (_interface._kernel_path == _lib.PATH_AUTO and q.is_cuda and q.dim() == k.dim() == v.dim() == 3 and q.shape[-1] <= 128
            and 0 < q.shape[0] <= 2 ** 19 and 0 < k.shape[0] <= 2 ** 20 and cu_q.dim() == cu_k.dim() == 1
            and cu_q.shape[0] == cu_k.shape[0] >= 2 and cu_q.dtype == cu_k.dtype == torch.int32)


class _WindowAttnFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, mask, scale, window, sinks):
        out, lse = torch.ops.flash_sparse_attn._window_forward(q, k, v, mask, scale, window, sinks)
        ctx.save_for_backward(q, k, v, mask, out, lse)
        ctx.args = (scale, window, sinks)
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    def backward(ctx, dout, *_):
        q, k, v, mask, out, lse = ctx.saved_tensors
        return (*torch.ops.flash_sparse_attn._window_backward(dout, q, k, v, mask, out, lse, *ctx.args), None, None, None, None)


class _PackedWindowAttnFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, scale, window, sinks):
        # (cu: the backward's own boundaries, since the caller may fill its buffers for the next call before)
        out, lse, cu = torch.ops.flash_sparse_attn._window_varlen_forward(q, k, v, cu_q, cu_k, scale, window, sinks)
        ctx.save_for_backward(q, k, v, cu, out, lse)
        ctx.args = (scale, window, sinks)
        ctx.mark_non_differentiable(lse, cu)
        return out, lse, cu

    @staticmethod
    def backward(ctx, dout, *_):
        q, k, v, cu, out, lse = ctx.saved_tensors
        return (*torch.ops.flash_sparse_attn._window_varlen_backward(dout, q, k, v, cu, out, lse, *ctx.args), None, None, None, None, None)


def _aligned(t: Optional[torch.Tensor], unit: int) -> Optional[torch.Tensor]:
    """The tensor as the kernels load it: 16-byte aligned base and strides, innermost dimension dense."""
    if t is None:
        return None
    ok = t.stride(-1) == 1 and t.data_ptr() % 16 == 0
    ok = ok and all(t.stride(i) % unit == 0 and (t.stride(i) > 0 or unit == 16) for i in range(t.dim() - 1) if t.shape[i] > 1)
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _prepare(q, k, v, mask):
    q, k, v, mask = _aligned(q, 8), _aligned(k, 8), _aligned(v, 8), _aligned(mask, 16)
    _interface._check_inputs(q, k, v, mask, None)
    return q, k, v, mask


def _launch_forward(q, k, v, mask, softmax_scale, window, sinks, cu=None):
    lib = _lib.load()
    with torch.cuda.device(q.device):
        _interface._raise_if_kernel_timed_out(lib)
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        lse = torch.empty((q.shape[0], q.shape[2], q.shape[1]), dtype=torch.float32, device=q.device)
        p = _lib.FwdParams()
        _interface._fill_fwd(p, q, k, v, mask, None, out, lse, softmax_scale, True)
        cu_q, cu_k, n = (None, None, 0) if cu is None else (cu[0].data_ptr(), cu[1].data_ptr(), cu.shape[1] - 1)
        size = lib.fdma_fwd_window_workspace_bytes(ctypes.byref(p), window, sinks, n)
        ws = torch.empty(size, dtype=torch.uint8, device=q.device)
        p.workspace, p.workspace_bytes = ws.data_ptr(), size
        _lib.check(lib.fdma_fwd_window(ctypes.byref(p), window, sinks, cu_q, cu_k, n, _interface._stream_ptr(q.device)), "fdma_fwd_window")
    return out, lse


def _launch_backward(dout, q, k, v, mask, out, lse, softmax_scale, window, sinks, cu=None):
    dout, out, lse = _aligned(dout, 8), _aligned(out, 8), lse.contiguous()
    lib = _lib.load()
    with torch.cuda.device(q.device):
        _interface._raise_if_kernel_timed_out(lib)
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        bp = _lib.BwdParams()
        _interface._fill_fwd(bp.f, q, k, v, mask, None, out, lse, softmax_scale, True)
        for name, t in (("do", dout), ("dq", dq), ("dk", dk), ("dv", dv)):
            setattr(bp, "dout" if name == "do" else name, t.data_ptr())
            for x, stride in zip(("batch", "row", "head"), _interface._bsh(t)):
                setattr(bp, f"{name}_{x}_stride", stride)
        cu_q, cu_k, n = (None, None, 0) if cu is None else (cu[0].data_ptr(), cu[1].data_ptr(), cu.shape[1] - 1)
        size = lib.fdma_bwd_window_workspace_bytes(ctypes.byref(bp), window, sinks, n)
        ws = torch.empty(size, dtype=torch.uint8, device=q.device)
        bp.f.workspace, bp.f.workspace_bytes = ws.data_ptr(), size
        _lib.check(lib.fdma_bwd_window(ctypes.byref(bp), window, sinks, cu_q, cu_k, n, _interface._stream_ptr(q.device)), "fdma_bwd_window")
    return dq, dk, dv


@torch.library.custom_op("flash_sparse_attn::_window_forward", mutates_args=(), device_types="cuda")
def _window_forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mask: Optional[torch.Tensor], softmax_scale: float, window: int,
                    sinks: int) -> Tuple[torch.Tensor, torch.Tensor]:
    return _launch_forward(*_prepare(q, k, v, mask), softmax_scale, window, sinks)


@torch.library.register_fake("flash_sparse_attn::_window_forward")
def _window_forward_fake(q, k, v, mask, softmax_scale, window, sinks):
    B, Sq, H, _ = q.shape
    return torch.empty(q.shape, dtype=q.dtype, device=q.device), torch.empty((B, H, Sq), dtype=torch.float32, device=q.device)


@torch.library.custom_op("flash_sparse_attn::_window_backward", mutates_args=(), device_types="cuda")
def _window_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mask: Optional[torch.Tensor], out: torch.Tensor,
                     softmax_lse: torch.Tensor, softmax_scale: float, window: int, sinks: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _launch_backward(dout, *_prepare(q, k, v, mask), out, softmax_lse, softmax_scale, window, sinks)


@torch.library.register_fake("flash_sparse_attn::_window_backward")
def _window_backward_fake(dout, q, k, v, mask, out, softmax_lse, softmax_scale, window, sinks):
    return tuple(torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))


# Packed sequences: (tokens, heads, d), lse (heads, tokens), cu (2, sequences + 1): the boundaries of the queries and of the keys
def _prepare_packed(q, k, v):
    return _prepare(q.unsqueeze(0), k.unsqueeze(0), v.unsqueeze(0), None)


@torch.library.custom_op("flash_sparse_attn::_window_varlen_forward", mutates_args=(), device_types="cuda")
def _window_varlen_forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor, cu_k: torch.Tensor, softmax_scale: float,
                           window: int, sinks: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    for cu in (cu_q, cu_k):
        if cu.dtype != torch.int32 or cu.dim() != 1 or cu.device != q.device or cu.shape != cu_q.shape or cu.shape[0] < 2:
            raise RuntimeError("cu_seqlens_q and cu_seqlens_k must be int32 tensors (sequences + 1) on the query's device")
    cu = torch.stack((cu_q, cu_k))
    out, lse = _launch_forward(*_prepare_packed(q, k, v), softmax_scale, window, sinks, cu)
    return out[0], lse[0], cu


@torch.library.register_fake("flash_sparse_attn::_window_varlen_forward")
def _window_varlen_forward_fake(q, k, v, cu_q, cu_k, softmax_scale, window, sinks):
    return (torch.empty(q.shape, dtype=q.dtype, device=q.device), torch.empty((q.shape[1], q.shape[0]), dtype=torch.float32, device=q.device),
            torch.empty((2, cu_q.shape[0]), dtype=torch.int32, device=q.device))


@torch.library.custom_op("flash_sparse_attn::_window_varlen_backward", mutates_args=(), device_types="cuda")
def _window_varlen_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu: torch.Tensor, out: torch.Tensor,
                            softmax_lse: torch.Tensor, softmax_scale: float, window: int,
                            sinks: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    res = _launch_backward(dout.unsqueeze(0), *_prepare_packed(q, k, v), out.unsqueeze(0), softmax_lse, softmax_scale, window, sinks, cu)
    return tuple(x[0] for x in res)


@torch.library.register_fake("flash_sparse_attn::_window_varlen_backward")
def _window_varlen_backward_fake(dout, q, k, v, cu, out, softmax_lse, softmax_scale, window, sinks):
    return tuple(torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
