"""The reference's HuggingFace glue
(flash_sparse_attn/integrations/modeling_flash_sparse_attention_utils.py:425-596): recast fp32 activations to the
model's half-precision dtype (:321-339), build the top-`window_size` mask from the bias only when the key length
exceeds the window (:570-583), and call `flash_sparse_attn_func`.

A 2-D padding mask (batch, seq_len) is handled without un-padding: the reference gathers the valid tokens, runs its
variable-length kernel with no bias and no dynamic mask, and pads the result with zeros (:511-536, `_upad_input`
:144-220). The same numbers come out of the dense operator when the padding mask is passed as a row-broadcast key
mask (B, 1, 1, Sk) -- valid tokens keep their order, so the causal test on padded positions equals the causal test
on gathered positions (for query_length < key_length under the left padding the reference assumes, :209-211) -- and
the padded query rows are zeroed afterwards. Few valid keys -> `flash_sparse_attn_func` takes its gathered-keys route.

Packed sequences given by position ids or cu_seqlens (:538-565, `_prepare_from_posids` :270-302) go through the
reference's varlen kernel as well. Here small packs (Tq x Tk up to `_PACKED_MASK_LIMIT` elements) run as ONE
sequence under a per-query visibility mask (same example, and causal inside the example with the bottom-right
alignment of its own lengths), which the full-range kernels skip tile by tile -- one launch however many examples
there are; larger packs go through `flash_sparse_attn_varlen_func`, which runs every example as a zero-copy slice.

`sliding_window`, which models hand over for their windowed layers (the reference drops it): a query sees the last so many keys, its own among
them. Dense, padded and packed calls go to the window's operators; with a bias, or a mask per query, the window becomes part of the mask.
"""
import math
import os
from typing import NamedTuple, Optional

import torch

from ..cache import BlockTables, CacheStep, QuantizedCache, cache_append, flash_sparse_attn_cache_func
from ..flash_sparse_attn_interface import flash_sparse_attn_func, flash_sparse_attn_varlen_func
from ..rotary import RotaryFrequencies
from ..utils.mask import create_kept_keys, create_mask
from ..window import check_window, flash_sparse_attn_window_func, flash_sparse_attn_window_varlen_func


def fsa_peft_integration_check(q, k, v, bias, target_dtype: Optional[torch.dtype] = None):
    """fp32 activations (PEFT keeps layer norms in fp32) go back to `target_dtype`; anything else passes through."""
    if target_dtype is not None and q.dtype == torch.float32:
        q, k, v = q.to(target_dtype), k.to(target_dtype), v.to(target_dtype)
        bias = bias.to(target_dtype) if bias is not None else None
    return q, k, v, bias


def _is_packed_sequence(position_ids: Optional[torch.Tensor], batch_size: int) -> bool:
    """Packed (padding-free) batches show up as one row of position ids that restarts from 0 somewhere
    (reference :279-296)."""
    if position_ids is None or position_ids.dim() != 2 or batch_size != 1 or position_ids.shape[1] < 2:
        return False
    expected = torch.arange(position_ids.shape[1], device=position_ids.device) + position_ids.min()
    return not bool((position_ids[0] == expected).all())


_PACKED_MASK_LIMIT = 1 << 24  # largest (Tq, Tk) visibility mask built for packed sequences; beyond: per-example calls


def _packed_visibility(cu_q: torch.Tensor, cu_k: torch.Tensor, total_q: int, total_k: int, causal: bool,
                       device) -> torch.Tensor:
    """(total_q, total_k) bool: query token i sees key token j iff both lie in the same example and, when causal,
    j_local <= i_local + len_k - len_q (the varlen kernels' bottom-right alignment per example). Tokens past the
    last boundary see nothing."""
    cu_q = cu_q.to(device=device, dtype=torch.int64)
    cu_k = cu_k.to(device=device, dtype=torch.int64)
    n = cu_q.numel() - 1
    tq = torch.arange(total_q, device=device)
    tk = torch.arange(total_k, device=device)
    sq = torch.bucketize(tq, cu_q[1:], right=True)   # example of each token; == n past the last boundary
    sk = torch.bucketize(tk, cu_k[1:], right=True)
    visible = (sq[:, None] == sk[None, :]) & (sq[:, None] < n) & (tq[:, None] >= cu_q[0]) & (tk[None, :] >= cu_k[0])
    if causal:
        sq_c = sq.clamp(max=n - 1)
        local_q = tq - cu_q[sq_c]
        local_k = tk - cu_k[sk.clamp(max=n - 1)]
        shift = (cu_k[1:] - cu_k[:-1] - (cu_q[1:] - cu_q[:-1]))[sq_c]
        visible &= local_k[None, :] <= (local_q + shift)[:, None]
    return visible


def _window_that_hides(sliding_window: Optional[int], keys: int, is_causal: bool, softcap: Optional[float]) -> Optional[int]:
    """The window, or None where `keys` keys are all in it."""
    if sliding_window is None:
        return None
    check_window(sliding_window, 0)
    if sliding_window >= keys:
        return None
    if not is_causal:
        raise NotImplementedError("sliding_window is built for causal attention only")
    if softcap:
        raise NotImplementedError("softcap > 0 is not built into the B200 kernels")
    return sliding_window


def _flash_sparse_attention_forward(
    query_states: torch.Tensor,
    key_states: torch.Tensor,
    value_states: torch.Tensor,
    attention_mask: Optional[torch.Tensor],
    attention_bias: Optional[torch.Tensor],
    query_length: int,
    key_length: int,
    is_causal: bool,
    position_ids: Optional[torch.Tensor] = None,
    softmax_scale: Optional[float] = None,
    window_size: Optional[int] = None,
    softcap: Optional[float] = None,
    deterministic: Optional[bool] = None,
    cu_seq_lens_q: Optional[torch.LongTensor] = None,
    cu_seq_lens_k: Optional[torch.LongTensor] = None,
    max_length_q: Optional[int] = None,
    max_length_k: Optional[int] = None,
    target_dtype: Optional[torch.dtype] = None,
    implementation: Optional[str] = None,
    sliding_window: Optional[int] = None,
    **kwargs,
):
    """query/key/value (B, S, H, d). Returns (B, Sq, H, d). Same argument list as the reference function, and `sliding_window`: of the keys
    that a call without it sees, a query sees the last so many (with `window_size`: those of the kept keys). A single query, which sees all keys,
    is at the last of them."""
    if attention_mask is not None and attention_mask.dim() == 2 and attention_bias is not None:
        raise ValueError("If shape of attention_mask is (batch_size, seq_len), attention_bias has to be None.")
    padded = attention_mask is not None and attention_mask.dim() == 2
    packed_kwargs = all(x is not None for x in (cu_seq_lens_q, cu_seq_lens_k, max_length_q, max_length_k))
    packed = not padded and (packed_kwargs or _is_packed_sequence(position_ids, query_states.size(0)))

    query_states, key_states, value_states, attention_bias = fsa_peft_integration_check(
        query_states, key_states, value_states, attention_bias, target_dtype)
    if deterministic is None:
        deterministic = os.getenv("FLASH_SPARSE_ATTENTION_DETERMINISTIC", "0") == "1"

    if packed:
        if cu_seq_lens_q is None or cu_seq_lens_k is None:  # boundaries from the position ids (reference :241-251)
            flat = position_ids.reshape(-1)
            starts = (flat == 0).nonzero().view(-1).to(torch.int64)
            cu_seq_lens_q = cu_seq_lens_k = torch.cat(
                (starts, torch.tensor([flat.numel()], dtype=torch.int64, device=flat.device)))
        B = query_states.size(0)
        q1 = query_states.reshape(1, -1, query_states.size(-2), query_states.size(-1))
        k1 = key_states.reshape(1, -1, key_states.size(-2), key_states.size(-1))
        v1 = value_states.reshape(1, -1, value_states.size(-2), value_states.size(-1))
        window = _window_that_hides(sliding_window, k1.size(1), is_causal, softcap)
        if window is not None or q1.size(1) * k1.size(1) > _PACKED_MASK_LIMIT:
            if max_length_q is None or max_length_k is None:
                max_length_q = int((cu_seq_lens_q[1:] - cu_seq_lens_q[:-1]).max())
                max_length_k = int((cu_seq_lens_k[1:] - cu_seq_lens_k[:-1]).max())
            if window is not None:
                cu = [x.to(device=q1.device, dtype=torch.int32) for x in (cu_seq_lens_q, cu_seq_lens_k)]
                out = flash_sparse_attn_window_varlen_func(q1[0], k1[0], v1[0], *cu, max_length_q, max_length_k, window,
                                                           softmax_scale=softmax_scale, deterministic=deterministic)
                return out.view(B, -1, out.size(-2), out.size(-1))
            out = flash_sparse_attn_varlen_func(q1[0], k1[0], v1[0], cu_seq_lens_q, cu_seq_lens_k, max_length_q,
                                                max_length_k, softmax_scale=softmax_scale, is_causal=is_causal,
                                                softcap=softcap, deterministic=deterministic)
            return out.view(B, -1, out.size(-2), out.size(-1))
        visible = _packed_visibility(cu_seq_lens_q, cu_seq_lens_k, q1.size(1), k1.size(1), is_causal, q1.device)
        out = flash_sparse_attn_func(q1, k1, v1, visible[None, None], None, softmax_scale=softmax_scale,
                                     is_causal=False, softcap=softcap, deterministic=deterministic)
        out = out[0] if isinstance(out, tuple) else out
        return out.view(B, -1, out.size(-2), out.size(-1))

    if padded:
        # static caches: k/v may be longer than the mask (reference :187-190)
        seq_len = attention_mask.shape[-1]
        if key_states.shape[1] > seq_len:
            key_states, value_states = key_states[:, :seq_len], value_states[:, :seq_len]
        key_valid = attention_mask.to(torch.bool)
        if query_length == key_states.shape[1]:
            query_valid = key_valid
        elif query_length == 1:
            query_valid = None
        else:
            query_valid = key_valid[:, -query_length:]  # left padding, as the reference assumes
        window = _window_that_hides(sliding_window, key_states.shape[1], is_causal or query_length == 1, softcap)
        if window is not None and query_length == 1:  # the last keys that are there, wherever the padding is
            key_valid = key_valid & (key_valid.flip(-1).cumsum(-1).flip(-1) <= window)
            window = None
        if window is not None:
            out = flash_sparse_attn_window_func(query_states, key_states, value_states, window, attn_mask=key_valid[:, None, None, :],
                                                softmax_scale=softmax_scale, deterministic=deterministic)
        else:
            out = flash_sparse_attn_func(
                query_states, key_states, value_states, key_valid[:, None, None, :], None,
                softmax_scale=softmax_scale, is_causal=is_causal and query_length != 1,
                softcap=softcap, deterministic=deterministic)
        out = out[0] if isinstance(out, tuple) else out
        if query_valid is not None:
            out = torch.where(query_valid[:, :, None, None], out, torch.zeros((), dtype=out.dtype, device=out.device))
        return out

    if attention_bias is not None and window_size is not None and key_length > window_size:
        attention_mask = create_mask(
            attention_bias, attention_mask, batch_size=query_states.size(0), query_len=query_length,
            key_len=key_length, window_size=window_size, min_dtype=torch.finfo(attention_bias.dtype).min)
    window = _window_that_hides(sliding_window, key_states.shape[1], is_causal or query_length == 1, softcap)
    if window is not None:
        Sq, Sk, mask = query_states.shape[1], key_states.shape[1], attention_mask
        # (gradients at head dims above 128 take no mask of its own for each query head beside a window)
        if attention_bias is None and (mask is None or (mask.dim() == 4 and mask.shape[2] == 1 and mask.shape[1] in (1, key_states.shape[2]))):
            return flash_sparse_attn_window_func(query_states, key_states, value_states, window, attn_mask=mask, softmax_scale=softmax_scale,
                                                 deterministic=deterministic)
        if mask is not None and mask.dtype != torch.bool:
            raise RuntimeError("attention_mask must be a bool tensor")
        inside = torch.arange(Sk, device=query_states.device) > torch.arange(Sk - Sq, Sk, device=query_states.device)[:, None] - window
        attention_mask = inside[None, None] if mask is None else mask[..., :Sk] & inside
    out = flash_sparse_attn_func(
        query_states, key_states, value_states, attention_mask, attention_bias,
        softmax_scale=softmax_scale, is_causal=is_causal and query_length != 1,
        softcap=softcap, deterministic=deterministic)
    return out[0] if isinstance(out, tuple) else out


class CachedLayer(NamedTuple):
    """What a layer needs to attend over the paged 8-bit cache in a step."""

    cache: QuantizedCache                             # the layer's own
    tables: BlockTables                               # of all layers
    step: CacheStep                                   # of this step, from `tables.extend`
    frequencies: Optional[RotaryFrequencies] = None   # query and key are turned here; None: they are already
    max_seqlen_q: Optional[int] = None                # bounds on the requests' new tokens and lengths, where the host knows them
    max_seqlen_k: Optional[int] = None


def _cached_attention_forward(query_states, key_states, value_states, attention_mask, attention_bias, kv_cache: CachedLayer,
                              softmax_scale: Optional[float] = None, window_size: Optional[int] = None, is_causal: bool = True,
                              target_dtype: Optional[torch.dtype] = None, sliding_window: Optional[int] = None):
    """The step's keys and values (1, tokens, Hk, d) go into the cache, and its queries (1, tokens, H, d) attend over it: everything, or
    with a bias of more than `window_size` keys the `window_size` keys of each request that each row of the bias ranks highest: one
    row for all heads, or one per kv head or query head; of these those in the `sliding_window`. Returns (1, tokens, H, d). What the attention would refuse is refused here,
    before anything is written."""
    if attention_mask is not None:
        raise ValueError("attention over a cache takes no attention_mask: the requests' lengths are in the step.")
    if query_states.shape[0] != 1 or key_states.shape[0] != 1:
        raise ValueError("attention over a cache takes the step's tokens as one row.")
    q, k, v, bias = fsa_peft_integration_check(query_states[0], key_states[0], value_states[0], attention_bias, target_dtype)
    cache, tables, step, frequencies, max_q, max_k = kv_cache
    R, H, Hk = step.lengths.shape[0], q.shape[1], k.shape[1]
    if Hk == 0 or H % Hk:
        raise ValueError("attention over a cache takes as many query heads for each kv head.")
    window = _window_that_hides(sliding_window, tables.table.shape[-1] * tables.block_size, is_causal, None)
    if any(bound is not None and bound < 0 for bound in (max_q, max_k)):
        raise ValueError("max_seqlen_q and max_seqlen_k must not be negative.")
    if bias is not None:
        if bias.dim() != 4 or bias.shape[0] not in (1, R) or bias.shape[1] not in (1, Hk, H) or bias.shape[2] != 1 or bias.shape[3] == 0:
            raise ValueError("attention over a cache takes a bias ({1|requests}, {1|Hk|H}, 1, keys).")
        if bias.dtype != q.dtype or bias.device != q.device:
            raise ValueError("attention over a cache takes a bias of the query's dtype and device.")
        if torch.is_grad_enabled() and bias.requires_grad:
            raise ValueError("attention over a cache has no gradients: call it under torch.no_grad().")
    kept = None
    if bias is not None and window_size is not None and bias.shape[-1] > window_size:
        keys, low = bias.shape[-1], torch.finfo(bias.dtype).min
        valid = torch.arange(keys, device=bias.device) < step.lengths[:, None]
        rows = bias.expand(R, -1, -1, -1)
        if bias.shape[1] in (1, Hk):
            kept = create_kept_keys(rows, valid, R, 1, keys, window_size, low)
        else:  # the attention takes one list for each kv head: keys that any of its query heads keeps, hidden from the others
            mask = create_mask(rows, valid, R, 1, keys, window_size, low)
            bias = rows.masked_fill(~mask, -math.inf)
            kept = mask.view(R, Hk, H // Hk, 1, keys).any(2)
    turned = cache_append(cache, tables, step, k, v, query=q if frequencies is not None else None, frequencies=frequencies)
    q = q if turned is None else turned
    out = flash_sparse_attn_cache_func(q, cache, tables, step, attn_mask=kept, attn_bias=bias, softmax_scale=softmax_scale,
                                       is_causal=is_causal, max_seqlen_q=max_q, max_seqlen_k=max_k, sliding_window=window)
    return out[None]
