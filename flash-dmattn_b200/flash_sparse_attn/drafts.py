"""Verification of drafted tokens in a serving step, on the GPU: which drafts of each request the target's probabilities accept, the token
that comes next, and the lengths to which the block tables go back. The reference has none.

    step = tables.extend(new_lengths, total_tokens)             # a request's last token and its drafts
    logits = model(token_ids, step, ...)                        # cache_append, flash_sparse_attn_cache_func
    done = verify_drafts(step, token_ids, logits, torch.rand(total_tokens, device="cuda"), draft_probs)
    tables.truncate(done.lengths)                               # the rejected drafts leave the cache
    # the next step's tokens: done.next_tokens, then new drafts behind them

Nothing synchronises, so that this too can be captured into the step's CUDA graph.
"""
import math
from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _native
from .cache import CacheStep

__all__ = ["VerifiedDrafts", "verify_drafts"]


class VerifiedDrafts(NamedTuple):
    accepted: torch.Tensor     # int32 (requests,): drafts that are accepted
    next_tokens: torch.Tensor  # int64 (requests,): the token behind them; -1 where there is none
    lengths: torch.Tensor      # int32 (requests,): tokens of the request without the drafts that are not, for `BlockTables.truncate`


def verify_drafts(
    step: CacheStep,
    token_ids: torch.Tensor,
    logits: torch.Tensor,
    uniforms: torch.Tensor,
    draft_probs: Optional[torch.Tensor] = None,
    temperature: Union[float, torch.Tensor] = 1.0,
) -> VerifiedDrafts:
    """Of a request's tokens in the step all but the first are drafts: token j + 1 is what the drafter made of token j. A request with one
    token has none, and its next token is drawn as in plain sampling.

    token_ids (tokens,), int32 or int64: the step's tokens. logits (tokens, vocabulary), bf16, fp16 or fp32: row i is the target's for what
    follows token i. uniforms (tokens,), float32 in [0, 1). draft_probs (tokens, vocabulary), bf16, fp16 or fp32: row i the probabilities
    that the draft behind token i was drawn from (the last row of a request is not read); None: drafts that were not drawn, such as looked up ones.
    temperature: a number or float32 (requests,).
    Of the step its cu_seqlens, lengths and granted count. Where others' prompt parts are in the step, gather the rows that matter (the last one
    of a part, all of a request with drafts) and give their boundaries: step._replace(cu_seqlens=...).

    With p = softmax(logits / temperature) and q the drafter's row, the draft x behind token i is accepted if uniforms[i] * q(x) < p(x), and the
    first one that is not ends the request's. The next token is drawn from what that row leaves, max(p - q, 0) (without draft_probs: p
    without x), or if all are accepted from p of the last row, so that tokens are distributed as the target's own: the first token whose running
    sum is above the total times the uniform of the request's last token. temperature 0 (or below): the largest logit, of equal ones the first, is accepted
    and comes next.

    What the random numbers are compared with is summed up in 64 bits, in one order: the same inputs give the same tokens. NaN
    logits count as -inf, +inf as the largest finite number, drafts outside the vocabulary are rejected. Requests without
    tokens in the step or refused by it: nothing accepted, next token -1, lengths as they are. There are no gradients: a call that would need them raises."""
    temperatures = None
    if isinstance(temperature, torch.Tensor):
        temperatures, temperature = temperature, 0.0
    else:
        temperature = float(temperature)
        if not 0.0 <= temperature < math.inf:
            raise ValueError(f"temperature must be a finite number of at least 0, got {temperature}.")
    args = (step.cu_seqlens, step.lengths, step.granted, token_ids, logits, uniforms, draft_probs, temperatures)
    out = None
    if not torch.compiler.is_compiling():
        out = _native.load().verify_drafts(args, temperature)
    if out is None:
        out = torch.ops.flash_sparse_attn._verify_drafts(*args, temperature)
    return VerifiedDrafts(*out)


# ---- the same as a custom operator, for tracing ------------------------------------------------------------------------
@torch.library.custom_op("flash_sparse_attn::_verify_drafts", mutates_args=(), device_types="cuda")
def _verify_drafts(cu_seqlens: torch.Tensor, lengths: torch.Tensor, granted: torch.Tensor, token_ids: torch.Tensor, logits: torch.Tensor,
                   uniforms: torch.Tensor, draft_probs: Optional[torch.Tensor], temperatures: Optional[torch.Tensor],
                   temperature: float) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    out = _native.load().verify_drafts((cu_seqlens, lengths, granted, token_ids, logits, uniforms, draft_probs, temperatures), temperature)
    if out is None:
        raise RuntimeError("verify_drafts: these tensors are not supported")
    return tuple(out)


@torch.library.register_fake("flash_sparse_attn::_verify_drafts")
def _verify_drafts_fake(cu_seqlens, lengths, granted, token_ids, logits, uniforms, draft_probs, temperatures, temperature):
    R = lengths.shape[0]
    return tuple(torch.empty((R,), dtype=t, device=logits.device) for t in (torch.int32, torch.int64, torch.int32))
