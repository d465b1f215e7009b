"""Rotary positions: queries and keys turned in pairs by position * frequency, forward and backward, in one launch.

The reference leaves this to the model around its attention call; here it stands beside the attention because the 8-bit cache's
writer (cache.py) turns keys on their way into the cache.
"""
import math
from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _native

__all__ = ["RotaryFrequencies", "rotary_frequencies", "apply_rotary"]


class RotaryFrequencies(NamedTuple):
    """What `rotary_frequencies` makes once per model and device."""

    turns: torch.Tensor        # int64 (rotary_dim / 2,): turns per position as 64-bit fractions of a turn
    interleaved: bool = False  # pairs (2 i, 2 i + 1) instead of (i, i + rotary_dim / 2)
    amplitude: float = 1.0     # factor on the cosines and sines


def _yarn(inv, base, dim, factor, original_length, beta_fast, beta_slow):
    """Frequencies that turn more than beta_fast times over the original length stay, those below beta_slow are divided by the
    factor, a linear ramp over the pairs lies between."""
    def pair_of(turns):
        return dim * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))

    low, high = max(math.floor(pair_of(beta_fast)), 0), min(math.ceil(pair_of(beta_slow)), dim - 1)
    ramp = ((torch.arange(dim // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
    return inv / factor * ramp + inv * (1 - ramp)


def _bands(inv, factor, original_length, low_freq_factor, high_freq_factor):
    """By wavelength: short ones (below original / high) stay, long ones (above original / low) are divided by the factor."""
    share = (original_length * inv / (2 * math.pi) - low_freq_factor) / (high_freq_factor - low_freq_factor)
    share = share.clamp(0, 1)
    return (1 - share) * inv / factor + share * inv


def rotary_frequencies(
    rotary_dim: int,
    base: float = 10000.0,
    scaling: str = "none",
    factor: float = 1.0,
    original_length: Optional[int] = None,
    beta_fast: float = 32.0,
    beta_slow: float = 1.0,
    low_freq_factor: float = 1.0,
    high_freq_factor: float = 4.0,
    amplitude: Optional[float] = None,
    interleaved: bool = False,
    inv_freq: Optional[torch.Tensor] = None,
    device: Optional[Union[str, torch.device]] = None,
) -> RotaryFrequencies:
    """Frequencies base^(-2 i / rotary_dim), i = 0 .. rotary_dim / 2 - 1, for `apply_rotary` and `cache_append`.

    scaling, for contexts longer than the model was trained at: "none"; "linear": every frequency divided by `factor`; "ntk": the
    base times factor^(rotary_dim / (rotary_dim - 2)); "yarn": low frequencies divided, high ones kept, a ramp between (from
    original_length, beta_fast, beta_slow), amplitude 0.1 ln(factor) + 1 unless given; "bands": the same by wavelengths (from
    original_length, low_freq_factor, high_freq_factor). inv_freq: frequencies in radians per position of the caller's own, in
    place of all that. The frequencies are computed in 64 bits; call this once, not per step."""
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be a positive even number, got {rotary_dim}.")
    if scaling not in ("none", "linear", "ntk", "yarn", "bands"):
        raise ValueError(f"Unsupported scaling: {scaling}. Supported are 'none', 'linear', 'ntk', 'yarn' and 'bands'.")
    if not factor > 0 or not base > 1:
        raise ValueError("factor must be positive and base greater than 1.")
    if scaling in ("yarn", "bands") and not original_length:
        raise ValueError(f"scaling '{scaling}' needs original_length.")
    if scaling == "bands" and not low_freq_factor < high_freq_factor:
        raise ValueError("low_freq_factor must be below high_freq_factor.")
    if inv_freq is not None:
        if inv_freq.shape != (rotary_dim // 2,):
            raise ValueError("inv_freq must hold rotary_dim / 2 frequencies.")
        inv = inv_freq.detach().to(device="cpu", dtype=torch.float64)
        device = inv_freq.device if device is None else device
        if not bool(inv.isfinite().all()):
            raise ValueError("inv_freq must be finite.")
    else:
        if scaling == "ntk":
            if rotary_dim <= 2:
                raise ValueError("scaling 'ntk' needs a rotary_dim above 2.")
            base = base * factor ** (rotary_dim / (rotary_dim - 2))
        inv = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
        if scaling == "linear":
            inv = inv / factor
        elif scaling == "yarn":
            inv = _yarn(inv, base, rotary_dim, factor, original_length, beta_fast, beta_slow)
            if amplitude is None:
                amplitude = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
        elif scaling == "bands":
            inv = _bands(inv, factor, original_length, low_freq_factor, high_freq_factor)
    # radians per position -> turns per position as a fraction of 2^64, the exact integer nearest to the 64-bit product
    turns = [round(f / (2 * math.pi) * 2.0 ** 64) % (1 << 64) for f in inv.tolist()]
    turns = [t - (1 << 64) if t >= 1 << 63 else t for t in turns]
    device = torch.device("cuda") if device is None else device
    return RotaryFrequencies(torch.tensor(turns, dtype=torch.int64, device=device), bool(interleaved),
                             1.0 if amplitude is None else float(amplitude))


def apply_rotary(
    query: torch.Tensor,
    key: Optional[torch.Tensor],
    frequencies: RotaryFrequencies,
    positions: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Turns query (B, S, H, d) and key (B, S, Hk, d) -- or packed tokens (T, H, d), (T, Hk, d) -- by their positions:
    elements x1, x2 of a pair become a (x1 cos - x2 sin), a (x2 cos + x1 sin); elements from rotary_dim on are copied. Returns new
    tensors (key None: (query, None)); gradients flow to query and key, any number of times.

    bf16, fp16 or fp32, any strides with a head's elements side by side (others are copied first). positions: int32 or int64,
    ({1|B}, S) or (S,), any value; None: 0 .. S - 1. Frequencies are held to 2^-65 of a turn per position and angles to
    2^-32 of a turn (at position 10^6, too), sums are 32-bit and the results are rounded once."""
    native = _native.load()
    if not torch.compiler.is_compiling():
        out = native.rotary((query, key, positions, frequencies.turns), frequencies.interleaved, frequencies.amplitude, False)
        if out is not None:
            return (out[0], out[1]) if key is not None else (out[0], None)
    out = torch.ops.flash_sparse_attn._apply_rotary(query, key, positions, frequencies.turns, frequencies.interleaved,
                                                    frequencies.amplitude, False)
    return (out[0], out[1]) if key is not None else (out[0], None)


@torch.library.custom_op("flash_sparse_attn::_apply_rotary", mutates_args=(), device_types="cuda")
def _apply_rotary(query: torch.Tensor, key: Optional[torch.Tensor], positions: Optional[torch.Tensor], turns: torch.Tensor,
                  interleaved: bool, amplitude: float, inverse: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    out = _native.load().rotary((query, key, positions, turns), interleaved, amplitude, inverse)
    if out is None:
        raise RuntimeError("apply_rotary: these tensors are not supported")
    return (out[0], out[1]) if key is not None else (out[0], query.new_empty((0,)))


@torch.library.register_fake("flash_sparse_attn::_apply_rotary")
def _apply_rotary_fake(query, key, positions, turns, interleaved, amplitude, inverse):
    def like(x):
        return torch.empty(x.shape, dtype=x.dtype, device=x.device)

    return like(query), like(key) if key is not None else query.new_empty((0,))


def _rotary_setup(ctx, inputs, output):
    _, key, positions, turns, ctx.interleaved, ctx.amplitude, ctx.inverse = inputs
    ctx.has_key = key is not None
    ctx.save_for_backward(positions, turns)


def _rotary_backward(ctx, dq, dk):
    positions, turns = ctx.saved_tensors
    out = torch.ops.flash_sparse_attn._apply_rotary(dq, dk if ctx.has_key else None, positions, turns, ctx.interleaved,
                                                    ctx.amplitude, not ctx.inverse)
    return out[0], out[1] if ctx.has_key else None, None, None, None, None, None


torch.library.register_autograd("flash_sparse_attn::_apply_rotary", _rotary_backward, setup_context=_rotary_setup)
