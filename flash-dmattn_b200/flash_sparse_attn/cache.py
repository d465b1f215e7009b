"""Serving from a paged cache in 8 bits: block tables and slot maps made on the GPU, the cache's writer, and attention over it.

    tables = block_tables(requests=64, blocks_per_request=1024, num_blocks=20000, device="cuda")   # one for all layers
    caches = [quantized_cache(20000, kv_heads, head_dim, device="cuda") for _ in layers]
    ...
    step = tables.extend(new_lengths, total_tokens)             # once per step: blocks for the new tokens, the step's plan
    q = cache_append(cache, tables, step, k, v, query=q, frequencies=freqs)     # per layer: turned, rounded, written
    out = flash_sparse_attn_cache_func(q, cache, tables, step)                  # per layer
    ...
    tables.truncate(lengths)                                    # drafts that were rejected, requests that are done (length 0)

None of these synchronises; a whole step can be captured into a CUDA graph and replayed with new contents of `new_lengths` and the
activations. The reference's packed-sequence call has a `block_table` argument for 16-bit caches
(flash_sparse_attn/flash_sparse_attn_interface.py:687-790); it has no 8-bit cache.
"""
from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _native
from .rotary import RotaryFrequencies
from .utils.mask import KeptKeys
from .window import check_window

__all__ = ["BlockTables", "CacheStep", "QuantizedCache", "block_tables", "quantized_cache", "cache_append",
           "flash_sparse_attn_cache_func"]


class CacheStep(NamedTuple):
    """The plan of a step, from `BlockTables.extend`: the same for all layers."""

    cu_seqlens: torch.Tensor  # int32 (requests + 1,): first of each request's tokens among the step's
    positions: torch.Tensor   # int32 (tokens,): position of each token in its request; 0 behind the last one
    slots: torch.Tensor       # int64 (tokens,): block * block_size + place in the block; -1 where there is none
    lengths: torch.Tensor     # int32 (requests,): tokens that each request holds now
    granted: torch.Tensor     # bool (requests,): False where a request got no blocks
    cu_blocks: torch.Tensor   # int32 (requests + 1,): blocks that the step's tokens go to, summed up
    cu_chunks: torch.Tensor   # int32 (requests + 1,): 64-token pieces of the requests with tokens in this step, summed up


class BlockTables(NamedTuple):
    """Which blocks of a cache each request holds, a block one request. The tensors live on the GPU and are updated in place, in stream
    order; two calls on the same tables must not run at once."""

    table: torch.Tensor       # int32 (requests, blocks per request): a request's blocks in order, -1 behind them
    lengths: torch.Tensor     # int32 (requests,): tokens that each request holds
    free: torch.Tensor        # int32 (num_blocks,): the first free_count entries are the blocks nobody holds
    free_count: torch.Tensor  # int32 (1,)
    ticket: torch.Tensor      # int32 (1,): scratch, 0 between calls
    block_size: int = 64

    def extend(self, new_lengths: torch.Tensor, total_tokens: int) -> CacheStep:
        """Gives request r new_lengths[r] more tokens (int32 on the GPU; 0: none in this step) and the blocks these need.
        total_tokens: tokens of the step's activations, at least the sum of new_lengths (more: a padded step). A request that
        would outgrow its table row or total_tokens, or for which no blocks are left, is refused: it keeps what it has,
        `step.granted` is False, its tokens are written nowhere and their attention is 0. Requests are served in order, and behind
        one for which no blocks were left none gets any, however few it asks for."""
        native = _native.load()
        args = (self.table, self.lengths, self.free, self.free_count, self.ticket, new_lengths)
        out = None
        if not torch.compiler.is_compiling():
            out = native.tables_extend(args, self.block_size, total_tokens)
        if out is None:
            out = torch.ops.flash_sparse_attn._tables_extend(*args, self.block_size, total_tokens)
        return CacheStep(*out)

    def truncate(self, lengths: torch.Tensor) -> None:
        """Requests keep their first lengths[r] tokens (int32 on the GPU; no less than they have: nothing changes; 0: the request
        is done). Blocks no longer needed are free again; taking back what `extend` gave restores the free list as it was."""
        native = _native.load()
        args = (self.table, self.lengths, self.free, self.free_count, self.ticket, lengths)
        if torch.compiler.is_compiling() or not native.tables_truncate(args, self.block_size):
            torch.ops.flash_sparse_attn._tables_truncate(*args, self.block_size)


class QuantizedCache(NamedTuple):
    """Keys and values of one layer in 8 bits: a value is its e4m3 number times the scale of its block and head."""

    k: torch.Tensor        # float8_e4m3fn (num_blocks, kv heads, block size, head dim)
    v: torch.Tensor
    k_scale: torch.Tensor  # float32 (num_blocks, kv heads), powers of two
    v_scale: torch.Tensor


def _check_block_size(block_size):
    if block_size not in (16, 32, 64, 128):
        raise ValueError(f"block_size must be 16, 32, 64 or 128, got {block_size}.")


def block_tables(requests: int, blocks_per_request: int, num_blocks: int, block_size: int = 64,
                 device: Union[str, torch.device] = "cuda") -> BlockTables:
    """Tables of `requests` requests (1 to 8192) that hold nothing yet; all blocks are free."""
    _check_block_size(block_size)
    if not 0 < requests <= 8192 or blocks_per_request <= 0 or num_blocks <= 0:
        raise ValueError("block_tables needs 1 to 8192 requests, and blocks.")

    def zeros(*shape):
        return torch.zeros(shape, dtype=torch.int32, device=device)

    return BlockTables(zeros(requests, blocks_per_request) - 1, zeros(requests),
                       torch.arange(num_blocks - 1, -1, -1, dtype=torch.int32, device=device), zeros(1) + num_blocks, zeros(1),
                       block_size)


def quantized_cache(num_blocks: int, kv_heads: int, head_dim: int, block_size: int = 64,
                    device: Union[str, torch.device] = "cuda") -> QuantizedCache:
    """An empty cache of one layer. Head dims that are multiples of 16, up to 256."""
    _check_block_size(block_size)
    if num_blocks <= 0 or kv_heads <= 0 or head_dim <= 0 or head_dim % 16 or head_dim > 256:
        raise ValueError("quantized_cache needs blocks, heads, and a head_dim that is a multiple of 16 up to 256.")
    shape = (num_blocks, kv_heads, block_size, head_dim)
    k, v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2))
    return QuantizedCache(k, v, *(torch.ones(shape[:2], dtype=torch.float32, device=device) for _ in range(2)))


def _cache_args(cache: QuantizedCache, tables: BlockTables, step: CacheStep):
    if cache.k.dim() == 4 and cache.k.shape[2] != tables.block_size:
        raise RuntimeError("the cache and the tables are of different block sizes")
    return (cache.k, cache.v, cache.k_scale, cache.v_scale, tables.table, step.cu_seqlens, step.positions, step.lengths,
            step.cu_blocks, step.cu_chunks)


def cache_append(
    cache: QuantizedCache,
    tables: BlockTables,
    step: CacheStep,
    key: torch.Tensor,
    value: torch.Tensor,
    query: Optional[torch.Tensor] = None,
    frequencies: Optional[RotaryFrequencies] = None,
) -> Optional[torch.Tensor]:
    """Writes the step's key and value (tokens, kv heads, d; bf16 or fp16) into the cache, in one launch.

    The scale of a block and head is the smallest power of two (at least 2^-100) whose 448-fold reaches the largest finite
    magnitude written to it, or, where the block holds earlier tokens of the request, the scale that it has if that is larger; if it
    grows, the earlier tokens are rounded to it once more. Infinities become +-448 scales, NaN stays NaN. Everything else in
    the cache is left as it is. Two requests must not hold one block that is not full yet.

    frequencies: keys are turned by their positions (step.positions) before they are rounded, as `apply_rotary` does, and so is
    query (tokens, heads, d), which is returned; without a query the result is None."""
    args = _cache_args(cache, tables, step)
    turns, interleaved, amplitude = frequencies if frequencies is not None else (None, False, 1.0)
    args = args + (key, value, query, turns)
    if not torch.compiler.is_compiling():
        out = _native.load().cache_append(args, interleaved, amplitude)
        if out is not None:
            return out[0]
    out = torch.ops.flash_sparse_attn._cache_append(*args, interleaved, amplitude)
    return out if query is not None else None


def flash_sparse_attn_cache_func(
    query: torch.Tensor,
    cache: QuantizedCache,
    tables: BlockTables,
    step: CacheStep,
    attn_mask: Optional[Union[KeptKeys, torch.Tensor]] = None,
    attn_bias: Optional[torch.Tensor] = None,
    softmax_scale: Optional[float] = None,
    is_causal: bool = True,
    max_seqlen_q: Optional[int] = None,
    max_seqlen_k: Optional[int] = None,
    sliding_window: Optional[int] = None,
    sink_tokens: int = 0,
) -> torch.Tensor:
    """Attention of the step's queries over the cache, after `cache_append` has written the step's keys and values.

    query (tokens, H, d), bf16 or fp16, H a multiple of the cache's heads. Query i of a request with n new tokens of L sees the
    keys at positions up to L - n + i (is_causal=False: all L). attn_mask: the dynamic mask of one row per request and kv head,
    a `KeptKeys` ({1|requests}, {1|Hk}) or a bool tensor ({1|requests}, {1|Hk}, 1, keys), False or beyond its keys = masked out.
    attn_bias ({1|requests}, {1|Hk|H}, 1, keys), dtype of query, added to the scaled scores; 0 beyond its keys. softmax_scale
    defaults to d ** -0.5. max_seqlen_q, max_seqlen_k: bounds on the new tokens and on the length of any request, where the
    host knows them (default: the step's tokens, the tables' width). They choose how the work is split and how much scratch a call
    takes: pass them where you can. Where a request goes beyond them, its queries from max_seqlen_q on are 0 (the first always counts), and
    keys from max_seqlen_k on are not seen; queries' positions stay those in the whole request.
    sliding_window, sink_tokens: as in `flash_sparse_attn_window_func`, of the keys seen so far a query sees the last sliding_window, its own
    among them, and those at positions below sink_tokens. Blocks that nobody sees are not read, so that a step's time goes with the window
    (with attn_mask: with the mask); the requests keep them.

    Returns (tokens, H, d). Rows of tokens behind the last request, of refused requests and of queries that see no key are 0. A key or
    value that is NaN reaches the queries that see it and no others.
    Scores, probabilities' sums and outputs are accumulated in 32 bits. Probabilities enter the second product in fp16 (2^-11 of
    themselves). Requests with 32 or more new tokens, without mask or bias, have their keys converted to the query's type where the step
    has enough work for it; their probabilities are of that type (bf16: 2^-9). So what else is in a step can change how a result is
    rounded. The conversion takes up to 2^20 keys, counted as requests that can have so many new tokens times max_seqlen_k, and 4 GiB
    of scratch: a call whose bounds allow for more reads the 8 bits, as one does that comes upon NaN in a value or numbers that 16 bits do not hold.
    There are no gradients: a call that would need them raises."""
    args = _cache_args(cache, tables, step)
    window = 0
    if sliding_window is not None:
        check_window(sliding_window, sink_tokens)
        if not is_causal:
            raise ValueError("sliding_window needs is_causal=True")
        window = sliding_window
    elif sink_tokens:
        raise ValueError("sink_tokens needs a sliding_window")
    key_pos = count = None
    if isinstance(attn_mask, KeptKeys):
        key_pos, count = attn_mask.key_pos, attn_mask.count
    elif attn_mask is not None:
        tag = None if torch.compiler.is_compiling() else getattr(attn_mask, "_fdma_kept", None)
        if tag is not None and tag[1] == attn_mask._version:
            key_pos, count = tag[0].key_pos, tag[0].count
        else:
            if attn_mask.dtype != torch.bool or attn_mask.dim() != 4 or attn_mask.shape[2] != 1:
                raise RuntimeError("attn_mask must be a KeptKeys or a bool tensor ({1|requests}, {1|num_heads_k}, 1, keys)")
            from .compaction import index_kept_keys

            m = attn_mask[:, :, 0]
            key_pos, count, _ = index_kept_keys(m if m.stride(-1) == 1 else m.contiguous(), m.shape[-1], False)
    max_q = query.shape[0] if max_seqlen_q is None else max_seqlen_q
    max_k = tables.table.shape[-1] * tables.block_size if max_seqlen_k is None else max_seqlen_k
    args = args + (query, key_pos, count, attn_bias)
    if not torch.compiler.is_compiling():
        out = _native.load().cache_attention(args, softmax_scale, is_causal, max_q, max_k, window, sink_tokens)
        if out is not None:
            return out
    return torch.ops.flash_sparse_attn._cache_attention(*args, softmax_scale, is_causal, max_q, max_k, window, sink_tokens)


# ---- the same as custom operators, for tracing -------------------------------------------------------------------------
def _plain(result, what):
    if result is None:
        raise RuntimeError(f"{what}: these tensors are not supported")
    return result


@torch.library.custom_op("flash_sparse_attn::_tables_extend", mutates_args=("table", "lengths", "free_count", "ticket"),
                         device_types="cuda")
def _tables_extend(table: torch.Tensor, lengths: torch.Tensor, free: torch.Tensor, free_count: torch.Tensor, ticket: torch.Tensor,
                   new_lengths: torch.Tensor, block_size: int, total_tokens: int) -> Tuple[
                       torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    out = _plain(_native.load().tables_extend((table, lengths, free, free_count, ticket, new_lengths), block_size, total_tokens),
                 "extend")
    return tuple(t.clone() for t in out)  # (parts of one buffer, which an operator must not return)


@torch.library.register_fake("flash_sparse_attn::_tables_extend")
def _tables_extend_fake(table, lengths, free, free_count, ticket, new_lengths, block_size, total_tokens):
    def new(n, dtype=torch.int32):
        return torch.empty((n,), dtype=dtype, device=table.device)

    R = table.shape[0]
    return new(R + 1), new(total_tokens), new(total_tokens, torch.int64), new(R), new(R, torch.bool), new(R + 1), new(R + 1)


@torch.library.custom_op("flash_sparse_attn::_tables_truncate",
                         mutates_args=("table", "lengths", "free", "free_count", "ticket"), device_types="cuda")
def _tables_truncate(table: torch.Tensor, lengths: torch.Tensor, free: torch.Tensor, free_count: torch.Tensor,
                     ticket: torch.Tensor, new_lengths: torch.Tensor, block_size: int) -> None:
    if not _native.load().tables_truncate((table, lengths, free, free_count, ticket, new_lengths), block_size):
        raise RuntimeError("truncate: these tensors are not supported")


@torch.library.register_fake("flash_sparse_attn::_tables_truncate")
def _tables_truncate_fake(table, lengths, free, free_count, ticket, new_lengths, block_size):
    return None


@torch.library.custom_op("flash_sparse_attn::_cache_append", mutates_args=("k", "v", "k_scale", "v_scale"), device_types="cuda")
def _cache_append(k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, table: torch.Tensor,
                  cu_seqlens: torch.Tensor, positions: torch.Tensor, lengths: torch.Tensor, cu_blocks: torch.Tensor,
                  cu_chunks: torch.Tensor, key: torch.Tensor, value: torch.Tensor, query: Optional[torch.Tensor],
                  turns: Optional[torch.Tensor], interleaved: bool, amplitude: float) -> torch.Tensor:
    out = _plain(_native.load().cache_append((k, v, k_scale, v_scale, table, cu_seqlens, positions, lengths, cu_blocks, cu_chunks, key,
                                              value, query, turns), interleaved, amplitude), "cache_append")[0]
    return out if out is not None else key.new_empty((0,))


@torch.library.register_fake("flash_sparse_attn::_cache_append")
def _cache_append_fake(k, v, k_scale, v_scale, table, cu_seqlens, positions, lengths, cu_blocks, cu_chunks, key, value, query,
                       turns, interleaved, amplitude):
    return key.new_empty((0,)) if query is None else torch.empty(query.shape, dtype=query.dtype, device=query.device)


@torch.library.custom_op("flash_sparse_attn::_cache_attention", mutates_args=(), device_types="cuda")
def _cache_attention(k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, table: torch.Tensor,
                     cu_seqlens: torch.Tensor, positions: torch.Tensor, lengths: torch.Tensor, cu_blocks: torch.Tensor,
                     cu_chunks: torch.Tensor, query: torch.Tensor, key_pos: Optional[torch.Tensor], count: Optional[torch.Tensor],
                     bias: Optional[torch.Tensor], softmax_scale: Optional[float], is_causal: bool, max_seqlen_q: int,
                     max_seqlen_k: int, window: int = 0, sinks: int = 0) -> torch.Tensor:
    return _plain(_native.load().cache_attention((k, v, k_scale, v_scale, table, cu_seqlens, positions, lengths, cu_blocks, cu_chunks,
                                                  query, key_pos, count, bias), softmax_scale, is_causal, max_seqlen_q, max_seqlen_k,
                                                 window, sinks),
                  "flash_sparse_attn_cache_func")


@torch.library.register_fake("flash_sparse_attn::_cache_attention")
def _cache_attention_fake(k, v, k_scale, v_scale, table, cu_seqlens, positions, lengths, cu_blocks, cu_chunks, query, key_pos, count,
                          bias, softmax_scale, is_causal, max_seqlen_q, max_seqlen_k, window=0, sinks=0):
    return torch.empty(query.shape, dtype=query.dtype, device=query.device)
