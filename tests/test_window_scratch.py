"""Scratch of the windowed backward on packed sequences: it goes with the tokens, however many sequences and sinks there are (no GPU needed)."""
import ctypes

import pytest

from flash_sparse_attn import _lib
from test_cabi_windows_and_drafts import entry, params


@pytest.mark.parametrize("sequences,length,h,h_k,d,window,sinks", [
    (200, 500, 32, 8, 128, 100, 4096), (200, 500, 32, 8, 128, 1, 100000), (1000, 50, 32, 8, 128, 256, 64), (1000, 50, 32, 8, 128, 16, 64),
    (100000, 5, 8, 2, 64, 3, 1000), (1, 32768, 32, 8, 128, 2048, 4), (3, 20000, 16, 4, 64, 300, 130)])
def test_packed_sequences(sequences, length, h, h_k, d, window, sinks):
    tokens = sequences * length
    p = params(_lib.BwdParams, h=h, h_k=h_k, d=d, seqlen_q=tokens, seqlen_k=tokens)
    for t, heads in (("q", h), ("k", h_k), ("v", h_k), ("o", h)):
        setattr(p.f, f"{t}_row_stride", heads * d), setattr(p.f, f"{t}_head_stride", d), setattr(p.f, f"{t}_batch_stride", tokens * heads * d)
    for t, heads in (("do", h), ("dq", h), ("dk", h_k), ("dv", h_k)):
        setattr(p, f"{t}_row_stride", heads * d), setattr(p, f"{t}_head_stride", d), setattr(p, f"{t}_batch_stride", tokens * heads * d)
    size = entry("fdma_bwd_window_workspace_bytes", ctypes.c_size_t)
    got = size(ctypes.byref(p), window, sinks, sequences)
    kept = 2 * (tokens + 128) * h_k * d * 4  # dK and dV in 32 bits
    vectors = 2 * (tokens + 64) * h * 4      # LSE and D
    # sums of the key tiles and of the sinks' first parts, and the sinks' rows of each further part of the queries
    parts = -(-tokens // 2048) - 1
    assert 0 < got <= 2 * kept + vectors + 2 * parts * min(sinks, tokens) * h_k * d * 4 + 4096
    # as one sequence the same tokens take no less than a part of that
    assert got <= 3 * size(ctypes.byref(p), window, sinks, 1) + 4096


def test_nobody_beyond_the_window():
    """No sequence can be longer than the window: the sinks cost nothing."""
    p = params(_lib.BwdParams)  # 500 tokens
    size = entry("fdma_bwd_window_workspace_bytes", ctypes.c_size_t)
    for n in (0, 1, 50):
        assert size(ctypes.byref(p), 400, 90, n) == size(ctypes.byref(p), 400, 0, n)
