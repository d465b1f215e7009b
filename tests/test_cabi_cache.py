"""C entry points of the rotary positions, the block tables and the 8-bit cache: wrong parameter blocks are refused with a status
before a device is touched (no GPU needed)."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest

from flash_sparse_attn import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "fdma.h")


def struct_fields(name):
    """(type, field) pairs of a struct of the header, in order."""
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    body = re.search(r"typedef struct " + name + r" \{(.*?)\} " + name + ";", text, flags=re.S).group(1)
    fields = []
    for line in body.split(";"):
        line = " ".join(line.split())
        if not line:
            continue
        kind, names = re.match(r"((?:const )?\w+)\s*(.*)", line).groups()
        for n in names.split(","):
            n = n.strip()
            fields.append(("*" if "*" in n else kind, n.replace("*", "").strip()))
    return fields


def mirror(name, known):
    kinds = {"*": ctypes.c_void_p, "int32_t": ctypes.c_int32, "int64_t": ctypes.c_int64, "float": ctypes.c_float, "size_t": ctypes.c_size_t,
             "uint32_t": ctypes.c_uint32, **known}
    return type(name, (ctypes.Structure,), {"_fields_": [(f, kinds[k]) for k, f in struct_fields(name)]})


Rotary = mirror("fdma_rotary_params", {})
Tables = mirror("fdma_tables_params", {})
Cache = mirror("fdma_cache", {})
Append = mirror("fdma_cache_append_params", {"fdma_cache": Cache})
Attention = mirror("fdma_cache_attention_params", {"fdma_cache": Cache})
BUF = ctypes.create_string_buffer(4096)
ADDR = (ctypes.addressof(BUF) + 255) // 256 * 256


def call(name, p):
    fn = getattr(_lib.load(), name)
    fn.restype, fn.argtypes = ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p]
    return fn(ctypes.byref(p) if p is not None else None, None)


def fill(p, pointers, **values):
    for f in pointers:
        setattr(p, f, ADDR)
    for k, v in values.items():
        setattr(p, k, v)
    return p


def cache(**change):
    c = fill(Cache(), ["k", "v", "k_scale", "v_scale", "table", "cu_seqlens", "lengths", "cu_blocks", "cu_chunks", "positions"], requests=1,
             width=1, num_blocks=1, block_size=16, tokens=1, h_k=1, d=64)
    for k, v in change.items():
        setattr(c, k, v)
    return c


def test_null():
    for name in ("fdma_rotary", "fdma_tables_extend", "fdma_tables_truncate", "fdma_cache_append", "fdma_cache_attention"):
        assert call(name, None) == -1
    fn = _lib.load().fdma_cache_attention_workspace_bytes
    fn.restype, fn.argtypes = ctypes.c_size_t, [ctypes.c_void_p]
    assert fn(None) == 0


@pytest.mark.parametrize("change,status", [
    ({}, 0), (dict(q=None), -1), (dict(turns=None), -1), (dict(h=0), -1), (dict(b=-1), -1), (dict(h_k=1), -1), (dict(rotary_dim=0), -1),
    (dict(rotary_dim=7), -1), (dict(rotary_dim=66), -1), (dict(positions=ADDR, position_bits=16), -1), (dict(d=8192, rotary_dim=8192), -2),
    (dict(h=1 << 19), -2), (dict(b=1, seqlen=1, dtype=3), -2)])
def test_rotary(change, status):
    p = fill(Rotary(), ["q", "q_out", "turns"], b=0, seqlen=0, h=1, d=64, rotary_dim=64)  # no tokens: nothing is launched
    for k, v in change.items():
        setattr(p, k, v)
    assert call("fdma_rotary", p) == status


@pytest.mark.parametrize("change,status", [
    (dict(table=None), -1), (dict(ticket=None), -1), (dict(new_lengths=None), -1), (dict(requests=-1), -1), (dict(width=0), -1),
    (dict(num_blocks=0), -1), (dict(tokens=-1), -1), (dict(block_size=48), -2), (dict(requests=8193), -2), (dict(width=1 << 30), -2)])
def test_tables(change, status):
    p = fill(Tables(), ["table", "lengths", "free_list", "free_count", "ticket", "new_lengths", "cu_seqlens", "positions", "slots",
                        "lengths_after", "granted", "cu_blocks", "cu_chunks"], requests=1, width=1, num_blocks=1, block_size=16, tokens=1)
    for k, v in change.items():
        setattr(p, k, v)
    assert call("fdma_tables_extend", p) == status
    assert call("fdma_tables_truncate", p) == status


def test_plan_fields():
    p = fill(Tables(), ["table", "lengths", "free_list", "free_count", "ticket", "new_lengths"], requests=1, width=1, num_blocks=1,
             block_size=16, tokens=1)
    assert call("fdma_tables_extend", p) == -1
    p.requests = 0
    assert call("fdma_tables_truncate", p) == 0


WRONG_CACHE = [(dict(k=None), -1), (dict(v_scale=None), -1), (dict(table=None), -1), (dict(cu_chunks=None), -1), (dict(width=0), -1),
               (dict(h_k=0), -1), (dict(d=0), -1), (dict(tokens=-1), -1), (dict(block_size=8), -2), (dict(d=72), -2), (dict(d=272), -2),
               (dict(k=ADDR + 8), -2), (dict(width=1 << 28), -2)]


@pytest.mark.parametrize("change,status", WRONG_CACHE)
def test_cache_of_both(change, status):
    a = fill(Append(), ["key", "value"], c=cache(**change))
    assert call("fdma_cache_append", a) == status
    b = fill(Attention(), ["query", "out"], c=cache(**change), h=1, max_seqlen_q=1, max_seqlen_k=1)
    assert call("fdma_cache_attention", b) == status


@pytest.mark.parametrize("change,status", [
    (dict(key=None), -1), (dict(value=None), -1), (dict(turns=ADDR), -1), (dict(turns=ADDR, rotary_dim=66), -1),
    (dict(turns=ADDR, rotary_dim=64, query=ADDR), -1), (dict(dtype=2), -2)])
def test_append(change, status):
    p = fill(Append(), ["key", "value"], c=cache())
    for k, v in change.items():
        setattr(p, k, v)
    assert call("fdma_cache_append", p) == status
    p.c = cache(tokens=0)
    assert call("fdma_cache_append", p) == 0  # nothing to write: nothing is looked at


@pytest.mark.parametrize("change,status", [
    (dict(query=None), -1), (dict(out=None), -1), (dict(h=0), -1), (dict(max_seqlen_q=-1), -1), (dict(max_seqlen_k=-1), -1),
    (dict(bias=ADDR, h_bias=3, bias_keys=1), -1), (dict(bias=ADDR, h_bias=1, bias_keys=0), -1), (dict(kept_pos=ADDR, kept_capacity=0), -1),
    (dict(dtype=2), -2), (dict(out=ADDR + 2), -2), (dict(out_row_stride=3), -2), ({}, -3), (dict(workspace=ADDR + 16, workspace_bytes=1 << 30), -3)])
def test_attention(change, status):
    p = fill(Attention(), ["query", "out"], c=cache(requests=500), h=1, max_seqlen_q=1, max_seqlen_k=1, softmax_scale=1.0)
    for k, v in change.items():
        setattr(p, k, v)
    assert call("fdma_cache_attention", p) == status


def test_workspace_of_few_requests():
    fn = _lib.load().fdma_cache_attention_workspace_bytes
    fn.restype, fn.argtypes = ctypes.c_size_t, [ctypes.c_void_p]
    for requests, some in ((1, False), (500, True)):
        p = fill(Attention(), ["query", "out"], c=cache(requests=requests), h=1, max_seqlen_q=1, max_seqlen_k=1, softmax_scale=1.0)
        assert (fn(ctypes.byref(p)) > 0) == some


def test_heads_must_divide():
    p = fill(Attention(), ["query", "out"], c=cache(h_k=2), h=3, max_seqlen_q=1, max_seqlen_k=1)
    assert call("fdma_cache_attention", p) == -1


def test_layout_of_the_parameter_blocks(tmp_path):
    """The mirrors above, read from the header's text, have the sizes that a C compiler gives."""
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no gcc")
    pairs = {c.__name__: c for c in (Rotary, Tables, Cache, Append, Attention)}
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "fdma.h"\nint main(void) {\n' +
                   "".join(f'printf("{n} %zu\\n", sizeof({n}));\n' for n in pairs) + "return 0; }\n")
    exe = tmp_path / "sizes"
    subprocess.run([gcc, "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()
    for n, size in zip(out[::2], out[1::2]):
        assert ctypes.sizeof(pairs[n]) == int(size), n
