"""Two host threads that call one operator with different sizes at once, each on a stream of its own: kernels whose shared memory depends
on the call must not take it from one another, and results are those of the calls one by one."""
import threading

import pytest
import torch

import flash_sparse_attn as fsa
from test_gpu_cache import dev, ints  # noqa: F401

pytestmark = pytest.mark.gpu


def at_once(calls, times=300):
    """Each call in a thread of its own, `times` times; what it returns last, or its exception."""
    out, start = [None] * len(calls), threading.Barrier(len(calls))

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait(timeout=60)
                for _ in range(times):
                    out[i] = calls[i]()
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            out[i] = e

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for x in out:
        if isinstance(x, Exception):
            raise x
    return out


def equal(a, b):
    return all(torch.equal(x.float(), y.float()) for x, y in zip(a, b))


def test_append(dev):  # noqa: F811
    def make(d):
        tables, cache = fsa.block_tables(1, 2, 2, 128, device=dev), fsa.quantized_cache(2, 1, d, 128, device=dev)
        step = tables.extend(ints([200], dev), 200)
        x = torch.randn((200, 1, d), device=dev, dtype=torch.bfloat16)
        f = fsa.rotary_frequencies(d, device=dev)
        return lambda: (fsa.cache_append(cache, tables, step, x, x, query=x, frequencies=f), *cache)

    calls = [make(256), make(128)]
    want = [[t.clone() for t in call()] for call in calls]
    torch.cuda.synchronize()
    for got, w in zip(at_once(calls), want):
        assert equal(got, w)


def test_tables(dev):  # noqa: F811
    def make(requests):
        tables, new = fsa.block_tables(requests, 1, requests, 16, device=dev), torch.ones(requests, dtype=torch.int32, device=dev)

        def call():
            step = tables.extend(new, requests)
            tables.truncate(new - 1)
            return step

        return call

    calls = [make(8192), make(4000)]
    want = [[t.clone() for t in call()] for call in calls]
    torch.cuda.synchronize()
    for got, w in zip(at_once(calls), want):
        assert equal(got, w)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rotary(dev, dtype):  # noqa: F811
    def make(d):
        x, f = torch.randn((4, 2, d), device=dev).to(dtype), fsa.rotary_frequencies(d, device=dev)
        return lambda: fsa.apply_rotary(x, x, f)

    calls = [make(4096), make(2048)]
    want = [[t.clone() for t in call()] for call in calls]
    torch.cuda.synchronize()
    for got, w in zip(at_once(calls), want):
        assert equal(got, w)
