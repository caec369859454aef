"""A step recorded before a fork, replayed after it: the source's tokens change, the fork's stay what they were."""
from __future__ import annotations

import pytest
import torch

from conftest import announce
from specdec_amd.engine.kv8_cache import KV8Cache
from specdec_amd.engine.paged_cache import PagedKVCache
from specdec_amd.kernels import ops

pytestmark = pytest.mark.gpu


def _rows(shape, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)


def _held(pool, seq):
    """A sequence's K, V and scales as every layer's gather gives them."""
    return [t.clone() for layer in range(pool.num_layers) for t in pool.gather(layer, seq)]


def _same(one, two):
    as_bytes = lambda t: t.contiguous().view(torch.uint8)  # noqa: E731  (V of the v_fp8 cache may hold any code)
    return all(torch.equal(as_bytes(x), as_bytes(y)) for x, y in zip(one, two))


@pytest.mark.parametrize("rope", [False, True])
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("at,rows", [(30, 5), (20, 24), (3, 1)])
def test_a_recorded_verify(cuda_device, fmt, rope, at, rows):
    dev = cuda_device
    inv, _ = ops.rope_frequencies(128, device=dev)
    pool, eager = (KV8Cache(2, 128, kv_format=fmt, num_layers=2, batch=2, num_blocks=16, device=dev) for _ in range(2))
    k, v = (_rows((50, 2, 128), i).to(dev) for i in (1, 2))
    q, kn, vn = (_rows((rows, n, 128), 3 + i).to(dev) for i, n in enumerate((12, 2, 2)))
    for p in (pool, eager):
        for layer in range(2):
            p.write(layer, k, v, [50, 0], [0, 0])
        p.set_length(0, at)

    def step(p):
        got = [p.append_attend(layer, q, kn, vn, [at, 0], counts=[rows, 0], rope=inv if rope else None) for layer in range(2)]
        return got[1]
    announce(f"a recorded verify {fmt} {rope} {at} {rows}: warm-up")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(pool)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step(pool)
    step(eager)
    graph.replay()
    torch.cuda.synchronize()
    assert pool.lengths == [at + rows, 0] and _same(_held(pool, 0), _held(eager, 0))
    pool.fork(0, 1)
    fork = _held(pool, 1)
    assert _same(fork, _held(eager, 0))
    for turn in range(3):
        for i, t in enumerate((q, kn, vn)):
            t.copy_(_rows(t.shape, 20 + 3 * turn + i))
        announce(f"a recorded verify {fmt} {rope} {at} {rows}: replay {turn}")
        graph.replay()
        eager.set_length(0, at)
        want = step(eager)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and _same(_held(pool, 0), _held(eager, 0))
        assert _same(_held(pool, 1), fork)
        torch.full((1 << 20,), float("nan"), device=dev)


def test_a_recorded_prefill(cuda_device):
    dev = cuda_device
    pool, eager = (PagedKVCache(2, 64, batch=2, num_blocks=16, device=dev) for _ in range(2))
    k, v = (_rows((40, 2, 64), i).to(dev) for i in (1, 2))
    announce("a recorded prefill: warm-up")
    slots = pool.prefill(0, k, v, [40, 0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pool.prefill(0, k, v, [40, 0], slots=slots)
    pool.fork(0, 1)
    fork = _held(pool, 1)
    for turn in range(3):
        for i, t in enumerate((k, v)):
            t.copy_(_rows(t.shape, 20 + 2 * turn + i))
        announce(f"a recorded prefill: replay {turn}")
        graph.replay()
        eager.prefill(0, k, v, [40, 0])
        torch.cuda.synchronize()
        assert _same(_held(pool, 0), _held(eager, 0)) and _same(_held(pool, 1), fork)
