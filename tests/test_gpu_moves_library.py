"""torch.ops.sdv.* of positions, page moves and shared prefixes on the GPU: torch.library.opcheck (schema, fake tensors, AOT
dispatch) on small real inputs, and torch.compile(fullgraph=True) of a layer's step giving the eager bits."""
from __future__ import annotations

import pytest
import torch

from conftest import announce
from specdec_amd.engine.kv8_cache import KV8Cache
from specdec_amd.kernels import ops

pytestmark = pytest.mark.gpu


def _pool(dev):  # INT8: opcheck compares mutated arguments by arithmetic that E4M3FN tensors have none of
    pool = KV8Cache(2, 128, kv_format="int8", num_layers=2, batch=3, num_blocks=24, device=dev, seed=3)
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn((6, n, 128), generator=g).to(torch.bfloat16).to(dev) for n in (12, 2, 2))
    x = torch.randn((60, 2, 128), generator=g).to(torch.bfloat16).to(dev)
    for layer in range(2):
        pool.prefill(layer, x, x, [60, 0, 0])
    pool.fork(0, [1, 2])
    pool.reserve_all(70)
    return pool, q, k, v, ops.rope_frequencies(128, device=dev)[0]


def _ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def test_opcheck(cuda_device):
    dev = cuda_device
    pool, q, k, v, inv = _pool(dev)
    pages, bt, cu, lens = pool.layer(0), pool.block_table(), _ints([0, 1, 3, 6], dev), _ints([61, 62, 63], dev)
    pos = _ints([60, 60, 61, 60, 61, 61], dev)
    for name, args in {
        "rope": (q, k, pos, inv, True, 0.5),
        "kv8_rope_append": (q, k, v, *pages, bt, cu, lens, 63, inv, False, 1.0, pos),
        "copy_blocks": (pool.k_pages, pool.v_pages, pool.scales, _ints([0, 1], dev), _ints([20, 21], dev)),
        "kv8_keep": (pool.k_pages, pool.v_pages, pool.scales, bt, _ints([0, 0, 1, 3], dev), _ints([1, 0, 2], dev), _ints([60, 60, 60], dev)),
        "kv8_shared_attention": (q, *pages, bt, cu, lens, 3, 63, _ints([0, 3], dev), _ints([48] * 3, dev), 48, None, None, 32),
    }.items():
        announce(f"opcheck sdv::{name}")
        torch.library.opcheck(getattr(torch.ops.sdv, name).default, args)


def test_compiled_step(cuda_device):
    dev = cuda_device
    one, q, k, v, inv = _pool(dev)
    two = _pool(dev)[0]
    cu, lens, prefix, groups = _ints([0, 1, 3, 6], dev), _ints([61, 62, 63], dev), _ints([48] * 3, dev), _ints([0, 3], dev)

    def step(q, k, v, kp, vp, sc, bt):
        turned = torch.ops.sdv.kv8_rope_append(q, k, v, kp, vp, sc, bt, cu, lens, 63, inv)
        return torch.ops.sdv.kv8_shared_attention(turned, kp, vp, sc, bt, cu, lens, 3, 63, groups, prefix, 48, None, None, 128)

    announce("torch.compile of a step of forks")
    want = step(q, k, v, *one.layer(0), one.block_table())
    got = torch.compile(step, fullgraph=True, backend="aot_eager")(q, k, v, *two.layer(0), two.block_table())
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    for a, b in zip(one.layer(0), two.layer(0)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
