"""Bookkeeping of the 8-bit cache pool and the kv8 pack on the CPU (no kernel launches)."""
from __future__ import annotations

import pytest
import torch

from oracle import engine as oeng
from specdec_amd import SdvError
from specdec_amd.engine import spec_cache as sc
from specdec_amd.engine.kv8_cache import KV8Cache, KV8LayerPages
from specdec_amd.kernels import patch


@pytest.mark.parametrize("fmt,dtype", [("fp8", torch.float8_e4m3fn), ("int8", torch.int8)])
def test_pool(fmt, dtype):
    pool = KV8Cache(2, 128, kv_format=fmt, num_layers=3, batch=2, num_blocks=4, device="cpu", seed=1)
    assert pool.k_pages.shape == (3, 4, 2, 4, 8, 4, 16) and pool.k_pages.dtype is dtype
    assert pool.v_pages.shape == (3, 4, 2, 128, 16) and pool.v_pages.dtype is dtype
    assert pool.scales.shape == (3, 4, 2, 2, 16) and pool.scales is pool.v_scales
    pool.reserve(0, 40)
    pool.k_pages.view(torch.uint8)[1, pool.blocks[0][2]] = 7
    pool.reserve(1, 100)                                          # the pool grows, its contents stay
    assert pool.alloc.num_blocks >= 10 and bool((pool.k_pages.view(torch.uint8)[1, pool.blocks[0][2]] == 7).all())
    assert pool.logical_bytes_per_token_layer() == 528
    pool.set_length(0, 40)
    pool.set_length(1, 100)
    f = pool.footprint()
    assert f["kv8_bytes"] == 140 * 3 * 528 and f["saved_frac"] == pytest.approx(1 - 528 / 1024)
    assert pool.block_table().shape == (2, 7)
    pool.free_sequence(1)
    assert pool.lengths == [40, 0] and pool.block_table().shape == (2, 3)


def test_pool_refusals():
    with pytest.raises(ValueError):
        KV8Cache(2, 128, kv_format="int4", device="cpu")
    with pytest.raises(ValueError):
        KV8Cache(2, 96, device="cpu")
    pool = KV8Cache(2, 64, batch=2, capacity_tokens=32, device="cpu", growable=False)
    x = torch.zeros((5, 2, 64), dtype=torch.bfloat16)
    for counts in ([5], [5, -1], [1, 1, 1]):
        with pytest.raises(ValueError):
            pool.write(0, x, x, counts)
    with pytest.raises(ValueError):
        pool.write(0, x, x, [2, 3], [0])
    with pytest.raises(ValueError):
        pool.write(0, x, x, [2, 3], [0, -1])
    with pytest.raises(SdvError):
        pool.write(0, x, x, [2, 2])
    with pytest.raises(RuntimeError):
        pool.write(0, x, x, [2, 3], [0, 100])                     # more blocks than there are
    with pytest.raises(SdvError):
        pool.write(0, x, x, [2, 3])                               # CPU tensors: no kernel
    assert pool.lengths == [0, 0]
    with pytest.raises(ValueError):
        pool.read(0, [1, 0])                                      # no tokens there
    q = torch.zeros((2, 4, 1, 64), dtype=torch.bfloat16)
    with pytest.raises(SdvError):
        pool.attend(0, q[0])
    with pytest.raises(SdvError):
        pool.attend(0, q[:1])
    with pytest.raises(SdvError):
        pool.attend(0, x, counts=[2, 2])
    with pytest.raises(SdvError):
        pool.attend(0, q, out=q[:, :2])


def test_layer_dicts_follow_the_cache_api():
    pool = KV8Cache(2, 128, batch=1, capacity_tokens=64, device="cpu", kv_format="int8")
    pool.reserve(0, 37)
    pool.set_length(0, 37)
    cache = [KV8LayerPages(pool).layer_dict(37) for _ in range(2)]
    assert sc.cache_length(cache) == 37 and cache[0]["k"].dtype is torch.int8 and cache[0]["k_scale"].shape == (1, 2, 37, 1)
    sc.check_consistent(cache)
    t = sc.trim_cache(cache, 30)
    assert sc.cache_length(t) == 30 and t[0]["k_scale"].shape[2] == 30 and t[0]["pages"] is cache[0]["pages"]
    with pytest.raises(RuntimeError):
        sc.check_consistent([KV8LayerPages(pool).layer_dict(65)])


def test_pack():
    orig = oeng.SelfAttention.forward
    try:
        assert patch.install("kv8", oeng, kv_format="int8") == "kv8" and patch.current_pack() == "kv8"
        assert oeng.SelfAttention.forward is patch._kv8_forward
        with pytest.raises(ValueError):
            patch.install("kv8", oeng, kv_format="int4")
        model = oeng.tiny_model(3, layers=1, dtype=torch.float32)
        ids = torch.tensor([[5, 9, 1]])
        got, cache = model._run(model.embed_tokens(ids), None)     # the BF16 format: the engine's own forward
        assert "pages" not in cache[0]
        patch.enable_fp8v(model)
        with pytest.raises(SdvError, match="kv8 pack runs on a HIP device"):
            model._run(model.embed_tokens(ids), None)
    finally:
        patch.restore()
    assert oeng.SelfAttention.forward is orig
