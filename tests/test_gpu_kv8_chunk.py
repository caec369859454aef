"""The kv8 attention kernel for many rows at sizes that a call with its own max_seq_len gives to the kernel
for few: the announced length is far above the sequences', so that the call counts as a long one."""
from __future__ import annotations

import math

import pytest
import torch

import kv8_reference as ref
from conftest import announce
from specdec_amd.kernels import ops
from test_gpu_kv8 import HEADS, _cu, _filled, _gen, _ints, _random_tree, _rows

pytestmark = pytest.mark.gpu
# one long sequence's tiles are units of a workgroup each (32768), or ranges (131072, or several sequences)
LENGTHS = [32768, 131072]


def _long(dev, heads, fmt, lens, new, length, seed=1, tree=None, pages=None, bt=None):
    h, kv, d = heads
    if pages is None:
        pages, bt = _filled(kv, d, fmt, lens, seed)
    q = torch.randn((sum(new), h, d), generator=_gen(seed + 7)).to(torch.bfloat16)
    got = ops.kv8_attention(q.to(dev), *pages.to(dev), bt.to(dev), _cu(new, dev), _ints(lens, dev), max(new), length,
                            tree_mask=None if tree is None else tree.to(dev))
    torch.cuda.synchronize()
    ref.within(got, *ref.attention(q, pages, bt, new, lens, None, tree))
    return got


@pytest.mark.parametrize("length", LENGTHS)
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("heads", list(HEADS))
@pytest.mark.parametrize("new,lens", [([33], [33]), ([34], [500]), ([65], [64 + 65]), ([300], [300]), ([257], [1025]), ([40, 0, 1, 90], [40, 9, 333, 95]),
                                      ([1, 1, 64, 2], [700, 1, 64, 65])])
def test_rows(cuda_device, length, fmt, heads, new, lens):
    announce(f"kv8 attention, many rows {fmt} {heads} {new} {lens} {length}")
    _long(cuda_device, HEADS[heads], fmt, lens, new, length)


@pytest.mark.parametrize("length", LENGTHS)
@pytest.mark.parametrize("heads", ["target", "draft"])
@pytest.mark.parametrize("new,lens", [([24], [500]), ([64], [64]), ([64, 3, 20], [1000, 70, 33])])
def test_tree(cuda_device, length, heads, new, lens):
    announce(f"kv8 attention, many rows of a tree {heads} {new} {lens} {length}")
    _long(cuda_device, HEADS[heads], "int8", lens, new, length, tree=_random_tree(new, 3))


@pytest.mark.parametrize("length", LENGTHS)
@pytest.mark.parametrize("new,lens", [([40, 10, 1], [2, 4, 0]), ([64], [10]), ([50, 40], [0, 0])])
def test_rows_that_see_nothing(cuda_device, length, new, lens):
    announce(f"kv8 attention, many rows that see nothing {new} {lens} {length}")
    _long(cuda_device, HEADS["target"], "fp8", lens, new, length)


@pytest.mark.parametrize("length", LENGTHS)
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_tokens_that_are_not_finite(cuda_device, length, fmt):
    h, kv, d = HEADS["target"]
    T, g = 190, _gen(21)
    bt = ref.table([12], 14)
    pages = ref.Pages(14, kv, d, fmt)
    k, v = _rows((T, kv, d), g), _rows((T, kv, d), g)
    k[T - 2, 0, 5], v[T - 3, 1, 9] = math.inf, math.nan
    pages.write(*ref.slots(bt[0], torch.arange(T)), k, v)
    announce(f"kv8 attention, many rows over tokens that are not finite {fmt} {length}")
    got = _long(cuda_device, (h, kv, d), fmt, [T], [40], length, pages=pages, bt=bt)
    assert bool(torch.isnan(got).any()) and bool(torch.isfinite(got).any())


@pytest.mark.parametrize("length", LENGTHS)
def test_blocks_that_the_table_does_not_name(cuda_device, length):
    pages, bt = _filled(2, 128, "fp8", [300], 8)
    bt = bt.clone()
    bt[0, 2], bt[0, 7], bt[0, 18] = -1, 10 ** 6, -5
    for T in (300, 400):  # the second passes the table
        announce(f"kv8 attention, many rows over blocks that are not there {T} {length}")
        _long(cuda_device, HEADS["target"], "fp8", [T], [40], length, pages=pages, bt=bt)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_scores_far_apart(cuda_device, fmt):
    h, kv, d = HEADS["target"]
    T, g = 900, _gen(17)
    k, v = _rows((T, kv, d), g), _rows((T, kv, d), g)
    k = (k.float() * torch.linspace(0.1, 20.0, T)[:, None, None]).to(torch.bfloat16)
    bt = ref.table([57], 60)
    pages = ref.Pages(60, kv, d, fmt)
    pages.write(*ref.slots(bt[0], torch.arange(T)), k, v)
    announce(f"kv8 attention, many rows, scores far apart {fmt}")
    _long(cuda_device, (h, kv, d), fmt, [T], [50], 131072, pages=pages, bt=bt)


@pytest.mark.parametrize("new,lens,short", [([300], [300], 300), ([48] * 4, [8192, 7000, 5000, 3000], 8192), ([200], [2048], 2048)])
def test_both_kernels_agree(cuda_device, new, lens, short):
    """The same rows by either kernel, each within its bound (a call's sizes choose)."""
    for length in (short, 131072):
        announce(f"kv8 attention by sizes {new} {length}")
        _long(cuda_device, HEADS["target"], "fp8", lens, new, length)
