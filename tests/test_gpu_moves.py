"""Page moves on the GPU against indexing in torch, byte for byte."""
from __future__ import annotations

import random

import pytest
import torch

import kv8_reference as ref
from conftest import announce
from specdec_amd._native import SdvError
from specdec_amd.kernels import ops

pytestmark = pytest.mark.gpu


def _pages(kind, layers, nb, kv, d, seed, dev):
    """Page tensors of random bytes: "fp8", "int8" (the 8-bit cache) or "v_fp8" (BF16 K)."""
    g = torch.Generator().manual_seed(seed)
    lead = (nb,) if layers is None else (layers, nb)
    raw = lambda *s: torch.randint(0, 256, (*lead, *s), generator=g, dtype=torch.uint8)  # noqa: E731
    if kind == "v_fp8":
        t = raw(kv, d // 8, 16, 16).view(torch.bfloat16), raw(kv, d, 16), raw(kv, 64).view(torch.float32)
    else:
        t = raw(kv, 4, d // 16, 4, 16).view(ref.TYPES[kind]), raw(kv, d, 16).view(ref.TYPES[kind]), raw(kv, 2, 64).view(torch.float32)
    return tuple(x.to(dev) for x in t)


def _bytes(t):
    return t.contiguous().view(torch.uint8).cpu() if t.dtype is not torch.uint8 else t.cpu()


def _ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("kind", ["fp8", "int8", "v_fp8"])
@pytest.mark.parametrize("layers,nb,kv,d,n", [(None, 5, 2, 128, 2), (1, 4, 1, 64, 1), (3, 40, 2, 64, 17), (28, 30, 2, 128, 13), (2, 20, 8, 128, 9), (None, 200, 2, 64, 99)])
def test_copy_blocks(cuda_device, kind, layers, nb, kv, d, n):
    announce(f"copy_blocks {kind} {layers} {nb} {kv} {d} {n}")
    dev = cuda_device
    pages = _pages(kind, layers, nb, kv, d, 1, dev)
    before = [_bytes(t) for t in pages]
    order = random.Random(n).sample(range(nb), 2 * n)
    src, dst = order[:n], order[n:]
    src[-1] = src[0]  # one block to two
    dim = 0 if layers is None else 1
    ops.copy_blocks(*pages, _ints(src, dev), _ints(dst, dev))
    for t, b in zip(pages, before):
        want = b.clone()
        want.index_copy_(dim, torch.tensor(dst), b.index_select(dim, torch.tensor(src)))
        assert torch.equal(_bytes(t), want)
    # to a pool of another size
    other = _pages(kind, layers, n + 1, kv, d, 2, dev)
    old = [_bytes(t) for t in other]
    ops.copy_blocks(*pages, _ints(src, dev), _ints(list(range(n)), dev), to=other)
    for t, o, x in zip(other, old, pages):
        want = o.clone()
        want.index_copy_(dim, torch.arange(n), _bytes(x).index_select(dim, torch.tensor(src)))
        assert torch.equal(_bytes(t), want)


def test_pairs_that_name_no_block(cuda_device):
    dev = cuda_device
    pages, other = _pages("int8", 2, 6, 2, 64, 1, dev), _pages("int8", 2, 3, 2, 64, 2, dev)
    old = [_bytes(t) for t in other]
    ops.copy_blocks(*pages, _ints([-1, 6, 5, 4, 1, 2 ** 31 - 1], dev), _ints([0, 1, 2, 3, -7, 0], dev), to=other)
    for t, o, x in zip(other, old, pages):
        o[:, 2] = _bytes(x)[:, 5]
        assert torch.equal(_bytes(t), o)
    ops.copy_blocks(*pages, _ints([], dev), _ints([], dev))


def test_copies_in_a_graph(cuda_device):
    dev = cuda_device
    pages = _pages("fp8", 4, 50, 2, 128, 1, dev)
    src, dst = _ints(list(range(10)), dev), _ints(list(range(10, 20)), dev)
    ops.copy_blocks(*pages, src, dst)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.copy_blocks(*pages, src, dst)
    for k in (20, 30, 40):
        dst.copy_(torch.arange(k, k + 10))
        graph.replay()
        torch.cuda.synchronize()
        for t in pages:
            b = _bytes(t)
            assert torch.equal(b[:, k:k + 10], b[:, :10])


def test_copy_refusals(cuda_device):
    dev = cuda_device
    pages, ids = _pages("int8", 2, 6, 2, 64, 1, dev), _ints([1], dev)
    for other in (_pages("int8", 3, 6, 2, 64, 1, dev), _pages("fp8", 2, 6, 2, 64, 1, dev), _pages("int8", 2, 6, 2, 128, 1, dev),
                  _pages("int8", 2, 6, 1, 64, 1, dev), _pages("int8", None, 6, 2, 64, 1, dev), pages[:2]):
        with pytest.raises(SdvError):
            ops.copy_blocks(*pages, ids, ids, to=other)
    for bad in ((ids.long(), ids), (ids, _ints([1, 2], dev)), (ids.cpu(), ids), (ids.view(1, 1), ids)):
        with pytest.raises(SdvError):
            ops.copy_blocks(*pages, *bad)
    for bad in ((pages[0][:, :5], *pages[1:]), (pages[0], pages[1][..., :8], pages[2]), (pages[0], pages[1], pages[2].double())):
        with pytest.raises(SdvError):
            ops.copy_blocks(*bad, ids, ids)


# ------------------------------------------------------------------------------ kept tokens
def _keep_reference(pages, table, starts, kept, nb):
    """kv8_keep on byte copies of layered pages: each sequence's tokens read, then written."""
    k, v, s = pages
    for b, (start, ids) in enumerate(zip(starts, kept)):
        pairs = []
        for i, x in enumerate(ids):
            ends = []
            for pos in (start + x, start + i):
                blk = int(table[b, pos // 16]) if 0 <= pos < 16 * table.shape[1] else -1
                ends.append((blk, pos % 16) if 0 <= blk < nb else None)
            if None not in ends:
                pairs.append(ends)
        read = [(k[:, x, :, o // 4, :, o % 4].clone(), v[:, x, :, :, o].clone(), s[:, x, :, :, o].clone()) for (x, o), _ in pairs]
        for (_, (x, o)), (a, c, e) in zip(pairs, read):
            k[:, x, :, o // 4, :, o % 4], v[:, x, :, :, o], s[:, x, :, :, o] = a, c, e


@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("layers,kv,d", [(None, 2, 128), (3, 2, 64), (28, 1, 128), (2, 8, 64)])
@pytest.mark.parametrize("starts,kept", [
    ([0], [[0]]), ([5], [[3]]), ([15], [[1, 2, 3]]), ([100, 31, 16, 7], [[0, 2, 5, 6], [], [63], [1, 4, 9, 20, 40]]),
    ([40], [[x for x in range(64) if x % 3]]), ([3], [[9, 0, 4, 4, 2]]), ([77, 3], [list(range(1, 65)), list(range(0, 128, 2))]),
    ([1], [sorted(random.Random(3).sample(range(400), 201))]), ([20], [list(range(20, 20 + 150))])])
def test_keep(cuda_device, kind, layers, kv, d, starts, kept):
    announce(f"kv8 keep {kind} {layers} {kv} {d} {starts} {kept}")
    dev = cuda_device
    counts = [(s + max(ids, default=0)) // 16 + 1 for s, ids in zip(starts, kept)]
    nb = sum(counts) + 3
    table = ref.table(counts, nb, 5)
    pages = _pages(kind, layers, nb, kv, d, 3, dev)
    cu = [0]
    for ids in kept:
        cu.append(cu[-1] + len(ids))
    lead = (lambda t: t) if layers else (lambda t: t.unsqueeze(0))
    want = [lead(t.cpu().view(torch.uint8) if t.element_size() == 1 else t.cpu().view(torch.int32)).clone() for t in pages]
    _keep_reference(want, table, starts, kept, nb)
    ops.kv8_keep(*pages, table.to(dev), _ints(cu, dev), _ints([x for ids in kept for x in ids], dev), _ints(starts, dev))
    for t, w in zip(pages, want):
        assert torch.equal(lead(t.cpu().view(w.dtype)), w)


def test_keep_of_tokens_in_no_block(cuda_device):
    """Sources and destinations outside the table, or in blocks that it does not name, negative positions: skipped."""
    dev = cuda_device
    table = torch.tensor([[4, -1, 2], [0, 9, 1]], dtype=torch.int32)
    starts, kept = [10, -3], [[0, 3, 9, 22, 38, 1000], [2, 5, 8, 21, 40]]
    pages = _pages("int8", 2, 6, 2, 64, 3, dev)
    want = [t.cpu().view(torch.uint8 if t.element_size() == 1 else torch.int32).clone() for t in pages]
    _keep_reference(want, table, starts, kept, 6)
    cu = _ints([0, 6, 11], dev)
    ids = _ints([x for y in kept for x in y], dev)
    announce("kv8 keep outside the table")
    ops.kv8_keep(*pages, table.to(dev), cu, ids, _ints(starts, dev))
    for t, w in zip(pages, want):
        assert torch.equal(t.cpu().view(w.dtype), w)
    ops.kv8_keep(*pages, table.to(dev), _ints([0, 0, 0], dev), ids[:0], _ints(starts, dev))


def test_keep_refusals(cuda_device):
    dev = cuda_device
    pages, table, one = _pages("int8", 2, 6, 2, 64, 3, dev), _ints([[1, 2]], dev), _ints([0], dev)
    good = dict(k_pages=pages[0], v_pages=pages[1], scales=pages[2], block_table=table, cu_kept=_ints([0, 1], dev), kept=one, starts=one)
    v8 = _pages("v_fp8", 2, 6, 2, 64, 3, dev)
    for bad in (dict(cu_kept=one), dict(kept=one.long()), dict(starts=_ints([0, 1], dev)), dict(block_table=table.long()),
                dict(k_pages=v8[0]), dict(scales=v8[2]), dict(kept=one.cpu()), dict(v_pages=pages[1][:1])):
        with pytest.raises(SdvError):
            ops.kv8_keep(**{**good, **bad})
