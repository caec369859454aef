"""More packed rows than one launch has threads for, along x."""
from __future__ import annotations

import pytest
import torch

import kv8_reference as ref
from conftest import announce
from specdec_amd.kernels import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,interleaved", [(128, False), (64, True)])
def test_rope(cuda_device, d, interleaved):
    """In place (17 GB): the rows around every 2^25th, and around 2^32 threads, are what a call of those alone gives."""
    dev = cuda_device
    n = (1 << 33) // d + 5
    inv, _ = ops.rope_frequencies(d, device=dev)
    positions = torch.arange(n, dtype=torch.int32, device=dev)
    rows = torch.empty((n, 1, d), dtype=torch.bfloat16, device=dev)
    at = torch.tensor(sorted({x + i for x in [2, *range(1 << 25, n, 1 << 25), n - 3] for i in (-2, -1, 0, 1, 2)}), device=dev)
    rows[at] = torch.randn((len(at), 1, d), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
    want, _ = ops.rope(rows[at], None, positions[at], inv, interleaved=interleaved)
    announce(f"rope of {n} rows of {d}")
    got, _ = ops.rope(rows, None, positions, inv, interleaved=interleaved, q_out=rows)
    torch.cuda.synchronize()
    assert got.data_ptr() == rows.data_ptr() and torch.equal(rows[at], want)


@pytest.mark.parametrize("tile", [32, 128])
def test_shared_attention(cuda_device, tile):
    """Two sequences whose rows lie behind 2^23 rows of none, which stay as they were."""
    dev = cuda_device
    n = (1 << 23) + 100
    g = torch.Generator().manual_seed(2)
    table = torch.tensor([[3, 1, 0], [3, 1, 4]], dtype=torch.int32)
    lens, new = [40, 45], [5, 4]
    pages = ref.Pages(5, 1, 64, "fp8")
    for b, t in enumerate(lens):
        first = 0 if b == 0 else 32
        k, v = (torch.randn((t - first, 1, 64), generator=g).to(torch.bfloat16) for _ in range(2))
        pages.write(*ref.slots(table[b], torch.arange(first, t)), k, v)
    q = torch.zeros((n, 1, 64), dtype=torch.bfloat16, device=dev)
    q[-9:] = torch.randn((9, 1, 64), generator=g).to(torch.bfloat16).to(dev)
    out = torch.full_like(q, 7.0)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    args = [*pages.to(dev), table.to(dev), ints([n - 9, n - 4, n]), ints(lens), 5, 45, ints([0, 2]), ints([32, 32]), 32]
    announce(f"shared attention of {n} rows, tiles of {tile}")
    ops.kv8_shared_attention(q, *args, tile_rows=tile, out=out)
    torch.cuda.synchronize()
    assert bool((out[:-9] == 7.0).all())
    ref.within(out[-9:], *ref.attention(q[-9:].cpu(), pages, table, new, lens))
    args[4] = ints([0, 5, 9])
    assert torch.equal(out[-9:], ops.kv8_shared_attention(q[-9:], *args, tile_rows=tile))


def test_copy_blocks(cuda_device):
    """2^26 pairs and a few: all but the first, the last and those around the launches' bounds name no block."""
    dev = cuda_device
    n = (1 << 26) + 5
    g = torch.Generator().manual_seed(3)
    pages = [torch.randint(0, 100, (40, 2, *s), generator=g, dtype=torch.int8).to(dev) for s in ((4, 4, 4, 16), (64, 16))]
    pages.append(torch.rand((40, 2, 2, 16), generator=g).to(dev))
    before = [t.clone() for t in pages]
    src, dst = (torch.full((n,), -1, dtype=torch.int32, device=dev) for _ in range(2))
    at = torch.tensor([0, 5, (1 << 25) - 1, 1 << 25, (1 << 26) - 1, 1 << 26, n - 1], device=dev)
    src[at] = torch.arange(7, dtype=torch.int32, device=dev)
    dst[at] = torch.arange(20, 27, dtype=torch.int32, device=dev)
    announce(f"copy_blocks of {n} pairs")
    ops.copy_blocks(*pages, src, dst)
    torch.cuda.synchronize()
    for t, b in zip(pages, before):
        b[20:27] = b[:7]
        assert torch.equal(t, b)


@pytest.mark.parametrize("d", [128, 64])
def test_keep(cuda_device, d):
    """2^25 sequences and a few, of a block each, which keep something in eight of them."""
    dev = cuda_device
    n = (1 << 25) + 5
    g = torch.Generator().manual_seed(4)
    pages = [torch.randint(0, 100, (2, 10, 1, *s), generator=g, dtype=torch.int8).to(dev) for s in ((4, d // 16, 4, 16), (d, 16))]
    pages.append(torch.rand((2, 10, 1, 2, 16), generator=g).to(dev))
    k, v, s = (t.clone() for t in pages)
    at = torch.tensor([0, 9, (1 << 23) - 1, 1 << 23, 1 << 24, (1 << 25) - 1, 1 << 25, n - 1], device=dev)
    table = torch.full((n, 1), -1, dtype=torch.int32, device=dev)
    table[at, 0] = torch.arange(1, 9, dtype=torch.int32, device=dev)
    starts = torch.zeros(n, dtype=torch.int32, device=dev)
    starts[at] = torch.arange(8, dtype=torch.int32, device=dev)
    counts = torch.zeros(n, dtype=torch.int32, device=dev)
    counts[at] = 1
    cu = torch.cat([counts.new_zeros(1), counts.cumsum(0, dtype=torch.int32)])
    kept = torch.tensor([3, 1, 4, 2, 5, 6, 7, 8], dtype=torch.int32, device=dev)
    announce(f"kv8_keep of {n} sequences")
    ops.kv8_keep(*pages, table, cu, kept, starts)
    torch.cuda.synchronize()
    for i, x in enumerate(kept.tolist()):
        a, b = i + x, i
        k[:, i + 1, :, b // 4, :, b % 4] = k[:, i + 1, :, a // 4, :, a % 4]
        v[:, i + 1, :, :, b] = v[:, i + 1, :, :, a]
        s[:, i + 1, :, :, b] = s[:, i + 1, :, :, a]
    assert all(torch.equal(x, y) for x, y in zip(pages, (k, v, s)))
