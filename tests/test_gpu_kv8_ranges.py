"""kv8 attention at the ends of its types' ranges: infinite queries, V near the largest BF16."""
from __future__ import annotations

import math

import pytest
import torch

import kv8_reference as ref
from conftest import announce
from specdec_amd.kernels import ops
from test_gpu_kv8 import HEADS, _cu, _filled, _gen, _ints, _rows

pytestmark = pytest.mark.gpu

# (new rows, lengths, announced length): a tile of 16 rows in one workgroup and in several, of 32, of 256 in one
# and in several (an announced length far above the sequences' sends many rows to the kernel for many)
SHAPES = [([1], [1], 1), ([1, 1], [3000, 40], 3000), ([5], [900], 900), ([5, 4], [4000, 4], 4000), ([40], [40], 131072),
          ([40, 9], [6000, 300], 131072), ([300], [300], 300)]


def _one_sign(kv, d, fmt, lens, channel, seed):
    """(pages, table) of random tokens whose K is positive throughout in one channel of the even KV heads and
    negative in the odd ones'."""
    g = _gen(seed)
    counts = [-(-t // 16) for t in lens]
    nb = sum(counts) + 2
    bt = ref.table(counts, nb, seed)
    pages = ref.Pages(nb, kv, d, fmt)
    sign = torch.tensor([1.0 if i % 2 == 0 else -1.0 for i in range(kv)])
    for b, t in enumerate(lens):
        k, v = _rows((t, kv, d), g), _rows((t, kv, d), g)
        k[..., channel] = ((k[..., channel].float().abs() + 0.5) * sign).to(torch.bfloat16)
        pages.write(*ref.slots(bt[b], torch.arange(t)), k, v)
    return pages, bt


@pytest.mark.parametrize("new,lens,length", SHAPES)
@pytest.mark.parametrize("fmt,heads", [("fp8", "target"), ("int8", "draft")])
@pytest.mark.parametrize("bad", [math.inf, -math.inf])
def test_rows_whose_scores_are_all_infinite(cuda_device, fmt, heads, new, lens, length, bad):
    """A query of +inf or -inf in a channel of one sign: every score it makes is +inf, or every one -inf, and
    the softmax is NaN either way; no other row has any of it."""
    dev, (h, kv, d) = cuda_device, HEADS[heads]
    pages, bt = _one_sign(kv, d, fmt, lens, 17, 8)
    q = torch.randn((sum(new), h, d), generator=_gen(5)).to(torch.bfloat16)
    for head in (0, h - 1):  # one of an even KV head, one of an odd
        q[0, head, 17] = q[-1, head, 17] = bad
    want, bound = ref.attention(q, pages, bt, new, lens)
    assert bool(torch.isnan(want[0, 0]).all()) and bool(torch.isnan(want[-1, h - 1]).all()) and not bool(torch.isnan(want[0, 1]).any())
    announce(f"kv8 attention, infinite scores {fmt} {new} {length} {bad}")
    got = ops.kv8_attention(q.to(dev), *pages.to(dev), bt.to(dev), _cu(new, dev), _ints(lens, dev), max(new), length)
    torch.cuda.synchronize()
    ref.within(got, want, bound)


@pytest.mark.parametrize("length", [64, 131072])
@pytest.mark.parametrize("new,lens", [([3, 2], [1, 0]), ([40, 7], [30, 7])])
def test_infinite_queries_that_see_nothing(cuda_device, new, lens, length):
    """Rows before position 0, rows over blocks that the table does not name and rows whose mask is empty are
    0 whatever their query holds."""
    dev, (h, kv, d) = cuda_device, HEADS["target"]
    pages, bt = _filled(kv, d, "fp8", lens, 3)
    q = torch.full((sum(new), h, d), -math.inf, dtype=torch.bfloat16, device=dev)
    announce(f"kv8 attention, infinite queries that see nothing {new} {length}")
    args = (q, *pages.to(dev))
    got = ops.kv8_attention(*args, bt.to(dev), _cu(new, dev), _ints(lens, dev), max(new), length)
    before = new[0] - lens[0]
    assert bool((got[:before] == 0).all()) and bool(torch.isnan(got[before:new[0]]).all())
    got = ops.kv8_attention(*args, torch.full_like(bt, -1).to(dev), _cu(new, dev), _ints(lens, dev), max(new), length)
    assert bool((got == 0).all())
    masks = torch.zeros(sum(new), dtype=torch.int64, device=dev)
    masks[new[0] - 1] = 1 << (new[0] - 1)  # itself alone
    got = ops.kv8_attention(*args, bt.to(dev), _cu(new, dev), _ints(lens, dev), max(new), length, tree_mask=masks)
    assert bool(torch.isnan(got[new[0] - 1]).all()) and bool((got[:new[0] - 1] == 0).all()) and bool((got[new[0]:] == 0).all())


def _large(kv, d, fmt, lens, top, seed):
    """(pages, table) of V up to `top`, some rows of it alike and some zero."""
    g = _gen(seed)
    counts = [-(-t // 16) for t in lens]
    nb = sum(counts) + 2
    bt = ref.table(counts, nb, seed)
    pages = ref.Pages(nb, kv, d, fmt)
    for b, t in enumerate(lens):
        v = torch.randn((t, kv, d), generator=g).clamp(-3, 3) / 3 * top
        v[::5] = top
        v[3::41] = 0.0
        pages.write(*ref.slots(bt[b], torch.arange(t)), _rows((t, kv, d), g), v.to(torch.bfloat16))
    return pages, bt


def _finite(dev, heads, fmt, new, lens, length, top):
    h, kv, d = heads
    pages, bt = _large(kv, d, fmt, lens, top, 4)
    q = torch.randn((sum(new), h, d), generator=_gen(6)).to(torch.bfloat16)
    announce(f"kv8 attention, V up to {top} {fmt} {new} {length}")
    got = ops.kv8_attention(q.to(dev), *pages.to(dev), bt.to(dev), _cu(new, dev), _ints(lens, dev), max(new), length)
    torch.cuda.synchronize()
    assert bool(torch.isfinite(got).all())
    ref.within(got, *ref.attention(q, pages, bt, new, lens))


@pytest.mark.parametrize("top", [1e33, 2.0 ** 121, 3.3e38])
@pytest.mark.parametrize("fmt,heads", [("fp8", "target"), ("int8", "draft"), ("int8", "target")])
@pytest.mark.parametrize("new,lens,length", [([40], [40], 131072), ([40, 9], [6000, 300], 131072), ([700, 1], [3000, 2500], 3000)])
def test_many_rows_over_large_v(cuda_device, fmt, heads, new, lens, length, top):
    """Finite V gives finite outputs, in tiles that one workgroup takes and in tiles whose parts are added up."""
    _finite(cuda_device, HEADS[heads], fmt, new, lens, length, top)


@pytest.mark.parametrize("top", [1e33, 2.0 ** 121, 3.3e38])
@pytest.mark.parametrize("fmt,heads", [("fp8", "target"), ("int8", "draft"), ("int8", "target")])
@pytest.mark.parametrize("new,lens,length", [([1], [1], 1), ([1, 1], [3000, 40], 3000), ([1], [20000], 20000), ([5], [90], 90),
                                             ([5, 4], [4000, 4], 4000), ([1] * 40, [700 + 31 * i for i in range(40)], 2000), ([300], [300], 300)])
def test_few_rows_over_large_v(cuda_device, fmt, heads, new, lens, length, top):
    _finite(cuda_device, HEADS[heads], fmt, new, lens, length, top)


@pytest.mark.parametrize("new,lens", [([1], [5000]), ([5], [900]), ([60], [900])])
def test_large_v_that_comes_late(cuda_device, new, lens):
    """V of 1 for most of the context, then a few tokens of 1e37, of which some rows see none: theirs are as
    near to the result as ever."""
    dev, (h, kv, d) = cuda_device, HEADS["target"]
    t = lens[0]
    g = _gen(9)
    bt = ref.table([-(-t // 16)], -(-t // 16) + 2, 5)
    pages = ref.Pages(-(-t // 16) + 2, kv, d, "fp8")
    k, v = _rows((t, kv, d), g), _rows((t, kv, d), g)
    v[t - 2:] = (v[t - 2:].float() * 1e37).to(torch.bfloat16)
    pages.write(*ref.slots(bt[0], torch.arange(t)), k, v)
    q = torch.randn((sum(new), h, d), generator=g).to(torch.bfloat16)
    want, bound = ref.attention(q, pages, bt, new, lens)
    early = new[0] - 2  # the rows that see none of it
    if early > 0 and new[0] * h // kv <= 32:
        # in the kernel for few rows the large scale takes no part in these: the bound of the context without it
        small = ref.Pages(-(-t // 16) + 2, kv, d, "fp8")
        small.write(*ref.slots(bt[0], torch.arange(t - 2)), k[:t - 2], v[:t - 2])
        near, tight = ref.attention(q[:early], small, bt, [early], [t - 2])
        want[:early], bound[:early] = near, tight
    announce(f"kv8 attention, large V among small {new}")
    got = ops.kv8_attention(q.to(dev), *pages.to(dev), bt.to(dev), _cu(new, dev), _ints(lens, dev), max(new), max(lens))
    torch.cuda.synchronize()
    ref.within(got, want, bound)


@pytest.mark.parametrize("zero", [True, False])
@pytest.mark.parametrize("below", [10, 17, 18, 19, 22, 25, 27, 29, 30, 31, 37, 60])
@pytest.mark.parametrize("fmt,heads", [("fp8", "target"), ("int8", "draft"), ("fp8", "draft"), ("int8", "target")])
@pytest.mark.parametrize("length", [190, 131072])
def test_small_v_beside_a_large_scale(cuda_device, length, fmt, heads, below, zero):
    """Rows that see only V some 2^-below of a token's that the tile holds and they do not see -- a row of
    zeros, whose scale is 1, or one of 448 or 127 --, and rows that see both.  What the large scale takes from the
    former is half of FP16's smallest step under it, 2^-30."""
    dev, (h, kv, d) = cuda_device, HEADS[heads]
    n, t = 60, 190
    g = _gen(below)
    k = _rows((t, kv, d), g)
    v = (torch.rand((t, kv, d), generator=g) + 0.5) * ref.LARGEST[fmt] * 2.0 ** -below
    v[t - 7] = 0.0 if zero else torch.where(torch.rand((kv, d), generator=g) < 0.5, -1.0, 1.0) * ref.LARGEST[fmt]
    v = v.to(torch.bfloat16)
    bt = ref.table([12], 14, 2)
    pages, small = ref.Pages(14, kv, d, fmt), ref.Pages(14, kv, d, fmt)
    pages.write(*ref.slots(bt[0], torch.arange(t)), k, v)
    early = n - 7
    small.write(*ref.slots(bt[0], torch.arange(t - 7)), k[:t - 7], v[:t - 7])
    q = torch.randn((n, h, d), generator=g).to(torch.bfloat16)
    want, bound = ref.attention(q, pages, bt, [n], [t])
    want[:early], bound[:early] = ref.attention(q[:early], small, bt, [early], [t - 7])
    bound[:early] += 2.0 ** -30
    announce(f"kv8 attention, small V beside a large scale {fmt} {heads} {below} {zero} {length}")
    got = ops.kv8_attention(q.to(dev), *pages.to(dev), bt.to(dev), _cu([n], dev), _ints([t], dev), n, length)
    torch.cuda.synchronize()
    ref.within(got, want, bound)


@pytest.mark.parametrize("fmt,heads", [("fp8", "target"), ("int8", "draft")])
@pytest.mark.parametrize("down", [True, False])
def test_v_of_every_size(cuda_device, fmt, heads, down):
    """V whose scales run over 2^-100 .. 2^100 within a context of several windows, in tiles that one workgroup
    takes whole and in cut ones.  The rows of the first sequences see all, those of the last only the first
    hundred keys (larger ones follow, or smaller)."""
    dev, (h, kv, d) = cuda_device, HEADS[heads]
    t, n, first = 9000, 40, 100
    g = _gen(3)
    k, v = _rows((t, kv, d), g), _rows((t, kv, d), g)
    e = torch.linspace(100, -100, t) if down else torch.linspace(-100, 100, t)
    v = (v.float() * torch.exp2(e.round())[:, None, None]).to(torch.bfloat16)
    nb = -(-t // 16)
    bt = ref.table([nb], nb + 2, 2)
    pages = ref.Pages(nb + 2, kv, d, fmt)
    pages.write(*ref.slots(bt[0], torch.arange(t)), k, v)
    q = torch.randn((2 * n, h, d), generator=g).to(torch.bfloat16)
    lens = [t, first]
    announce(f"kv8 attention, V of every size {fmt} {heads} {down}")
    table = bt.expand(2, -1).contiguous()
    got = ops.kv8_attention(q.to(dev), *pages.to(dev), table.to(dev), _cu([n, n], dev), _ints(lens, dev), n, 131072)
    torch.cuda.synchronize()
    ref.within(got, *ref.attention(q, pages, table, [n, n], lens))
    many = 100  # so many sequences that a workgroup's range holds several windows
    rows = q[:n].repeat(many, 1, 1)
    table = bt.expand(many, -1).contiguous()
    again = ops.kv8_attention(rows.to(dev), *pages.to(dev), table.to(dev), _cu([n] * many, dev), None, n, t)
    torch.cuda.synchronize()
    want, bound = ref.attention(q[:n], pages, bt, [n], [t])
    for i in (0, 1, many // 2, many - 1):
        ref.within(again[i * n:(i + 1) * n], want, bound)
