"""The kv8 operators where sizes are extreme: pools past 4 GiB, contexts of several scale windows, batches
of more sequences than threads, V of very different sizes, one row count announced and another given,
calls side by side on two streams, and a workspace that comes dirty."""
from __future__ import annotations

import math

import pytest
import torch

import kv8_reference as ref
from conftest import announce
from specdec_amd.kernels import ops
from test_gpu_kv8 import HEADS, _attend, _cu, _filled, _gen, _ints, _rows

pytestmark = pytest.mark.gpu


def test_pool_past_4_gib(cuda_device):
    """The same tokens in the last blocks of a pool whose K and V pages take more than 4 GiB each, and in
    a small pool: the same bytes and the same bits."""
    dev = cuda_device
    h, kv, d = HEADS["target"]
    nb = (4 << 30) // (kv * d * 16) + 40
    types = ref.TYPES["fp8"]
    big = (torch.empty((nb, kv, 4, d // 16, 4, 16), dtype=torch.uint8, device=dev).view(types),
           torch.empty((nb, kv, d, 16), dtype=torch.uint8, device=dev).view(types), torch.empty((nb, kv, 2, 16), device=dev))
    small = ref.Pages(30, kv, d, "fp8").to(dev)
    bt = ref.table([13, 5], 30, 3).to(dev)
    high = torch.where(bt >= 0, bt + (nb - 30), bt)
    lens = [200, 71]
    rows = _rows((271, h + 2 * kv, d), _gen(4)).to(dev)
    announce(f"kv8 pool of {nb} blocks")
    for pool, t in ((small, bt), (big, high)):
        ops.kv8_append(rows[:, h:h + kv], rows[:, h + kv:], *pool, t, _cu(lens, dev), _ints(lens, dev))
    torch.cuda.synchronize()
    for a, b in zip(small, big):
        # the tokens of a sequence's last block, past its end, may hold anything
        full = torch.cat([bt[0, :12], bt[1, :4]]).long()
        assert torch.equal(a.view(torch.uint8)[full], b.view(torch.uint8)[full + (nb - 30)])
    for new in ([1, 1], [5, 2], [40, 71]):
        announce(f"kv8 attention over a pool of {nb} blocks, {new}")
        q = rows[:sum(new), :h]
        one = ops.kv8_attention(q, *small, bt, _cu(new, dev), _ints(lens, dev), max(new), 200)
        two = ops.kv8_attention(q, *big, high, _cu(new, dev), _ints(lens, dev), max(new), 200)
        assert torch.equal(one.view(torch.int16), two.view(torch.int16))
    one = ops.kv8_gather(*small, bt, _cu(lens, dev), _ints([0, 0], dev), 271)
    two = ops.kv8_gather(*big, high, _cu(lens, dev), _ints([0, 0], dev), 271)
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])


def _uneven(kv, d, fmt, T, grow, seed):
    """T tokens whose V grows (or shrinks) by 2^24 over the context, with rows of zeros among them."""
    g = _gen(seed)
    k, v = _rows((T, kv, d), g), _rows((T, kv, d), g)
    e = torch.linspace(-12, 12, T) * (1 if grow else -1)
    v = (v.float() * torch.exp2(e.round())[:, None, None]).to(torch.bfloat16)
    v[::17] = 0.0
    k[5::31] = 0.0
    nb = -(-T // 16)
    bt = ref.table([nb], nb + 3, seed)
    pages = ref.Pages(nb + 3, kv, d, fmt)
    pages.write(*ref.slots(bt[0], torch.arange(T)), k, v)
    return pages, bt


@pytest.mark.parametrize("grow", [True, False])
@pytest.mark.parametrize("fmt,heads", [("fp8", (2, 2, 128)), ("int8", (2, 2, 64))])
@pytest.mark.parametrize("new", [1, 20, 33])
def test_many_windows(cuda_device, fmt, heads, grow, new):
    """Sequences that share one context of 9000 tokens; where they have many rows, so many sequences that
    a workgroup's range of a tile has more than 64 stages (200 tiles of 141 on 256 workgroups): windows of
    scales whose largest differ."""
    n, T = 100 if new * heads[0] // heads[1] > 32 else 40, 9000
    pages, bt = _uneven(heads[1], heads[2], fmt, T, grow, 6)
    lens = [T - 211 * (i % 5) for i in range(n)]
    announce(f"kv8 attention over several windows {fmt} {heads} {grow} {new}")
    got, want, bound = _attend(cuda_device, heads, fmt, lens, [new] * n, pages=pages, bt=bt.expand(n, -1).contiguous())
    ref.within(got, want, bound)


@pytest.mark.parametrize("heads,largest", [("draft", 1), ("draft", 4), ("target", 40)])
def test_more_sequences_than_threads(cuda_device, heads, largest):
    """1100 sequences (runs of several for each thread of the plan), some with no rows, some with no tokens."""
    h, kv, d = HEADS[heads]
    n = 1100
    pages, bt = _filled(kv, d, "int8", [300], 2)
    g = _gen(9)
    new = torch.randint(0, largest + 1, (n,), generator=g).tolist()
    lens = [t if i % 13 else 0 for i, t in enumerate(torch.randint(1, 300, (n,), generator=g).tolist())]
    new[500:540] = [0] * 40
    announce(f"kv8 attention of {n} sequences {heads} {largest}")
    got, want, bound = _attend(cuda_device, HEADS[heads], "int8", lens, new, pages=pages, bt=bt.expand(n, -1).contiguous())
    ref.within(got, want, bound)


@pytest.mark.parametrize("said,new,lens", [(1, [40, 3], [300, 90]), (5, [70], [500]), (2, [1, 300, 1], [50, 310, 4000])])
def test_more_rows_than_announced(cuda_device, said, new, lens):
    """max_q_len chooses the tile; sequences with more rows take more tiles of it."""
    dev = cuda_device
    h, kv, d = HEADS["target"]
    pages, bt = _filled(kv, d, "fp8", lens, 12)
    q = torch.randn((sum(new), h, d), generator=_gen(3)).to(torch.bfloat16)
    announce(f"kv8 attention, max_q_len {said} and rows {new}")
    got = ops.kv8_attention(q.to(dev), *pages.to(dev), bt.to(dev), _cu(new, dev), _ints(lens, dev), said, max(lens))
    torch.cuda.synchronize()
    want, bound = ref.attention(q, pages, bt, new, lens)
    ref.within(got, want, bound)


def test_two_streams_at_once(cuda_device):
    """Eager calls that overlap on two streams have a workspace each; the same calls one after another
    give the same bits."""
    dev = cuda_device
    h, kv, d = HEADS["target"]
    cases = []
    for i, (new, lens) in enumerate((([5] * 8, [4000 - 300 * j for j in range(8)]), ([300, 9], [5000, 700]))):
        pages, bt = _filled(kv, d, "int8", lens, 30 + i)
        q = torch.randn((sum(new), h, d), generator=_gen(i)).to(torch.bfloat16).to(dev)
        cases.append((q, *pages.to(dev), bt.to(dev), _cu(new, dev), _ints(lens, dev), max(new), max(lens)))
    want = [ops.kv8_attention(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    announce("kv8 attention on two streams")
    outs = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i].append(ops.kv8_attention(*cases[i]))
    torch.cuda.synchronize()
    for got, w in zip(outs, want):
        assert all(torch.equal(x.view(torch.int16), w.view(torch.int16)) for x in got)


@pytest.mark.parametrize("new", [[1, 1], [5, 4], [40, 1]])
def test_a_workspace_that_others_wrote(cuda_device, new):
    dev = cuda_device
    h, kv, d = HEADS["target"]
    lens = [3000, 2000]
    pages, bt = _filled(kv, d, "fp8", lens, 40)
    q = torch.randn((sum(new), h, d), generator=_gen(1)).to(torch.bfloat16).to(dev)
    args = (q, *pages.to(dev), bt.to(dev), _cu(new, dev), _ints(lens, dev), max(new), max(lens))
    want = ops.kv8_attention(*args)
    nbytes = ops.kv8_attention_workspace_bytes(2, sum(new), h, kv, d, max(new), max(lens))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    announce(f"kv8 attention with a workspace of the caller's {new}")
    for byte in (0xFF, 0x01, 0x7F):
        ws.fill_(byte)
        assert torch.equal(ops.kv8_attention(*args, workspace_tensor=ws).view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("new,lens,length", [([1, 1, 1], [700, 90, 300], 700), ([5, 4, 5], [700, 90, 300], 700), ([40, 7, 50], [700, 90, 300], 700),
                                             ([40, 7, 50], [700, 90, 300], 131072)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_query_rows_that_are_not_finite(cuda_device, new, lens, length, bad):
    """A query row with an infinity or a NaN is NaN in its own output (its head's) and reaches no other."""
    dev = cuda_device
    h, kv, d = HEADS["target"]
    pages, bt = _filled(kv, d, "fp8", lens, 14)
    q = torch.randn((sum(new), h, d), generator=_gen(5)).to(torch.bfloat16)
    want, bound = ref.attention(q, pages, bt, new, lens)
    row = new[0]  # the second sequence's first
    q[row, 3, 17] = bad
    want[row, 3] = math.nan
    announce(f"kv8 attention, a query of {bad} {new} {length}")
    got = ops.kv8_attention(q.to(dev), *pages.to(dev), bt.to(dev), _cu(new, dev), _ints(lens, dev), max(new), length)
    torch.cuda.synchronize()
    ref.within(got, want, bound)


@pytest.mark.parametrize("new,lens", [([1, 1], [800, 70]), ([4, 5], [800, 70]), ([60, 3], [800, 70])])
def test_a_scale_of_zero_and_a_negative_one(cuda_device, new, lens):
    for scale in (0.0, -0.2):
        announce(f"kv8 attention, scale {scale} {new}")
        got, want, bound = _attend(cuda_device, HEADS["target"], "int8", lens, new, scale=scale)
        ref.within(got, want, bound)


def test_recorded_calls_of_one_graph(cuda_device):
    """Calls of one recording share a workspace where their stream orders them: small and large ones after
    each other and on a forked stream; two graphs from the same stream replayed side by side."""
    dev = cuda_device
    h, kv, d = HEADS["target"]
    cases = []
    for i, (new, lens, length) in enumerate((([1, 1], [3000, 2500], 3000), ([40, 3], [900, 2000], 131072), ([5, 5], [4000, 70], 4000),
                                             ([1], [6000], 6000))):
        pages, bt = _filled(kv, d, "fp8", lens, 60 + i)
        q = torch.randn((sum(new), h, d), generator=_gen(i)).to(torch.bfloat16).to(dev)
        cases.append((q, *pages.to(dev), bt.to(dev), _cu(new, dev), _ints(lens, dev), max(new), length))
    want = [ops.kv8_attention(*c) for c in cases]
    torch.cuda.synchronize()
    main, fork = torch.cuda.Stream(), torch.cuda.Stream()
    graphs, outs = [], []
    for _ in range(2):
        graph, got = torch.cuda.CUDAGraph(), []
        with torch.cuda.graph(graph, stream=main):
            for c in cases:
                got.append(ops.kv8_attention(*c))
            fork.wait_stream(main)
            with torch.cuda.stream(fork):
                aside = [ops.kv8_attention(*c) for c in cases]
            for c in cases[::-1]:
                got.append(ops.kv8_attention(*c))
            main.wait_stream(fork)
        graphs.append(graph)
        outs.append(got[:4] + got[4:][::-1] + aside)
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(4):
        announce(f"kv8 attention, two graphs of several calls, replay {turn}")
        for got in outs:
            for o in got:
                o.zero_()
        torch.cuda.synchronize()
        for st, graph in zip(sides, graphs):
            with torch.cuda.stream(st):
                graph.replay()
        again = ops.kv8_attention(*cases[turn])
        torch.cuda.synchronize()
        assert torch.equal(again.view(torch.int16), want[turn].view(torch.int16))
        for got in outs:
            for k, o in enumerate(got):
                assert torch.equal(o.view(torch.int16), want[k % 4].view(torch.int16)), k
