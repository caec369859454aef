"""Attention of sequences that begin with the same pages, against plain torch in 64 bits over each sequence's whole context
(tests/kv8_reference.py, with its bound)."""
from __future__ import annotations

import math
import random

import pytest
import torch

import kv8_reference as ref
from conftest import announce
from specdec_amd._native import SdvError
from specdec_amd.kernels import ops

pytestmark = pytest.mark.gpu
HEADS = {"target": (12, 2, 128), "draft": (14, 2, 64), "mha": (4, 4, 128), "mqa": (20, 1, 64)}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rows(shape, g, outliers=8.0):
    x = torch.randn(shape, generator=g)
    x[..., 3] *= outliers
    return x.to(torch.bfloat16)


def _ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _sums(x):
    out = [0]
    for n in x:
        out.append(out[-1] + n)
    return out


class Case:
    """groups: [(prefix blocks, [(own tokens, new ones among them), ...]), ...]; a prefix of None: sequences in no group."""

    def __init__(self, heads, fmt, groups, seed=1):
        self.h, self.kv, self.d = HEADS[heads]
        self.fmt, g = fmt, _gen(seed)
        self.new = [n for _, seqs in groups for _, n in seqs]
        self.prefix = [16 * (p or 0) for p, seqs in groups for _ in seqs]
        self.lens = [16 * (p or 0) + t for p, seqs in groups for t, _ in seqs]
        own = [-(-t // 16) for _, seqs in groups for t, _ in seqs]
        counts = [p or 0 for p, _ in groups] + own
        nb = sum(counts) + 3
        owned = ref.table(counts, nb, seed)
        self.table = torch.full((len(own), max(1, max(-(-t // 16) for t in self.lens))), -1, dtype=torch.int32)
        self.pages = ref.Pages(nb, self.kv, self.d, fmt)
        b, cu = 0, [0]
        for i, (p, seqs) in enumerate(groups):
            p = p or 0
            if p:
                self._fill(owned[i], 16 * p, g)
            for t, _ in seqs:
                self.table[b, :p], self.table[b, p:p + own[b]] = owned[i, :p], owned[len(groups) + b, :own[b]]
                if t:
                    self._fill(owned[len(groups) + b], t, g)
                b += 1
            cu.append(b)
        # groups without a prefix are left out where that leaves the others' bounds whole (at the end)
        self.groups = cu
        while len(groups) > 1 and groups[-1][0] is None:
            groups, self.groups = groups[:-1], self.groups[:-1]
        self.q = torch.randn((sum(self.new), self.h, self.d), generator=_gen(seed + 7)).to(torch.bfloat16)

    def _fill(self, row, n, g):
        self.pages.write(*ref.slots(row, torch.arange(n)), _rows((n, self.kv, self.d), g), _rows((n, self.kv, self.d), g, 20.0))

    def args(self, dev, lens=True):
        return (*self.pages.to(dev), self.table.to(dev), _ints(_sums(self.new), dev), _ints(self.lens, dev) if lens else None,
                max(1, *self.new), max(1, *self.lens), _ints(self.groups, dev), _ints(self.prefix, dev), max(self.prefix))

    def run(self, dev, **kw):
        got = ops.kv8_shared_attention(self.q.to(dev), *self.args(dev), **kw)
        torch.cuda.synchronize()
        return got

    def want(self, **kw):
        return ref.attention(self.q, self.pages, self.table, self.new, self.lens, **kw)


CASES = {
    "one": [(1, [(1, 1)])],
    "pair": [(4, [(1, 1), (17, 1)])],
    "eight": [(128, [(t, 1) for t in (1, 16, 17, 300, 64, 65, 5, 128)])],
    "verify": [(33, [(t, 5) for t in (5, 16, 21, 100)])],
    "ragged": [(20, [(9, 1), (40, 7), (3, 0), (30, 16), (2, 2)])],
    "groups": [(3, [(1, 1), (2, 1), (3, 1)]), (70, [(15, 1), (200, 3)]), (1, [(1, 1)])],
    "some in none": [(8, [(5, 1), (6, 2)]), (None, [(50, 1), (7, 7)])],
    "none between": [(8, [(5, 1), (6, 2)]), (None, [(50, 1)]), (5, [(4, 4), (90, 1)])],
    "many": [(5, [(1 + 3 * (i % 7), 1) for i in range(150)]), (2, [(2, 1)] * 150)],
    "rows": [(40, [(50, 40), (90, 64), (33, 33)])],
    "long": [(700, [(300, 3)] * 6)],
    "no new": [(6, [(4, 0), (9, 0), (3, 1)])],
}


TILES = pytest.mark.parametrize("tile", [32, 128])


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("heads", list(HEADS))
@pytest.mark.parametrize("name", list(CASES))
def test_shared(cuda_device, name, heads, fmt):
    case = Case(heads, fmt, CASES[name])
    want = case.want()
    for tile in (0, 32, 128):
        announce(f"shared {name} {heads} {fmt} {tile}")
        ref.within(case.run(cuda_device, tile_rows=tile), *want)


@TILES
@pytest.mark.parametrize("heads", ["target", "draft"])
@pytest.mark.parametrize("name", ["verify", "ragged", "rows", "groups"])
def test_trees(cuda_device, name, heads, tile):
    announce(f"shared trees {name} {heads} {tile}")
    case = Case(heads, "fp8", CASES[name])
    rng, words = random.Random(3), []
    for n in case.new:
        for i in range(n):
            words.append((words[len(words) - 1 - rng.randrange(min(i, 4))] if i else 0) | 1 << i)
    tree = torch.tensor([w - (1 << 64) if w >> 63 else w for w in words], dtype=torch.int64)
    ref.within(case.run(cuda_device, tree_mask=tree.to(cuda_device), tile_rows=tile), *case.want(tree=tree))


@TILES
def test_one_length_a_scale_and_a_given_output(cuda_device, tile):
    case = Case("draft", "int8", [(10, [(37, 3)] * 3)])
    dev = cuda_device
    wide = torch.full((9 + 2, 20, 64), 7.0, dtype=torch.bfloat16, device=dev)
    q = torch.cat((case.q, case.q[:2])).to(dev)  # two rows behind the last sequence
    got = ops.kv8_shared_attention(q, *case.args(dev, lens=False), tile_rows=tile, scale=0.05, out=wide[:, 3:17])
    assert got.data_ptr() == wide[:, 3:17].data_ptr()
    ref.within(got[:9], *case.want(scale=0.05))
    assert bool((wide[9:] == 7.0).all()) and bool((wide[:, :3] == 7.0).all()) and bool((wide[:, 17:] == 7.0).all())
    odd = torch.empty((11, 14 * 64 + 3), dtype=torch.bfloat16, device=dev)[:, 3:].view(11, 14, 64).copy_(q)  # copied
    assert torch.equal(ops.kv8_shared_attention(odd, *case.args(dev), tile_rows=tile, scale=0.05)[:9], got[:9])
    assert ops.kv8_shared_attention(q[:0], *case.args(dev), tile_rows=tile).shape == (0, 14, 64)


@TILES
def test_prefixes_are_whole_blocks(cuda_device, tile):
    """A length inside a block counts down to its start; a bound below the lengths cuts them: the rest is read through each table."""
    case = Case("target", "fp8", CASES["verify"])
    case.table, dev = case.table.clone(), cuda_device
    args = list(case.args(dev))
    want = case.want()
    for prefix, most in (([527, 527, 527, 527], 600), ([528] * 4, 100), ([528] * 4, 527), ([15] * 4, 15), ([0] * 4, 0)):
        args[-2], args[-1] = _ints(prefix, dev), most
        announce(f"shared prefixes {prefix} {most}")
        if most > 16 * case.table.shape[1]:
            most = args[-1] = 16 * case.table.shape[1]
        ref.within(ops.kv8_shared_attention(case.q.to(dev), *args, tile_rows=tile), *want)
    args[-3] = _ints([0], dev)  # no groups, no prefixes
    ref.within(ops.kv8_shared_attention(case.q.to(dev), *args, tile_rows=tile), *want)


@TILES
def test_every_row_sees_the_whole_prefix(cuda_device, tile):
    """A prefix that reaches past a context: as documented, its keys for every row, then what is left of the sequence's own."""
    case, dev = Case("mha", "fp8", [(4, [(2, 2), (20, 9)])]), cuda_device
    args = list(case.args(dev))
    args[5] = _ints([60, 84], dev)  # the first sequence ends within the prefix
    announce("shared prefix past a context")
    got = ops.kv8_shared_attention(case.q.to(dev), *args, tile_rows=tile)
    want, bound = ref.attention(case.q[:2], case.pages, case.table[:1], [2], [64], tree=torch.tensor([3, 3]))
    ref.within(got[:2], want, bound)
    ref.within(got[2:], *(x[2:] for x in case.want()))


@TILES
@pytest.mark.parametrize("heads", ["target", "draft"])
def test_what_is_not_seen_or_not_finite(cuda_device, heads, tile):
    """NaN scales where a sequence ends and in unnamed blocks; NaN and infinities in the prefix reach its group alone; infinite
    queries; sequences of length 0 and tables without blocks."""
    dev = cuda_device
    case = Case(heads, "fp8", [(3, [(5, 2), (9, 1)]), (2, [(7, 3), (30, 1)]), (None, [(0, 0), (40, 1)])])
    case.pages.s[case.table[0, 1], 0, 1, 5] = math.nan   # a token of the first group's prefix
    case.pages.s[case.table[0, 1], -1, 0, 9] = math.inf  # and its K scale: scores of both signs
    case.table[2, 1] = case.table[3, 1] = -1             # a block of the second's that the table does not name
    case.table[5, 0], case.table[5, 2] = 10 ** 6, -5
    case.q[4, 0] = math.inf
    announce(f"shared not finite {heads}")
    got = case.run(dev, tile_rows=tile)
    want, bound = case.want()
    bad = torch.isnan(want)
    assert bool(torch.isnan(got.cpu())[bad].all())
    rest = torch.ones(len(case.q), dtype=torch.bool)
    rest[:3] = False  # the first group's other heads hold what an infinite scale makes of them
    h = case.h // case.kv
    ref.within(got[rest], want[rest], bound[rest])
    if case.kv == 2:
        assert bool(torch.isnan(got[:3, :h]).all())


@TILES
def test_rows_that_see_nothing(cuda_device, tile):
    dev = cuda_device
    case = Case("target", "int8", [(2, [(3, 2), (20, 5)])])
    case.table[:] = -1
    assert bool((case.run(dev, tile_rows=tile) == 0).all())
    case = Case("target", "int8", [(None, [(0, 0), (6, 2)])])
    args = list(case.args(dev))
    args[5] = _ints([0, 1], dev)  # two rows of a sequence of one token
    got = ops.kv8_shared_attention(case.q.to(dev), *args, tile_rows=tile)
    assert bool((got[0] == 0).all()) and bool((got[1] != 0).any())
    # scores of -inf alone are NaN, as in kv8_attention: a query of -inf over keys of one sign
    case = Case("mha", "int8", [(2, [(3, 1), (20, 1)])])
    case.pages.k.view(torch.int8).fill_(3)
    case.q.fill_(-math.inf)
    assert bool(torch.isnan(case.run(dev, tile_rows=tile)).all())


@TILES
def test_large_scales_stay_finite(cuda_device, tile):
    case = Case("target", "fp8", [(12, [(9, 2), (30, 2), (60, 2)])])
    case.pages.s[:, :, 1] *= 2.0 ** 118
    got = case.run(cuda_device, tile_rows=tile)
    want, bound = case.want()
    assert bool(torch.isfinite(got).all())
    ref.within(got, want, bound)


@pytest.mark.parametrize("heads,fmt", [("target", "fp8"), ("draft", "int8")])
def test_scales_that_lie_far_apart(cuda_device, heads, fmt):
    """V of some of a prefix's tokens 2^-30 of the others': tiles of 128 rows go over to narrow ones where they meet both, and
    what those tokens give is as exact as ever for the rows that see hardly anything else."""
    case = Case(heads, fmt, [(24, [(9, 3), (30, 3), (60, 3), (2, 1), (5, 2)])])
    small = case.table[0, 3:7].long()
    case.pages.s[small, :, 1] *= 2.0 ** -30
    case.pages.s[case.table[0, 12].long(), :, 1, 5] = 0.0  # a scale of 0, as no writer leaves it, is no scale
    # keys of the others far below those: their scores are -60 and less
    case.pages.s[:, :, 0] *= 1e-3
    for tile in (32, 128):
        ref.within(case.run(cuda_device, tile_rows=tile), *case.want())


@pytest.mark.parametrize("heads,groups,rows", [
    ("target", [(16, [(9, 1)] * 3)], 0),                      # short
    ("target", [(4096 // 16, [(20, 1)] * 70)], 32),           # single tokens
    ("mha", [(4096 // 16, [(20, 17)] * 2)], 32),              # more rows than one tile of 16 holds
    ("draft", [(8192 // 16, [(40, 5)] * 20)], 128),           # verify blocks
    ("target", [(8192 // 16, [(40, 20)] * 20)], 0)])          # 120 rows a sequence and KV head
def test_the_faster_way_is_chosen(cuda_device, heads, groups, rows):
    from specdec_amd import _native

    announce(f"shared choice {heads} {rows}")
    case = Case(heads, "fp8", groups)
    got = _native.load().sdv_kv8_shared_attention_tile_rows(len(case.new), len(case.groups) - 1, sum(case.new), case.h, case.kv, case.d, max(case.new),
                                                            max(case.lens), max(case.prefix))
    assert got == rows
    args, q = case.args(cuda_device), case.q.to(cuda_device)
    out = ops.kv8_shared_attention(q, *args)
    same = ops.kv8_shared_attention(q, *args, tile_rows=rows) if rows else ops.kv8_attention(q, *args[:8])
    assert torch.equal(out, same)
    at = case.new[0]  # the first sequence's rows, in 64 bits
    want, bound = ref.attention(case.q[:at], case.pages, case.table[:1], case.new[:1], case.lens[:1])
    ref.within(out[:at], want, bound)


@TILES
def test_recorded_calls_follow_their_inputs(cuda_device, tile):
    """Two graphs of the same call and eager calls between them: lengths, rows and pages as they are at each replay."""
    dev = cuda_device
    case = Case("draft", "fp8", [(40, [(60, 2)] * 5)])
    args, q = case.args(dev), case.q.to(dev)
    ops.kv8_shared_attention(q, *args, tile_rows=tile)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = ops.kv8_shared_attention(q, *args, tile_rows=tile)
        graphs.append((graph, got))
    for step in range(6):
        lens = [640 + 60 - (step * 7 + b) % 50 for b in range(5)]
        args[5].copy_(_ints(lens, dev))
        q.copy_(torch.randn(q.shape, generator=_gen(step)).to(torch.bfloat16))
        for graph, got in graphs:
            graph.replay()
            torch.cuda.synchronize()
            eager = ops.kv8_shared_attention(q, *args, tile_rows=tile)
            assert torch.equal(got, eager)
        ref.within(eager, *ref.attention(q.cpu(), case.pages, case.table, case.new, lens))


@TILES
def test_streams_and_repeats(cuda_device, tile):
    """Calls that overlap on two streams, and the same call again, give the same bits."""
    dev = cuda_device
    a, b = Case("target", "fp8", CASES["eight"]), Case("target", "int8", CASES["many"], seed=5)
    xa, xb, qa, qb = a.args(dev), b.args(dev), a.q.to(dev), b.q.to(dev)
    want = ops.kv8_shared_attention(qa, *xa, tile_rows=tile), ops.kv8_shared_attention(qb, *xb, tile_rows=tile)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = []
    for _ in range(10):
        got.append((ops.kv8_shared_attention(qa, *xa, tile_rows=tile), want[0]))
        with torch.cuda.stream(side):
            got.append((ops.kv8_shared_attention(qb, *xb, tile_rows=tile), want[1]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in got)


@TILES
def test_tables_that_decrease_stay_in_bounds(cuda_device, tile):
    """Bad row and group tables, negative and huge lengths: whatever comes out, nothing else is written."""
    dev = cuda_device
    case = Case("target", "fp8", CASES["groups"])
    args, q = list(case.args(dev)), case.q.to(dev)
    B, total = len(case.new), sum(case.new)
    guard = torch.full((total + 4, 12, 128), 7.0, dtype=torch.bfloat16, device=dev)
    tables = [([0, total, 0, total, 0, total, 2], [0, B, 0, B]), ([-5, 99, 3, 2, 1, 10 ** 9, -(2 ** 31)], [5, 1, 2 ** 31 - 1, -7]),
              (list(range(B + 1)), [B, B, B, B])]
    for cu, groups in tables:
        for lens, prefix in ((case.lens, case.prefix), ([2 ** 31 - 1, -1, 0, -(2 ** 31), 5, 10 ** 6], [2 ** 31 - 1, -9, 48, 10 ** 9, 7, 16])):
            args[4], args[8], args[5], args[9] = _ints(cu, dev), _ints(groups, dev), _ints(lens, dev), _ints(prefix, dev)
            announce(f"shared bad tables {cu} {groups} {lens} {prefix}")
            ops.kv8_shared_attention(q, *args, tile_rows=tile, out=guard[2:-2])
            torch.cuda.synchronize()
            assert bool((guard[:2] == 7.0).all()) and bool((guard[-2:] == 7.0).all())


def test_refusals(cuda_device):
    dev = cuda_device
    case = Case("target", "fp8", CASES["groups"])
    names = ("k_pages", "v_pages", "scales", "block_table", "cu_rows", "seq_lens", "max_q_len", "max_seq_len", "cu_groups", "prefix_lens",
             "max_prefix_len")
    good = dict(zip(names, case.args(dev)), q=case.q.to(dev))
    tree = torch.ones(len(case.q), dtype=torch.int64, device=dev)
    for bad in (dict(cu_groups=good["prefix_lens"].repeat(3)), dict(cu_groups=good["cu_groups"].long()), dict(cu_groups=good["cu_groups"][:0]),
                dict(prefix_lens=good["prefix_lens"][:2]), dict(prefix_lens=good["prefix_lens"].cpu()), dict(max_prefix_len=-1),
                dict(max_prefix_len=10 ** 6), dict(max_seq_len=0), dict(max_q_len=0), dict(q=good["q"][:, :7]), dict(q=good["q"].float()),
                dict(cu_rows=good["cu_rows"][:3]), dict(out=torch.empty_like(good["q"])[:2]), dict(tree_mask=tree[:3]),
                dict(tree_mask=tree, max_q_len=65), dict(max_seq_len=2 ** 31 - 1), dict(tile_rows=128, max_prefix_len=10 ** 6),
                dict(tile_rows=32, max_seq_len=2 ** 31 - 1)):
        with pytest.raises(SdvError):
            ops.kv8_shared_attention(**{**good, **bad})
    with pytest.raises(ValueError):
        ops.kv8_shared_attention(**good, tile_rows=64)


def test_sizes_that_only_plain_attention_takes(cuda_device):
    """Bounds of the lengths and the prefix that are too large together for shared attention's plan: sequence by sequence."""
    dev = cuda_device
    case = Case("target", "fp8", CASES["pair"])
    args = list(case.args(dev))
    wide = torch.full((2, 5_000_000), -1, dtype=torch.int32, device=dev)
    wide[:, :case.table.shape[1]] = args[3]
    args[3], args[7], args[10] = wide, 100_000_000, 80_000_000
    announce("shared with bounds of 100 and 80 million tokens")
    ref.within(ops.kv8_shared_attention(case.q.to(dev), *args), *case.want())
    with pytest.raises(SdvError, match="unsupported sizes"):
        ops.kv8_shared_attention(case.q.to(dev), *args, tile_rows=32)
