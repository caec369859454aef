"""Forks, copies before a write, compaction and kept paths in the pools' bookkeeping, on the CPU (block copies by indexing in
torch, no kernel launches)."""
from __future__ import annotations

import random

import pytest
import torch

from specdec_amd import SdvError
from specdec_amd.engine import kv8_cache, paged_cache
from specdec_amd.engine.kv8_cache import KV8Cache
from specdec_amd.engine.paged_cache import BlockAllocator, PagedKVCache

KINDS = pytest.mark.parametrize("kind", [PagedKVCache, KV8Cache])


@pytest.fixture(autouse=True)
def _copies(monkeypatch):
    def copy(k, v, s, src, dst, *, to=None):
        for x, y in zip((k, v, s), to or (k, v, s)):
            y.view(torch.uint8)[:, dst.long()] = x.view(torch.uint8)[:, src.long()]
    monkeypatch.setattr(paged_cache.ops, "copy_blocks", copy)


class Model:
    """A pool whose every token is written as its number into its scale slots, and what each sequence should hold."""

    def __init__(self, kind, batch, blocks, seed=None, growable=True):
        self.pool = kind(2, 64, num_layers=2, batch=batch, num_blocks=blocks, device="cpu", seed=seed, growable=growable)
        self.want = [[] for _ in range(batch)]
        self.next = 2.0

    def write(self, b, n):
        p, at = self.pool, len(self.want[b])
        p.reserve(b, at + n)
        starts, ends = list(p.lengths), list(p.lengths)
        ends[b] += n
        if p.alloc.shared:
            p._own(starts, ends)
        for i in range(at, at + n):
            p.v_scales[:, p.blocks[b][i // 16], ..., i % 16] = self.next
            self.want[b].append(self.next)
            self.next += 1
        p.set_length(b, at + n)

    def trim(self, b, n):
        self.pool.set_length(b, n)
        del self.want[b][n:]

    def fork(self, src, dst, n=None):
        self.pool.fork(src, dst, n)
        for d in [dst] if isinstance(dst, int) else dst:
            self.want[d] = self.want[src][:n]

    def free(self, b):
        self.pool.free_sequence(b)
        self.want[b] = []

    def check(self):
        p = self.pool
        assert p.lengths == [len(w) for w in self.want]
        held = {}
        for blocks in p.blocks:
            assert len(set(blocks)) == len(blocks)
            for x in blocks:
                held[x] = held.get(x, 0) + 1
        assert p.alloc.shared == {x: n - 1 for x, n in held.items() if n > 1}
        assert sorted([*held, *p.alloc.free]) == list(range(p.alloc.num_blocks)) == list(range(p.k_pages.shape[1]))
        for b, w in enumerate(self.want):
            for layer in range(2):
                s = p.layer(layer)[2]
                got = [s[p.blocks[b][i // 16], ..., i % 16].flatten() for i in range(len(w))]
                assert all(bool((g == x).all()) for g, x in zip(got, w)), (b, layer)


@KINDS
@pytest.mark.parametrize("seed", range(12))
def test_any_order_of_calls(kind, seed):
    rng = random.Random(seed)
    m = Model(kind, 5, rng.choice([1, 8, 40]), seed if seed % 2 else None)
    for _ in range(60):
        b = rng.randrange(5)
        what = rng.choice(["write", "write", "write", "fork", "fork", "trim", "free", "compact"])
        if what == "write":
            m.write(b, rng.choice([0, 1, 5, 16, 17, 40]))
        elif what == "fork":
            n = rng.choice([None, rng.randint(0, len(m.want[b]))])
            m.fork(b, rng.sample([x for x in range(5) if x != b], rng.randint(0, 3)), n)
        elif what == "trim":
            m.trim(b, rng.randint(0, len(m.want[b])))
        elif what == "free":
            m.free(b)
        else:
            used = len({x for blocks in m.pool.blocks for x in blocks})
            m.pool.compact(rng.choice([None, used + 3]))
        m.check()
        if isinstance(m.pool, KV8Cache):
            _check_groups(m.pool, [rng.randint(0, 3) for _ in range(5)], m.pool.lengths)


def _check_groups(pool, counts, lengths):
    got = pool._groups(counts, lengths)
    if got is None:
        return
    cu, prefix, longest = got[0].tolist(), got[1].tolist(), got[2]
    assert cu[0] == 0 and cu[-1] <= pool.batch and all(a < b for a, b in zip(cu, cu[1:])) and longest == max(prefix) > 0
    for a, b in zip(cu, cu[1:]):
        p = prefix[a]
        assert prefix[a:b] == [p] * (b - a) and p % 16 == 0 and (p == 0 or b - a > 1)
        for x in range(a, b):
            assert p <= max(0, lengths[x] - counts[x]) and pool.blocks[x][:p // 16] == pool.blocks[a][:p // 16]
    assert not any(prefix[cu[-1]:])


@KINDS
def test_fork_shares_whole_blocks(kind):
    m = Model(kind, 4, 8)
    m.write(0, 37)
    m.fork(0, [1, 3])
    p = m.pool
    assert p.blocks[1][:2] == p.blocks[3][:2] == p.blocks[0][:2] and len({p.blocks[b][2] for b in (0, 1, 3)}) == 3
    assert p.alloc.shared == {b: 2 for b in p.blocks[0][:2]} and len(p.alloc.free) == 3
    for b in (0, 1, 3):
        m.write(b, 3)
    m.check()
    m.fork(3, 2, 32)                     # a whole number of blocks: nothing is copied
    assert p.blocks[2] == p.blocks[0][:2] and len(p.alloc.free) == 3
    m.fork(1, 2, 0)
    assert p.blocks[2] == [] and p.lengths[2] == 0
    m.free(0)
    m.check()
    m.free(1)
    assert p.alloc.shared == {}          # only sequence 3 holds them now
    m.check()


@KINDS
def test_a_write_below_the_fork_leaves_the_others(kind):
    m = Model(kind, 3, 8)
    m.write(0, 64)
    m.fork(0, [1, 2])
    m.trim(1, 20)
    m.write(1, 30)
    m.check()
    assert m.pool.blocks[1][0] == m.pool.blocks[0][0] and not set(m.pool.blocks[1][1:]) & set(m.pool.blocks[0])
    m.trim(0, 0)
    m.write(0, 64)                       # the one that was forked
    m.check()
    assert not set(m.pool.blocks[0]) & (set(m.pool.blocks[1]) | set(m.pool.blocks[2]))


@KINDS
def test_reserve_all_gives_a_sequence_its_own_blocks(kind):
    m = Model(kind, 2, 8)
    m.write(0, 48)
    m.fork(0, 1)
    m.trim(1, 16)
    m.pool.reserve_all(48)
    assert m.pool.blocks[1][0] == m.pool.blocks[0][0] and not set(m.pool.blocks[1][1:]) & set(m.pool.blocks[0])
    m.check()


@KINDS
def test_refusals(kind):
    m = Model(kind, 3, 4, growable=False)
    m.write(0, 40)
    for args in ((0, 0), (0, [1, 1]), (0, 3), (0, -1), (3, 0), (-1, 0), (0, 1, 41), (0, 1, -1)):
        with pytest.raises(ValueError):
            m.pool.fork(*args)
    m.check()
    m.fork(0, 1)
    with pytest.raises(RuntimeError):
        m.pool.fork(0, 2)                # a fifth block
    m.check()
    m.fork(0, 2, 32)
    with pytest.raises(ValueError):
        m.pool.compact(3)
    m.pool.set_length(2, 10)
    m.want[2] = m.want[2][:10]
    with pytest.raises(RuntimeError):
        m.write(2, 1)                    # no block for the copy
    m.check()


@KINDS
@pytest.mark.parametrize("call", ["fork", "compact", "write"])
def test_a_copy_that_fails_loses_no_blocks(kind, call, monkeypatch):
    m = Model(kind, 3, 12)
    m.write(0, 40)
    m.fork(0, 1)
    m.trim(1, 20)

    def fails(*a, **kw):
        raise SdvError("no copy")
    monkeypatch.setattr(paged_cache.ops, "copy_blocks", fails)
    with pytest.raises(SdvError, match="no copy"):
        {"fork": lambda: m.pool.fork(0, 2), "compact": m.pool.compact, "write": lambda: m.write(1, 1)}[call]()
    m.check()


@KINDS
@pytest.mark.parametrize("call", ["fork", "compact", "write"])
def test_a_recording_is_refused(kind, call, monkeypatch):
    m = Model(kind, 3, 12)
    m.write(0, 40)
    m.fork(0, 1)
    m.trim(1, 20)
    monkeypatch.setattr(paged_cache, "_recording", lambda dev: True)
    with pytest.raises(SdvError, match="recorded"):
        {"fork": lambda: m.pool.fork(0, 2), "compact": m.pool.compact, "write": lambda: m.write(1, 1)}[call]()
    monkeypatch.undo()
    m.check()


def test_a_prefill_over_a_fork_refuses_old_slots():
    m = Model(PagedKVCache, 2, 12)
    m.write(0, 40)
    slots = m.pool.varlen_slots([40, 0])
    m.fork(0, 1)
    x = torch.zeros((40, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(SdvError, match="slots"):
        m.pool.prefill(0, x, x, [40, 0], slots=slots)


def test_release_without_forks_is_as_it_was():
    a = BlockAllocator(8)
    x = a.alloc(3)
    a.share(x[:1])
    a.share(x[:1])
    a.release(x)
    assert a.shared == {x[0]: 1} and a.free[-2:] == [x[2], x[1]]
    a.release(x[:1])
    assert a.shared == {} and x[0] not in a.free
    a.release(x[:1])
    assert a.free[-1] == x[0] and len(a.free) == 8


def test_groups():
    m = Model(KV8Cache, 7, 64)
    m.write(0, 40)
    m.write(1, 100)
    m.fork(1, [2, 3])
    m.write(2, 10)
    m.write(4, 16)
    m.write(5, 64)
    m.fork(5, 6)
    groups = lambda counts, lens=None: [x if isinstance(x, int) else x.tolist() for x in m.pool._groups(counts, lens or m.pool.lengths)]  # noqa: E731
    assert groups([0] * 7) == [[0, 1, 4, 5, 7], [0, 96, 96, 96, 0, 64, 64], 96]
    assert groups([1] * 7) == [[0, 1, 4, 5, 7], [0, 96, 96, 96, 0, 48, 48], 96]            # of 63 tokens before the new ones
    assert groups([0, 0, 0, 5, 0, 49, 0]) == [[0, 1, 4, 7], [0, 80, 80, 80, 0, 0, 0], 80]   # less than a block: none
    assert groups([0] * 7, [40, 100, 40, 10, 16, 64, 64]) == [[0, 1, 3, 5, 7], [0, 32, 32, 0, 0, 64, 64], 64]
    m.free(6)
    m.fork(3, 6, 40)                                                                     # not a neighbour
    assert groups([0] * 7) == [[0, 1, 4, 7], [0, 96, 96, 96, 0, 0, 0], 96]
    m.fork(3, 4, 32)                                                                     # less than half of what they share
    assert groups([0] * 7)[:2] == [[0, 1, 4, 7], [0, 96, 96, 96, 0, 0, 0]]
    m.fork(3, 4, 50)
    assert groups([0] * 7)[:2] == [[0, 1, 5, 7], [0, 48, 48, 48, 48, 0, 0]]
    m.free(2)
    assert groups([0] * 7)[:2] == [[0, 3, 5, 7], [0, 0, 0, 48, 48, 0, 0]]
    for b in (1, 3, 4, 6):
        m.free(b)
    assert m.pool._groups([0] * 7, m.pool.lengths) is None


def test_blocks_behind_a_block_of_ones_own_are_not_shared():
    """After a trim and a rewrite the blocks behind are the old ones until they are written: they are no prefix."""
    m = Model(KV8Cache, 2, 16)
    m.write(0, 64)
    m.fork(0, 1)
    m.trim(1, 16)
    m.write(1, 16)
    m.pool.set_length(1, 64)
    assert m.pool.blocks[1][2:] == m.pool.blocks[0][2:]
    assert m.pool._groups([0, 0], [64, 64])[1].tolist() == [16, 16]


@pytest.mark.parametrize("shared", [False, True])
def test_attend_reads_shared_blocks_once(monkeypatch, shared):
    m = Model(KV8Cache, 2, 16)
    m.write(0, 64)
    m.fork(0, 1)
    if not shared:
        m.free(0)
        m.pool.reserve(0, 64)
    seen = []
    for name in ("kv8_attention", "kv8_shared_attention"):
        monkeypatch.setattr(kv8_cache.ops, name, lambda q, *a, name=name, **kw: (seen.append((name, a)), q)[1])
    m.pool.attend(0, torch.zeros((2, 4, 1, 64), dtype=torch.bfloat16), lengths=[64, 64])
    (name, args), = seen
    if shared:
        assert name == "kv8_shared_attention" and args[6:8] == (1, 64) and [args[8].tolist(), args[9].tolist(), args[10]] == [[0, 2], [48, 48], 48]
    else:
        assert name == "kv8_attention"


def test_keep(monkeypatch):
    m = Model(KV8Cache, 3, 16)
    for b, n in enumerate((20, 40, 33)):
        m.write(b, n)
    seen = []
    monkeypatch.setattr(kv8_cache.ops, "kv8_keep", lambda *a: seen.append([x.tolist() for x in a[4:]]))
    for paths, starts in (([[0], [0]], [1, 1, 1]), ([[0], [0], []], [1, 1]), ([[1, 0], [], []], [10, 40, 33]), ([[0, 0], [], []], [10, 40, 33]),
                          ([[10], [], []], [10, 40, 33]), ([[-1], [], []], [10, 40, 33]), ([[], [], []], [21, 40, 33]), ([[], [], []], [-1, 40, 33])):
        with pytest.raises(ValueError):
            m.pool.keep(paths, starts)
    assert m.pool.lengths == [20, 40, 33]
    m.pool.keep([[0, 1, 2], [], []], [10, 40, 30])
    assert m.pool.lengths == [13, 40, 30] and seen == []  # nothing to move
    m.pool.keep([[0, 2], [0, 1, 3, 9], []], [10, 30, 30])
    assert m.pool.lengths == [12, 34, 30] and seen == [[[0, 1, 3, 3], [1, 1, 7], [11, 32, 30]]]


def test_keep_does_not_move_tokens_of_a_fork(monkeypatch):
    m = Model(KV8Cache, 2, 16)
    m.write(0, 48)
    m.fork(0, 1)
    tables = []
    monkeypatch.setattr(kv8_cache.ops, "kv8_keep", lambda k, v, s, bt, *a: tables.append(bt.tolist()))
    m.pool.keep([[], [0, 9]], [48, 20])
    assert tables[0][0] == m.pool.blocks[0] and tables[0][1][0] == tables[0][0][0] and tables[0][1][1] != tables[0][0][1]
    assert m.pool.lengths == [48, 22]
    m.want[1] = m.want[0][:22]
    m.check()                            # the copy holds what the block held (nothing was moved here)


def test_rope_arguments_need_frequencies():
    pool = KV8Cache(2, 64, batch=1, capacity_tokens=32, device="cpu")
    q, k = torch.zeros((1, 4, 64), dtype=torch.bfloat16), torch.zeros((1, 2, 64), dtype=torch.bfloat16)
    for kw in (dict(interleaved=True), dict(rope_scale=2.0), dict(positions=torch.zeros(1, dtype=torch.int32))):
        with pytest.raises(ValueError):
            pool.append_attend(0, q, k, k, counts=[1], **kw)
    with pytest.raises(SdvError):
        pool.append_attend(0, q, k, k, counts=[1], rope=torch.ones(32, dtype=torch.float64))  # CPU tensors: no kernel
    with pytest.raises(SdvError):
        pool.append_attend(0, q[None].transpose(1, 2), k[None, :0], k[None, :0], rope=torch.ones(32, dtype=torch.float64))
    assert pool.lengths == [0]
