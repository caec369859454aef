"""Blocks that a recorded step writes are not shared by a later fork, in the pools' bookkeeping (block copies by indexing in torch,
no kernel launches)."""
from __future__ import annotations

import pytest
import torch

from specdec_amd import SdvError
from specdec_amd.engine import kv8_cache, paged_cache
from specdec_amd.engine.kv8_cache import KV8Cache
from specdec_amd.engine.paged_cache import PagedKVCache
from test_fork import KINDS, Model, _copies  # noqa: F401  (the fixture)


def _record(m, monkeypatch, counts, starts, rope=False):
    """A step of counts[b] rows from positions starts[b] on, recorded: the pool's side of it.  The lengths are set back."""
    p, n = m.pool, sum(counts)
    lengths = list(p.lengths)
    with monkeypatch.context() as patch:
        for name in ("kv8_append", "kv8_rope_append", "quant_append_pages", "append_attend_pages", "attention_workspace_bytes"):
            patch.setattr(paged_cache.ops, name, lambda *a, **kw: 64)
        patch.setattr(paged_cache.ops, "new_workspace", lambda dev, n: torch.empty(n, dtype=torch.uint8))

        def step():
            q, k = torch.zeros((n, 4, 64), dtype=torch.bfloat16), torch.zeros((n, 2, 64), dtype=torch.bfloat16)
            if isinstance(p, KV8Cache):
                if rope:
                    p.rope_write(0, q, k, k, counts, torch.ones(32, dtype=torch.float64), starts)
                else:
                    p.write(0, k, k, counts, starts)
            else:
                s = counts[0]
                p.append_attend(0, q.view(-1, 4, s, 64), k.view(-1, s, 2, 64), k.view(-1, s, 2, 64), starts)
        step()
        for module in (paged_cache, kv8_cache):
            patch.setattr(module, "_recording", lambda dev: True)
        step()
    p.lengths[:] = lengths


@KINDS
@pytest.mark.parametrize("rope", [False, True])
@pytest.mark.parametrize("at,rows,fork,own", [
    (30, 5, 35, [1, 2]),      # the block that the fork would share, and the last one
    (30, 5, 32, [1]),
    (30, 5, 16, []),          # what is recorded lies behind the fork
    (100, 1, 112, [6]),
    (32, 24, 56, [2, 3]),     # a tree whose tokens are part of the fork
    (35, 5, 35, [2])])        # from the fork on
def test_a_fork_copies_what_a_recorded_step_writes(kind, rope, at, rows, fork, own, monkeypatch):
    m = Model(kind, 3, 64)
    for b in range(3):
        m.write(b, 120)
    _record(m, monkeypatch, [rows] * 3, [at] * 3, rope)
    for b in range(3):
        m.trim(b, fork)
    before = list(m.pool.blocks[0])
    m.fork(0, [1, 2])
    m.check()
    a = m.pool.blocks[0]
    assert a == before                       # the source goes on as it was
    for b in (1, 2):
        assert [j for j, x in enumerate(m.pool.blocks[b]) if x != a[j]] == own
    for x in a[at // 16:-(-(at + rows) // 16)]:
        assert x not in m.pool.alloc.shared


@KINDS
def test_a_later_owner_shares_again(kind, monkeypatch):
    """A block that has been given back and out again is its new owner's, whatever was recorded before."""
    m = Model(kind, 2, 6)
    m.write(0, 48)
    m.write(1, 48)
    _record(m, monkeypatch, [48] * 2, [0] * 2)
    assert len(m.pool.alloc.recorded) == 6
    m.free(0)
    m.write(0, 48)
    m.fork(0, 1)
    assert m.pool.blocks[0] == m.pool.blocks[1] and m.pool.alloc.shared
    m.check()


@KINDS
@pytest.mark.parametrize("call", ["compact", "grow"])
def test_new_pages_are_shared_again(kind, call, monkeypatch):
    """What a graph writes after the pool has grown or moved does not reach its new pages."""
    m = Model(kind, 2, 6)
    m.write(0, 48)
    m.write(1, 48)
    _record(m, monkeypatch, [48] * 2, [0] * 2)
    m.pool.compact() if call == "compact" else m.write(1, 1)
    m.fork(0, 1)
    assert m.pool.blocks[0] == m.pool.blocks[1]
    m.check()


@KINDS
def test_a_fork_that_fails_forgets_no_recording(kind, monkeypatch):
    m = Model(kind, 2, 6, growable=False)
    m.write(0, 48)
    m.write(1, 48)
    _record(m, monkeypatch, [20] * 2, [0] * 2)
    recorded = set(m.pool.alloc.recorded)

    def fails(*a, **kw):
        raise SdvError("no copy")
    with monkeypatch.context() as patch:
        patch.setattr(paged_cache.ops, "copy_blocks", fails)
        with pytest.raises(SdvError, match="no copy"):
            m.pool.fork(0, 1)
    assert m.pool.alloc.recorded == recorded and len(recorded) == 4
    m.check()
    m.fork(0, 1)                             # two blocks of its own, from those it gave back
    assert [x == y for x, y in zip(*m.pool.blocks)] == [False, False, True]
    m.check()


def test_a_recorded_prefill(monkeypatch):
    m = Model(PagedKVCache, 2, 16)
    m.write(0, 40)
    x = torch.zeros((40, 2, 64), dtype=torch.bfloat16)
    seen = []
    monkeypatch.setattr(m.pool, "_hold_writes", lambda starts, ends: seen.append((list(starts), list(ends))))
    monkeypatch.setattr(paged_cache.ops, "quant_append_pages", lambda *a, **kw: True)
    monkeypatch.setattr(paged_cache.ops, "_stream", lambda dev: 0)
    monkeypatch.setattr(m.pool, "_layer_pointers", lambda *a: None)
    slots = m.pool.prefill(0, x, x, [40, 0])
    assert seen == []
    m.pool.device = torch.device("cuda")
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    m.pool.prefill(0, x, x, [40, 0], slots=slots)
    assert seen == [([0, 0], [40, 0])]
