"""A fork that fails leaves the destinations what they held (block copies by indexing in torch, no kernel launches)."""
from __future__ import annotations

import pytest

from specdec_amd import SdvError
from specdec_amd.engine import paged_cache
from test_fork import KINDS, Model, _copies  # noqa: F401  (the fixture)


def _snapshot(pool):
    return [list(b) for b in pool.blocks], list(pool.lengths), dict(pool.alloc.shared), sorted(pool.alloc.free)


@KINDS
@pytest.mark.parametrize("spare", [5, 1, 0])  # blocks besides what the sequences hold; two are copied
@pytest.mark.parametrize("first", ["own", "each other's", "fork", "forks of one"])
def test_a_copy_that_fails(kind, spare, first, monkeypatch):
    m = Model(kind, 4, (5 if "fork" in first else 7) + spare, growable=False)
    m.write(0, 40)
    if first == "own":
        m.write(1, 20)
        m.write(2, 17)
    elif first == "each other's":
        m.write(1, 40)
        m.fork(1, 2)
    else:
        m.fork(0, 1)
        m.fork(1 if first == "fork" else 0, 2, 33)
    before = _snapshot(m.pool)

    def fails(*a, **kw):
        raise SdvError("no copy")
    with monkeypatch.context() as patch:
        patch.setattr(paged_cache.ops, "copy_blocks", fails)
        with pytest.raises(SdvError, match="no copy"):
            m.pool.fork(0, [1, 2])
    assert _snapshot(m.pool) == before
    m.check()
    m.fork(0, [1, 2])
    m.check()


@KINDS
def test_an_exhausted_pool(kind):
    m = Model(kind, 4, 6, growable=False)
    m.write(0, 20)
    m.write(1, 37)
    m.fork(1, 2, 32)
    m.fork(1, [0, 2, 3])                     # three copies: the free block and the two that sequence 0 gives back
    assert m.pool.alloc.free == []
    m.check()
    m = Model(kind, 4, 6, growable=False)
    m.write(0, 20)
    m.write(1, 60)                           # the pool is full
    before = _snapshot(m.pool)
    with pytest.raises(RuntimeError, match="exhausted"):
        m.pool.fork(0, [2, 3])
    assert _snapshot(m.pool) == before
    with pytest.raises(RuntimeError, match="exhausted"):
        m.pool.fork(1, [0, 2, 3])            # three copies where two blocks would be given back
    assert _snapshot(m.pool) == before
    m.check()
    m.fork(1, [0, 2])                        # from what sequence 0 gives back
    m.check()


@KINDS
def test_a_pool_that_cannot_grow(kind, monkeypatch):
    m = Model(kind, 4, 6)
    m.write(0, 20)
    m.write(1, 60)
    before = _snapshot(m.pool)

    def fails(*a):
        raise MemoryError("no pages")
    monkeypatch.setattr(m.pool, "_new_pages", fails)
    with pytest.raises(MemoryError):
        m.pool.fork(1, [0, 2, 3])
    assert _snapshot(m.pool) == before
    m.check()
