"""Writes and reads of the 8-bit cache that touch more page blocks than a launch has wavefronts for are refused on the host."""
from __future__ import annotations

import pytest

from specdec_amd import _native
from test_kv8_abi import _append, _gather, lib  # noqa: F401  (the fixture)
from test_moves_abi import _step


@pytest.mark.parametrize("call", [_append, _gather, _step])
def test_more_blocks_than_wavefronts(lib, call):  # noqa: F811
    for bad in (dict(n=1 << 26, B=1 << 26), dict(n=1 << 30, B=1), dict(n=(1 << 30) - 32, B=1), dict(n=1 << 27, B=29360128)):
        assert call(lib, **bad) == _native.SDV_ERR_SHAPE, bad


def test_more_tiles_than_wavefronts():
    from test_native_abi import N, P

    lib = _native.load()  # noqa: F811
    quant = lambda n, tiles: lib.sdv_quant_append_tiles(P, P, P, n, 2, 64, 64, 1, 0, P, P, P, 8, 0, 0, 0, _native.SCALE_DIV, P, tiles, N)  # noqa: E731
    for n, tiles in ((1 << 27, 1 << 26), (1 << 27, (1 << 31) - 1)):
        assert quant(n, tiles) == _native.SDV_ERR_SHAPE
    assert lib.sdv_quant_append(P, P, P, (1 << 30) + 1, 1, 64, 64, 1, 0, P, P, P, 8, 0, 0, 0, _native.SCALE_DIV, N) == _native.SDV_ERR_SHAPE
    for kv, t in ((1, 1 << 30), (64, 1 << 24)):
        assert lib.sdv_pack_contiguous(P, P, P, 1, kv, t, 64, P, P, P, P, N) == _native.SDV_ERR_SHAPE
