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
