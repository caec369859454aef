"""Where kv8_shared_attention takes kv8_attention: up to 16 rows a sequence and KV head below 2^18 keys that are not read again."""
from __future__ import annotations

import pytest

from test_shared_abi import _rows, lib  # noqa: F401  (the fixture)


@pytest.mark.parametrize("batch,prefix,rows", [
    (16, 8192, 0),        # 15 x 8192 x 2 keys: either way takes 19 us
    (32, 4096, 0),        # 31 x 4096 x 2, either way 17
    (9, 16384, 32),       # 8 x 16384 x 2 = 2^18
    (9, 16368, 0),
    (8, 32768, 32),
    (2, 32768, 0)])
def test_the_least_worth_sharing(lib, batch, prefix, rows):  # noqa: F811
    assert _rows(lib, B=batch, groups=1, total=batch, H=12, KV=2, D=128, rows=1, longest=prefix + 64, prefix=prefix) == rows
