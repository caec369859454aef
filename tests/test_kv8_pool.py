"""KV8Cache's bookkeeping beyond the plain calls, on the CPU (no kernel launches)."""
from __future__ import annotations

import pytest
import torch

from specdec_amd.engine import kv8_cache
from specdec_amd.engine.kv8_cache import KV8Cache


def test_lengths_of_another_batch_are_refused():
    pool = KV8Cache(2, 64, batch=2, capacity_tokens=32, device="cpu")
    q = torch.zeros((2, 4, 1, 64), dtype=torch.bfloat16)
    for lengths in ([5], [5, 5, 5], [-1, 3]):
        with pytest.raises(ValueError):
            pool.attend(0, q, lengths=lengths)


@pytest.mark.parametrize("lengths,table,longest", [([0, 0], [0, 0], 1), ([0, 3], [0, 3], 3), ([3, 3], None, 3), ([0], [0], 1)])
def test_lengths_that_attention_is_given(monkeypatch, lengths, table, longest):
    """Equal lengths are one number, which cannot be 0."""
    pool = KV8Cache(2, 64, batch=len(lengths), capacity_tokens=32, device="cpu")
    for b, n in enumerate(lengths):
        pool.reserve(b, max(n, 1))
    seen = []
    monkeypatch.setattr(kv8_cache.ops, "kv8_attention", lambda q, *a, **kw: (seen.append(a), q)[1])
    pool.attend(0, torch.zeros((len(lengths), 4, 1, 64), dtype=torch.bfloat16), lengths=lengths)
    *_, lens, most_rows, most_len = seen[0]
    assert (lens if lens is None else lens.tolist()) == table and most_len == longest and most_rows == 1
