"""KV8Cache at the ends of its use: sequences without tokens."""
from __future__ import annotations

import pytest
import torch

from conftest import announce
from specdec_amd.engine.kv8_cache import KV8Cache

pytestmark = pytest.mark.gpu


def _rows(shape, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)


@pytest.mark.parametrize("batch", [1, 2])
@pytest.mark.parametrize("rows", [1, 40])
def test_attend_without_tokens(cuda_device, batch, rows):
    """Rows of sequences of length 0 see nothing and are 0, whatever the pages hold from before; the same beside
    a sequence that has tokens."""
    dev = cuda_device
    pool = KV8Cache(2, 128, batch=batch, capacity_tokens=64, device=dev)
    k, v, q = (_rows((batch * rows, n, 128), n).to(dev) for n in (2, 3, 12))
    v = v[:, :2]
    announce(f"kv8 pool without tokens {batch} {rows}")
    full = pool.append_attend(0, q, k, v, counts=[rows] * batch)
    assert bool((full != 0).any())
    for b in range(batch):
        pool.set_length(b, 0)
    assert bool((pool.attend(0, q, counts=[rows] * batch) == 0).all())
    grid = q.view(batch, rows, 12, 128)
    assert bool((pool.attend(0, grid, q_token_major=True, lengths=[0] * batch) == 0).all())
    if batch > 1:
        got = pool.attend(0, q, counts=[rows] * batch, lengths=[0, rows])
        assert bool((got[:rows] == 0).all()) and torch.equal(got[rows:], full[rows:])
    pool.write(0, k[:0], v[:0], [0] * batch)
    assert pool.lengths == [0] * batch and pool.attend(0, q[:0], counts=[0] * batch).shape == (0, 12, 128)
