"""KV8Cache at the ends of its use: sequences without tokens, streams that overlap, growth after a recording, prompts
layer after layer."""
from __future__ import annotations

import pytest
import torch

from conftest import announce
from specdec_amd.engine.kv8_cache import KV8Cache
from specdec_amd.engine.paged_cache import PagedKVCache

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


def _busy(stream):
    """About 100 ms of work on `stream`, and an event behind it."""
    with torch.cuda.stream(stream):
        torch.cuda._sleep(200_000_000)
    done = torch.cuda.Event()
    done.record(stream)
    return done


@pytest.mark.parametrize("what", ["table", "pages"])
def test_what_a_busy_stream_reads_is_not_given_away(cuda_device, what):
    """The block table, or the pages, are replaced on one stream while a call that reads the old ones waits on
    another: what the first stream allocates meanwhile, and writes, is other memory."""
    dev = cuda_device
    pool = KV8Cache(2, 128, batch=2, num_blocks=24, device=dev, seed=3)
    rows, q = _rows((200, 4, 128), 1).to(dev), _rows((2, 12, 128), 2).to(dev)
    pool.write(0, rows[:, :2], rows[:, 2:], [120, 80])
    want = pool.attend(0, q, counts=[1, 1])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        pool.attend(0, q, counts=[1, 1])  # its own row table and lengths
    torch.cuda.synchronize()
    old = [pool.block_table()] if what == "table" else [pool.k_pages, pool.v_pages, pool.scales]
    addresses, sizes = [t.data_ptr() for t in old], [t.numel() * t.element_size() for t in old]
    del old
    announce(f"kv8 pool: {what} replaced while a stream is busy")
    done = _busy(side)
    with torch.cuda.stream(side):
        late = pool.attend(0, q, counts=[1, 1])
    pool.reserve(0, 130 if what == "table" else 600)
    assert torch.equal(pool.attend(0, q, counts=[1, 1]), want)
    kept = []
    for size in sizes:
        for _ in range(64):
            kept.append(torch.full((size,), 1, dtype=torch.uint8, device=dev))
            assert kept[-1].data_ptr() not in addresses
    assert not done.query(), "the other stream was not busy for long enough to tell"
    torch.cuda.synchronize()
    assert torch.equal(late, want)


def test_two_streams_without_waits_of_the_host(cuda_device):
    """Steps that alternate between two streams, ordered by events alone, while the other allocates and writes
    memory of the tables' sizes: the same as on one stream."""
    dev = cuda_device
    counts = [[120, 60], [1, 5], [40, 1], [1, 5], [3, 3], [1, 1], [64, 64], [1, 1]]
    steps = [(_rows((sum(c), 12, 128), 10 + i).to(dev), _rows((sum(c), 2, 128), 30 + i).to(dev), _rows((sum(c), 2, 128), 50 + i).to(dev))
             for i, c in enumerate(counts)]
    one, two = (KV8Cache(2, 128, batch=2, num_blocks=4, device=dev, seed=3) for _ in range(2))
    want = [one.append_attend(0, *x, counts=c) for x, c in zip(steps, counts)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    announce("kv8 pool on two streams, ordered by events")
    got = []
    for i, (x, c) in enumerate(zip(steps, counts)):
        st, other = streams[i % 2], streams[1 - i % 2]
        st.wait_stream(other)
        with torch.cuda.stream(st):
            torch.cuda._sleep(2_000_000)
            got.append(two.append_attend(0, *x, counts=c))
        with torch.cuda.stream(other):
            for n in (3, 2, 8, 16, 40, 4096):
                torch.full((n,), 1, dtype=torch.int32, device=dev)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("kind", [KV8Cache, PagedKVCache])
def test_a_recorded_step_after_the_pool_has_grown(cuda_device, kind):
    """Growth replaces the pages and the block table: a graph recorded before keeps its own, whose memory nobody
    else is given, and repeats its results."""
    dev = cuda_device
    pool = kind(2, 128, batch=2, num_blocks=24, device=dev, seed=3)
    k, v = _rows((2, 100, 2, 128), 1).to(dev), _rows((2, 100, 2, 128), 2).to(dev)
    step = _rows((2, 1, 12, 128), 3).to(dev), _rows((2, 1, 2, 128), 4).to(dev), _rows((2, 1, 2, 128), 5).to(dev)
    pool.append(0, k, v, [0, 0])

    def run():
        return pool.append_attend(0, *step, [100, 100], q_token_major=True)

    want = run()
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        out = run()
    old = [pool.k_pages, pool.v_pages, pool.v_scales, pool.block_table()]
    addresses, sizes = [t.data_ptr() for t in old], [t.numel() * t.element_size() for t in old]
    del old
    pool.reserve_all(600)
    assert pool.k_pages.data_ptr() not in addresses and pool.block_table().data_ptr() not in addresses
    kept = []
    for size in sizes:
        for _ in range(64):
            kept.append(torch.zeros(size, dtype=torch.uint8, device=dev))
            assert kept[-1].data_ptr() not in addresses
    for turn in range(3):
        announce(f"{kind.__name__}: a graph from before the growth, replay {turn}")
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(run(), want)


@pytest.mark.parametrize("kind", [KV8Cache, PagedKVCache])
def test_prefill_of_layer_after_layer(cuda_device, kind):
    """A loop that hands a layer's slots on to the next, whichever the pool; each layer's tokens read back."""
    dev = cuda_device
    pool = kind(2, 128, num_layers=3, batch=2, capacity_tokens=64, device=dev, seed=2)
    pool.reserve_all(70, q_heads=12, q_len=5)
    k, v = _rows((3, 75, 2, 128), 1).to(dev), _rows((3, 75, 2, 128), 2).to(dev)
    slots = None
    announce(f"{kind.__name__}: prefill of three layers")
    for layer in range(3):
        slots = pool.prefill(layer, k[layer], v[layer], [70, 5], slots)
    assert pool.lengths == [70, 5]
    for layer in range(3):
        for seq, rows in enumerate((slice(0, 70), slice(70, 75))):
            got = pool.gather(layer, seq)[0].transpose(0, 1).float()
            want = k[layer, rows].float()
            # the code is off by half a step, 2^-4 of it or half of the smallest, 2^-10 (scale max / 448); what is
            # read back then by 2^-8 (BF16; the scale's and the product's roundings of 2^-24 are within the 2^-9 more)
            off = want.abs() * 2.0 ** -4 + want.abs().amax(-1, keepdim=True) / 448 * 2.0 ** -10
            assert bool(((got - want).abs() <= off + (want.abs() + off) * (2.0 ** -8 + 2.0 ** -9)).all())


def test_growth_gives_the_old_pages_back(cuda_device):
    """Where nothing was recorded the pool that has grown holds its new pages alone."""
    pool = KV8Cache(2, 128, batch=1, num_blocks=1024, device=cuda_device)
    rows = _rows((20, 4, 128), 1).to(cuda_device)
    pool.write(0, rows[:, :2], rows[:, 2:], [20])
    torch.cuda.synchronize()
    old = sum(t.numel() * t.element_size() for t in (pool.k_pages, pool.v_pages, pool.scales))
    before = torch.cuda.memory_allocated()
    pool.reserve(0, 1025 * 16)
    assert torch.cuda.memory_allocated() - before <= old  # twice the blocks, and the old ones free again
