"""The pools' forks, rotary writes, trees, kept paths and compaction as a server uses them together, against a pool whose sequences
each have their own copy of everything, and against attention in 64 bits (tests/kv8_reference.py, with its bound)."""
from __future__ import annotations

import random

import pytest
import torch

import kv8_reference as ref
from conftest import announce
from specdec_amd import _native
from specdec_amd.engine.kv8_cache import KV8Cache
from specdec_amd.engine.paged_cache import PagedKVCache
from specdec_amd.kernels import ops

pytestmark = pytest.mark.gpu
HEADS = {"target": (12, 2, 128), "draft": (14, 2, 64), "mha": (4, 4, 128)}


def _rows(shape, seed):
    x = torch.randn(shape, generator=torch.Generator().manual_seed(seed))
    x[..., 3] *= 8.0
    return x.to(torch.bfloat16)


def _trees(rng, batch, most):
    """Per sequence: (parents of its nodes, ancestor words, depths)."""
    out = []
    for _ in range(batch):
        n = rng.randint(1, most)
        parents = [-1] + [rng.randrange(i) for i in range(1, n)]
        words, depth = [], []
        for i, p in enumerate(parents):
            words.append((words[p] if p >= 0 else 0) | 1 << i)
            depth.append(depth[p] + 1 if p >= 0 else 0)
        out.append((parents, words, depth))
    return out


def _path(rng, parents):
    """The nodes from the root to one of the tree's."""
    at, path = rng.randrange(len(parents)), []
    while at >= 0:
        path.append(at)
        at = parents[at]
    return path[::-1]


def _bytes(pool):
    """Codes and scales of every sequence's tokens, all layers: [(k, v, scales)], each with the tokens first, on the CPU."""
    k, v, s = (t.view(torch.uint8).cpu() for t in (pool.k_pages, pool.v_pages, pool.scales))
    s = s.view(torch.float32)
    out = []
    for blocks, n in zip(pool.blocks, pool.lengths):
        i = torch.arange(n)
        blk, off = torch.tensor(blocks, dtype=torch.long)[i // 16], i % 16
        out.append((k[:, blk, :, off // 4, :, off % 4], v[:, blk, :, :, off], s[:, blk, :, :, off]))
    return out


def _same(one, two):
    assert one.lengths == two.lengths
    for a, b in zip(_bytes(one), _bytes(two)):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def _exact(pool, layer, q, counts, words):
    pages = ref.Pages(pool.alloc.num_blocks, pool.kv_heads, pool.head_dim, pool.kv_format)
    pages.k, pages.v, pages.s = (t.cpu() for t in pool.layer(layer))
    pages.k, pages.v = pages.k.view(torch.uint8), pages.v.view(torch.uint8)
    return ref.attention(q.cpu(), pages, pool.block_table().cpu(), list(counts), pool.lengths, tree=words)


@pytest.mark.parametrize("seed", [None, 5])
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("heads", list(HEADS))
def test_a_prompt_that_many_continue(cuda_device, heads, fmt, seed):
    dev = cuda_device
    h, kv, d = HEADS[heads]
    L, B, rng = 2, 6, random.Random(11)
    inv, scale = ops.rope_frequencies(d, scaling={"type": "yarn", "factor": 4.0, "original": 128}, device=dev)
    how = dict(interleaved=heads == "draft", rope_scale=scale)
    prompts = [150, 40]                                 # of sequences 0 (to be forked into 1 to 4) and 5
    shared = KV8Cache(kv, d, kv_format=fmt, num_layers=L, batch=B, num_blocks=16, device=dev, seed=seed)
    alone = KV8Cache(kv, d, kv_format=fmt, num_layers=L, batch=B, num_blocks=96, device=dev, seed=seed)
    for layer in range(L):
        q, k, v = (_rows((n, heads_, d), 10 * layer + i).to(dev) for i, (n, heads_) in enumerate([(190, h), (190, kv), (190, kv)]))
        announce(f"fork {heads} {fmt} {seed}: prompts, layer {layer}")
        got = shared.rope_write(layer, q, k, v, [150, 0, 0, 0, 0, 40], inv, [0] * B, **how)
        each = [torch.cat([t[:150]] * 5 + [t[150:]]) for t in (q, k, v)]
        want = alone.rope_write(layer, *each, [150] * 5 + [40], inv, [0] * B, **how)
        assert torch.equal(got[:150], want[:150]) and torch.equal(got[150:], want[750:])
    shared.fork(0, [1, 2, 3, 4])
    assert len({b for blocks in shared.blocks for b in blocks}) == 9 + 5 + 3 and prompts == [shared.lengths[0], shared.lengths[5]]
    _same(shared, alone)
    for step in range(4):
        trees = _trees(rng, B, [1, 5, 24, 24][step])
        counts = [len(t[0]) for t in trees]
        words = [w for t in trees for w in t[1]]
        starts = list(shared.lengths)
        pos = torch.tensor([s + x for s, t in zip(starts, trees) for x in t[2]], dtype=torch.int32, device=dev)
        mask = torch.tensor(words, dtype=torch.int64, device=dev)
        for layer in range(L):
            q, k, v = (_rows((sum(counts), n, d), 100 * step + 10 * layer + i).to(dev) for i, n in enumerate((h, kv, kv)))
            announce(f"fork {heads} {fmt} {seed}: step {step}, layer {layer}, {counts}")
            args = (layer, q, k, v, starts)
            kw = dict(counts=counts, tree_mask=mask, rope=inv, positions=pos, **how)
            got, other = shared.append_attend(*args, **kw), alone.append_attend(*args, **kw)
            turned = ops.rope(q, None, pos, inv, interleaved=how["interleaved"], scale=scale)[0]
            want = _exact(shared, layer, turned, counts, mask.cpu())
            ref.within(got, *want)
            ref.within(other, *want)
        _same(shared, alone)
        before = _bytes(shared)
        paths = [_path(rng, t[0]) for t in trees]
        shared.keep(paths, starts)
        alone.keep(paths, starts)
        assert shared.lengths == [s + len(p) for s, p in zip(starts, paths)]
        for old, new, s, p in zip(before, _bytes(shared), starts, paths):
            rows = torch.tensor(list(range(s)) + [s + i for i in p])
            assert all(torch.equal(b, a[rows]) for a, b in zip(old, new))
        _same(shared, alone)
        if step == 1:
            shared.compact()
            assert shared.alloc.free == [] and shared.k_pages.shape[1] == len({b for blocks in shared.blocks for b in blocks})
            _same(shared, alone)
        if step == 2:                                   # the one that was forked goes, the others stay
            shared.free_sequence(0)
            alone.free_sequence(0)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_grids_of_rows_take_positions_too(cuda_device, fmt):
    """(B, H, S, D) and (B, S, H, D) with rope, and out, give what the packed rows give."""
    dev = cuda_device
    inv, _ = ops.rope_frequencies(128, device=dev)
    x = [_rows((3, 5, n, 128), n + i).to(dev) for i, n in enumerate((12, 2, 2))]
    packed, token, head = (KV8Cache(2, 128, kv_format=fmt, batch=3, device=dev) for _ in range(3))
    announce(f"rope in grids {fmt}")
    want = packed.append_attend(0, *(t.flatten(0, 1) for t in x), counts=[5] * 3, rope=inv)
    out = torch.empty_like(x[0])
    got = token.append_attend(0, *x, q_token_major=True, rope=inv, out=out)
    assert got is out and torch.equal(out.flatten(0, 1), want)
    got = head.append_attend(0, x[0].transpose(1, 2).contiguous(), *x[1:], rope=inv)
    assert torch.equal(got.transpose(1, 2).flatten(0, 1), want)
    _same(packed, token)
    _same(packed, head)


@pytest.mark.parametrize("kind", ["fp8", "int8", "v_fp8"])
def test_a_write_below_the_fork(cuda_device, kind):
    """A fork trimmed below what it shares and written on: both go on as sequences of their own; the same after compact()."""
    dev = cuda_device
    new = lambda: (PagedKVCache(2, 64, num_layers=3, batch=2, num_blocks=8, device=dev) if kind == "v_fp8" else  # noqa: E731
                   KV8Cache(2, 64, kv_format=kind, num_layers=3, batch=2, num_blocks=8, device=dev))
    shared, alone = new(), new()
    k, v = (_rows((100, 2, 64), i).to(dev) for i in (1, 2))
    more = [_rows((2, 40, 2, 64), 5 + i).to(dev) for i in range(2)]
    q = _rows((2, 14, 40, 64), 9).to(dev)
    announce(f"a write below the fork {kind}")
    for layer in range(3):
        shared.prefill(layer, k, v, [100, 0])
        alone.prefill(layer, torch.cat([k, k]), torch.cat([v, v]), [100, 100])
    shared.fork(0, 1)
    for turn in range(2):
        starts = [[100, 21], [140, 61]][turn]
        for layer in range(3):
            got = shared.append_attend(layer, q, *more, starts)
            want = alone.append_attend(layer, q, *more, starts)
            assert torch.equal(got, want)               # what is shared here is less than shared attention is taken for
        for b in range(2):
            for layer in range(3):
                assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(shared.gather(layer, b), alone.gather(layer, b)))
        # positions 64 to 95 are still the fork's until the second turn writes there
        assert shared.alloc.shared == {b: 1 for b in shared.blocks[0][:1] + shared.blocks[0][4:6] * (turn == 0)}
        shared.compact()


def test_a_recorded_step_of_a_fork(cuda_device):
    """One token of each of 16 forks of a long prompt, recorded and replayed over new inputs between eager calls: the plan of shared
    attention, its workspace and the prefixes are the graph's own."""
    dev = cuda_device
    inv, _ = ops.rope_frequencies(128, device=dev)
    pool, eager = (KV8Cache(2, 128, batch=16, capacity_tokens=1024, device=dev) for _ in range(2))
    k, v = (_rows((20000, 2, 128), i).to(dev) for i in (1, 2))
    for p in (pool, eager):
        p.write(0, k, v, [20000] + [0] * 15)
        p.fork(0, range(1, 16))
        p.reserve_all(20016)
    q, kn, vn = (torch.zeros((16, n, 128), dtype=torch.bfloat16, device=dev) for n in (12, 2, 2))
    step = lambda p: p.append_attend(0, q, kn, vn, [20000] * 16, counts=[1] * 16, rope=inv)  # noqa: E731
    announce("a recorded step of a fork: warm-up")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(pool)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step(pool)
    for turn in range(4):
        for i, t in enumerate((q, kn, vn)):
            t.copy_(_rows(t.shape, 20 + 3 * turn + i))
        announce(f"a recorded step of a fork: replay {turn}")
        graph.replay()
        want = step(eager)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        _same(pool, eager)
        torch.full((1 << 20,), float("nan"), device=dev)


def test_two_streams_use_a_fork(cuda_device):
    """Steps of the forks on two streams in turn, ordered by events, while the host allocates: pages, tables and prefixes that are
    replaced stay until they have been read."""
    dev = cuda_device
    inv, _ = ops.rope_frequencies(128, device=dev)
    one, two = (KV8Cache(2, 128, batch=4, num_blocks=40, device=dev, seed=3) for _ in range(2))
    k, v = (_rows((300, 2, 128), i).to(dev) for i in (1, 2))
    steps = [[_rows((sum(c), n, 128), 10 * i + n + j).to(dev) for j, n in enumerate((12, 2, 2))] for i, c in
             enumerate([[1] * 4, [5, 3, 1, 9], [16] * 4, [1, 0, 2, 40], [1] * 4])]
    counts = [[1] * 4, [5, 3, 1, 9], [16] * 4, [1, 0, 2, 40], [1] * 4]
    paths = [None, [[0, 2, 4], [1], [0], []], None, [[0], [], [1], list(range(1, 40, 2))], None]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    announce("forks on two streams")
    torch.cuda.synchronize()
    results = []
    for pool in (one, two):
        out = []
        for i, (x, c, p) in enumerate(zip(steps, counts, paths)):
            on, other = (streams[i % 2], streams[1 - i % 2]) if pool is two else (torch.cuda.current_stream(),) * 2
            on.wait_stream(other)
            with torch.cuda.stream(on):
                if pool is two:
                    torch.cuda._sleep(2_000_000)
                if i == 0:
                    pool.write(0, k, v, [300, 0, 0, 0])
                    pool.fork(0, [1, 2, 3])
                starts = list(pool.lengths)
                out.append(pool.append_attend(0, *x, counts=c, rope=inv))
                if p is not None:
                    pool.keep(p, starts)
                if i == 2:
                    pool.compact()
            with torch.cuda.stream(other):
                for n in (3, 9, 64, 4096, 1 << 18):
                    torch.full((n,), 1, dtype=torch.int32, device=dev)
        torch.cuda.synchronize()
        results.append(out)
    for a, b in zip(*results):
        assert torch.equal(a, b)
    _same(one, two)


@pytest.mark.parametrize("heads,fmt", [("target", "int8"), ("draft", "fp8")])
def test_a_long_prompt_is_read_once(cuda_device, heads, fmt):
    """Forks of a prompt for which shared attention is taken, beside a sequence of its own, after a trim into the prompt too."""
    dev = cuda_device
    h, kv, d = HEADS[heads]
    pool = KV8Cache(kv, d, kv_format=fmt, batch=9, num_blocks=420, device=dev, seed=2)
    inv, _ = ops.rope_frequencies(d, device=dev)
    q, k, v = (_rows((5500, n, d), n + i).to(dev) for i, n in enumerate((h, kv, kv)))
    pool.rope_write(0, q, k, v, [500, 5000] + [0] * 7, inv, [0] * 9)
    pool.fork(1, range(2, 9))
    for turn in range(3):
        counts = [[3, 5, 5, 1, 4, 2, 5, 0, 5], [1] * 9, [5] * 9][turn]
        if turn == 2:
            pool.set_length(8, 4700)
        args = [_rows((sum(counts), n, d), 30 * turn + n + i).to(dev) for i, n in enumerate((h, kv, kv))]
        ends = [a + b for a, b in zip(pool.lengths, counts)]
        pos = torch.tensor([a + i for a, n in zip(pool.lengths, counts) for i in range(n)], dtype=torch.int32, device=dev)
        announce(f"a long prompt {heads} {fmt} {turn}")
        got = pool.append_attend(0, *args, counts=counts, rope=inv)
        assert pool.lengths == ends
        cu, prefix, longest = pool._groups(counts, ends)
        assert cu.tolist() == [0, 1, 9] and longest == (4688 if turn == 2 else 4992)
        if turn != 1:
            assert _native.load().sdv_kv8_shared_attention_tile_rows(9, 2, sum(counts), h, kv, d, 5, max(ends), longest) != 0
        want = _exact(pool, 0, ops.rope(args[0], None, pos, inv)[0], counts, None)
        ref.within(got, *want)
