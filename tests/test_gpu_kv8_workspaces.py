"""Where kv8 attention's workspaces come from: calls of several threads, recordings, private memory pools."""
from __future__ import annotations

import subprocess
import sys
import threading

import pytest
import torch

from conftest import ROOT, announce
from specdec_amd.kernels import ops
from test_gpu_kv8 import HEADS, _cu, _filled, _gen, _ints

pytestmark = pytest.mark.gpu


def _call(dev, new, lens, length, seed, fmt="fp8"):
    """(arguments of ops.kv8_attention, its result)."""
    h, kv, d = HEADS["target"]
    pages, bt = _filled(kv, d, fmt, lens, seed)
    q = torch.randn((sum(new), h, d), generator=_gen(seed)).to(torch.bfloat16).to(dev)
    args = (q, *pages.to(dev), bt.to(dev), _cu(new, dev), _ints(lens, dev), max(new), length)
    want = ops.kv8_attention(*args)
    torch.cuda.synchronize()
    return args, want


def _same(a, b):
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize("general", [False, True])
def test_threads_on_one_stream(cuda_device, general):
    """Host threads that call on one stream at once, with outputs of their own: many rows (two launches a call) of
    different counts, and few.  `general`: a scale that is a whole number takes the general Python path."""
    dev = cuda_device
    scale = 1 if general else 1.0
    cases = [_call(dev, new, lens, 131072, i)[0] for i, (new, lens) in enumerate((([300], [2000]), ([40, 3], [900, 60]), ([120], [5000])))]
    cases.append(_call(dev, [5, 1], [3000, 200], 3000, 7)[0])
    wants = [ops.kv8_attention(*c, scale=1.0) for c in cases]
    turns = 40
    outs = [[torch.zeros_like(w) for _ in range(turns)] for w in wants]
    torch.cuda.synchronize()
    start, wrong = threading.Barrier(len(cases)), []

    def work(i):
        try:
            start.wait(30)
            for o in outs[i]:
                if ops.kv8_attention(*cases[i], scale=scale, out=o) is not o:
                    wrong.append(i)
        except Exception as e:  # noqa: BLE001  (shown by the test's thread)
            wrong.append(e)

    announce(f"kv8 attention from {len(cases)} threads, general {general}")
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    torch.cuda.synchronize()
    assert not wrong, wrong
    for got, want in zip(outs, wants):
        assert all(_same(o, want) for o in got)


def _live_blocks(pool_id):
    """(address, size) of the allocated blocks in the segments of a private pool."""
    return [(b["address"], b["size"]) for s in torch.cuda.memory_snapshot() if tuple(s["segment_pool_id"]) == tuple(pool_id)
            for b in s["blocks"] if b["state"] != "inactive"]


CASES = [([1, 1], [3000, 2500], 3000), ([40, 3], [900, 2000], 131072), ([5, 5], [4000, 70], 4000)]


def test_a_recording_keeps_no_memory_but_its_outputs(cuda_device):
    """What a graph's calls allocate beside their outputs is free again in its pool when they return, on the
    recording stream and on a forked one; replays still give the same bits."""
    cases = [_call(cuda_device, *c, seed=i) for i, c in enumerate(CASES)]
    graph, main, fork = torch.cuda.CUDAGraph(), torch.cuda.Stream(), torch.cuda.Stream()
    own = [torch.zeros_like(want) for _, want in cases]  # outputs of the caller's
    with torch.cuda.graph(graph, stream=main):
        outs = [ops.kv8_attention(*a) for a, _ in cases]
        assert all(ops.kv8_attention(*a, out=o) is o for (a, _), o in zip(cases, own))
        fork.wait_stream(main)
        with torch.cuda.stream(fork):
            outs += [ops.kv8_attention(*a) for a, _ in cases]
        main.wait_stream(fork)
    assert {a for a, _ in _live_blocks(graph.pool())} == {o.data_ptr() for o in outs}
    for turn in range(3):
        announce(f"kv8 attention, a graph's replay {turn}")
        for o in outs + own:
            o.zero_()
        graph.replay()
        eager = [ops.kv8_attention(*a) for a, _ in cases]
        torch.cuda.synchronize()
        for i, o in enumerate(outs + own + eager):
            assert _same(o, cases[i % len(cases)][1])


def test_an_eager_call_keeps_nothing_of_a_private_pool(cuda_device):
    cases = [_call(cuda_device, *c, seed=i) for i, c in enumerate(CASES)]
    pool, stream = torch.cuda.MemPool(), torch.cuda.Stream()  # a stream of its own: its first call
    announce("kv8 attention in a private pool")
    with torch.cuda.stream(stream), torch.cuda.use_mem_pool(pool):
        outs = [ops.kv8_attention(*a) for a, _ in cases]
    stream.synchronize()
    assert all(_same(o, want) for o, (_, want) in zip(outs, cases))
    assert {a for a, _ in _live_blocks(pool.id)} == {o.data_ptr() for o in outs}
    del outs
    assert _live_blocks(pool.id) == []


@pytest.mark.parametrize("how", [dict(backend="cudagraphs"), dict(mode="reduce-overhead")])
def test_compiled_into_graphs(cuda_device, how):
    """torch.compile's own graphs, which warm up in their pool and check what is left there."""
    cases = [_call(cuda_device, *c, seed=i) for i, c in enumerate(CASES)]
    for args, want in cases:
        most_q, most_len = args[-2:]

        def step(*a):
            return torch.ops.sdv.kv8_attention(*a, most_q, most_len) * 2

        torch._dynamo.reset()
        compiled = torch.compile(step, **how)
        for turn in range(4):  # eager, warm-up, recording, replay
            announce(f"torch.compile of sdv::kv8_attention {how} {most_q}, call {turn}")
            torch.compiler.cudagraph_mark_step_begin()
            got = compiled(*args[:-2]).clone()
            torch.cuda.synchronize()
            assert _same(got, want * 2)


_MANY = """
import sys
sys.path[:0] = {path!r}
import torch
from test_gpu_kv8_workspaces import CASES, _call, _same
dev = torch.device("cuda", 0)
args, want = _call(dev, *CASES[2], seed=1)
from specdec_amd.kernels import ops
stream, kept, at = torch.cuda.Stream(), [], {at!r}
pool = torch.cuda.graph_pool_handle()
for i in range(max(at) + 1):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, pool=pool):
        out = ops.kv8_attention(*args)
    if i in at:
        kept.append((graph, out))
    if i % 500 == 0:
        print("recorded", i, flush=True)
sides = [torch.cuda.Stream() for _ in kept]
for turn in range(3):
    for _, o in kept:
        o.zero_()
    torch.cuda.synchronize()
    for st, (graph, _) in zip(sides, kept):
        with torch.cuda.stream(st):
            graph.replay()
    torch.cuda.synchronize()
    assert all(_same(o, want) for _, o in kept), turn
    assert _same(ops.kv8_attention(*args), want)
print("as ever", flush=True)
"""


def test_more_recordings_than_slots(cuda_device):
    """More recordings than the library has slots of counts, in a process of their own: the last ones zero
    their workspace's instead."""
    root = str(ROOT)
    path = [root, f"{root}/specdec-context-scaling_amd", f"{root}/tests"]
    announce("kv8 attention, 2000 recordings")
    got = subprocess.run([sys.executable, "-u", "-c", _MANY.format(path=path, at=[0, 1, 1791, 1792, 1999])], capture_output=True, text=True, timeout=100)
    assert got.returncode == 0 and got.stdout.endswith("as ever\n"), got.stdout + got.stderr
