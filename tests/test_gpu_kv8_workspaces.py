"""Where kv8 attention's workspaces come from: calls of several threads, recordings, private memory pools."""
from __future__ import annotations

import threading

import pytest
import torch

from conftest import announce
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
