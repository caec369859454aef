"""The ways into the kv8 operators give the same bits: the extension module's plain calls, the general
Python path, and torch.ops.sdv (opcheck, torch.compile)."""
from __future__ import annotations

import pytest
import torch

import kv8_reference as ref
from conftest import announce
from specdec_amd import _native
from specdec_amd.kernels import ops

pytestmark = pytest.mark.gpu


def _case(dev, fmt="fp8", h=12, kv=2, d=128, lens=(90, 333), new=(3, 40), seed=5):
    g = torch.Generator().manual_seed(seed)
    counts = [-(-t // 16) for t in lens]
    bt = ref.table(counts, sum(counts) + 2, seed)
    pages = ref.Pages(sum(counts) + 2, kv, d, fmt)
    for b, t in enumerate(lens):
        pages.write(*ref.slots(bt[b], torch.arange(t)), torch.randn((t, kv, d), generator=g).to(torch.bfloat16),
                    torch.randn((t, kv, d), generator=g).to(torch.bfloat16))
    n = sum(new)
    cu = torch.tensor([0, new[0], n], dtype=torch.int32, device=dev)
    rows = torch.randn((n, h + 2 * kv, d), generator=g).to(torch.bfloat16).to(dev)
    return pages.to(dev), bt.to(dev), cu, torch.tensor(lens, dtype=torch.int32, device=dev), rows, max(new), max(lens), n


@pytest.mark.parametrize("fmt,h,d", [("fp8", 12, 128), ("int8", 14, 64)])
def test_plain_and_general_paths(cuda_device, fmt, h, d):
    dev, kv = cuda_device, 2
    pages, bt, cu, lens, rows, max_new, max_len, n = _case(dev, fmt, h, kv, d)
    b = _native.binding()
    q = rows[:, :h]
    announce(f"kv8 paths {fmt}")
    plain = b.attention(q, *pages, bt, cu, lens, max_new, max_len, None, None)
    assert isinstance(plain, torch.Tensor)
    ws = ops.kv8_workspace(dev, ops.kv8_attention_workspace_bytes(2, n, h, kv, d, max_new, max_len))
    general = ops.kv8_attention(q, *pages, bt, cu, lens, max_new, max_len, workspace_tensor=ws)
    copied = ops.kv8_attention(q.transpose(0, 1).contiguous().transpose(0, 1), *pages, bt, cu, lens, max_new, max_len)
    assert torch.equal(plain, general) and torch.equal(plain, copied)
    assert bool((ws[:_native.KV8_SYNC_BYTES] == 0).all())  # left as it was found
    again = ops.kv8_attention(q, *pages, bt, cu, lens, max_new, max_len, workspace_tensor=ws)
    assert torch.equal(plain, again)
    own = torch.full((ws.numel(),), 0xA5, dtype=torch.uint8, device=dev)  # a caller's buffer, as it comes
    assert torch.equal(plain, ops.kv8_attention(q, *pages, bt, cu, lens, max_new, max_len, workspace_tensor=own))
    got = b.gather(*pages, bt, cu, lens - torch.tensor([3, 40], dtype=torch.int32, device=dev), n)
    k_out = torch.empty((n, kv, d), dtype=torch.bfloat16, device=dev)
    want = ops.kv8_gather(*pages, bt, cu, lens - torch.tensor([3, 40], dtype=torch.int32, device=dev), n, k_out=k_out)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and want[0] is k_out
    one, two = [t.clone() for t in pages], [t.clone() for t in pages]
    k, v = rows[:, h:h + kv], rows[:, h + kv:]
    assert b.append(k, v, *one, bt, cu, lens, 0) == 0
    ops.kv8_append(k.transpose(0, 1).contiguous().transpose(0, 1), v, *two, bt, cu, lens)
    for x, y in zip(one, two):
        assert torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))
    # what the extension module does not take
    for bad in (dict(q=q.float()), dict(q=q.transpose(0, 1)), dict(q=q[:0]), dict(cu=cu.long()), dict(bt=bt.t()), dict(m=float(max_new)),
                dict(m=True), dict(s=1)):
        assert b.attention(bad.get("q", q), *pages, bad.get("bt", bt), bad.get("cu", cu), lens, bad.get("m", max_new), max_len,
                           bad.get("s"), None) is None, bad
    assert b.append(k, v, *one, bt, cu, None, 0) is None and b.gather(*pages, bt, cu, lens, 0) is None


def test_whole_numbers_of_other_types(cuda_device):
    """NumPy-like whole numbers and integer scales take the general path."""
    pages, bt, cu, lens, rows, max_new, max_len, n = _case(cuda_device)
    a = ops.kv8_attention(rows[:, :12], *pages, bt, cu, lens, max_new, max_len, scale=1.0)
    b = ops.kv8_attention(rows[:, :12], *pages, bt, cu, lens, torch.tensor(max_new), float(max_len), scale=1)
    assert torch.equal(a, b)


def test_opcheck(cuda_device):
    pages, bt, cu, lens, rows, max_new, max_len, n = _case(cuda_device, "int8")
    announce("opcheck sdv::kv8_*")
    torch.library.opcheck(torch.ops.sdv.kv8_attention.default, (rows[:, :12].contiguous(), *pages, bt, cu, lens, max_new, max_len))
    torch.library.opcheck(torch.ops.sdv.kv8_gather.default, (*pages, bt, cu, torch.zeros_like(lens), n))
    torch.library.opcheck(torch.ops.sdv.kv8_append.default, (rows[:, 12:14].contiguous(), rows[:, 14:].contiguous(), *pages, bt, cu, lens))


def test_compiled(cuda_device):
    pages, bt, cu, lens, rows, max_new, max_len, n = _case(cuda_device, "fp8")
    q = rows[:, :12].contiguous()

    def step(q, k, v, s, bt, cu, lens):
        return torch.ops.sdv.kv8_attention(q, k, v, s, bt, cu, lens, max_new, max_len) * 2

    announce("torch.compile of sdv::kv8_attention")
    want = step(q, *pages, bt, cu, lens)
    got = torch.compile(step, fullgraph=True, backend="aot_eager")(q, *pages, bt, cu, lens)
    assert torch.equal(got, want)
