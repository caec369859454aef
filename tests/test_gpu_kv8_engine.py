"""The 8-bit cache inside the engine: the pool's calls, recorded steps, the kv8 pack."""
from __future__ import annotations

import pytest
import torch

import kv8_reference as ref
from conftest import announce
from oracle import engine as oeng
from specdec_amd import SdvError
from specdec_amd.engine import spec_cache as sc
from specdec_amd.engine.kv8_cache import KV8Cache
from specdec_amd.engine.paged_cache import PagedKVCache
from specdec_amd.kernels import ops, patch

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rows(shape, seed):
    return torch.randn(shape, generator=_gen(seed)).to(torch.bfloat16)


def _mirror(pool):
    """CPU pages over the same block table."""
    n = pool.k_pages.shape[1]
    return ref.Pages(n, pool.kv_heads, pool.head_dim, pool.kv_format)


def _write(pages, pool, starts, counts, k, v):
    at = 0
    bt = pool.block_table().cpu()
    for b, (s, c) in enumerate(zip(starts, counts)):
        if c:
            pages.write(*ref.slots(bt[b], torch.arange(s, s + c)), k[at:at + c], v[at:at + c])
        at += c


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_pool_calls(cuda_device, fmt):
    """Prompts, a step that mixes a chunk, a verify block and a single token, a uniform step, a tree,
    a trim, and everything read back."""
    dev = cuda_device
    h, kv, d = 12, 2, 128
    pool = KV8Cache(kv, d, kv_format=fmt, num_layers=2, batch=3, num_blocks=60, device=dev, seed=4)
    pages = _mirror(pool)
    announce(f"kv8 pool prefill {fmt}")
    lengths = [70, 5, 200]
    k, v = _rows((275, kv, d), 1), _rows((275, kv, d), 2)
    pool.prefill(1, k.to(dev), v.to(dev), lengths)
    _write(pages, pool, [0, 0, 0], lengths, k, v)
    assert pool.lengths == lengths
    counts = [40, 5, 1]
    announce(f"kv8 pool mixed step {fmt}")
    k, v, q = _rows((46, kv, d), 3), _rows((46, kv, d), 4), _rows((46, h, d), 5)
    got = pool.append_attend(1, q.to(dev), k.to(dev), v.to(dev), counts=counts)
    _write(pages, pool, lengths, counts, k, v)
    lengths = [n + c for n, c in zip(lengths, counts)]
    assert pool.lengths == lengths
    want, bound = ref.attention(q, pages, pool.block_table().cpu(), counts, lengths)
    ref.within(got, want, bound)
    announce(f"kv8 pool uniform step {fmt}")
    starts = [100, 10, 201]  # the first sequence trimmed
    k, v, q = _rows((3, 4, kv, d), 6), _rows((3, 4, kv, d), 7), _rows((3, h, 4, d), 8)
    got = pool.append_attend(1, q.to(dev), k.to(dev), v.to(dev), starts)
    _write(pages, pool, starts, [4] * 3, k.reshape(12, kv, d), v.reshape(12, kv, d))
    lengths = [s + 4 for s in starts]
    flat = q.transpose(1, 2).reshape(12, h, d)
    want, bound = ref.attention(flat, pages, pool.block_table().cpu(), [4] * 3, lengths)
    ref.within(got.transpose(1, 2).reshape(12, h, d), want, bound)
    major = pool.attend(1, q.transpose(1, 2).contiguous().to(dev), q_token_major=True)
    out = torch.empty_like(got)
    assert pool.attend(1, q.to(dev), out=out) is out and torch.equal(out, got)
    assert torch.equal(major.transpose(1, 2), got)
    announce(f"kv8 pool tree {fmt}")
    tree = torch.tensor([1, 3, 5, 11], dtype=torch.int64).repeat(3)
    got = pool.attend(1, flat.to(dev), counts=[4] * 3, tree_mask=tree.to(dev), scale=0.2)
    want, bound = ref.attention(flat, pages, pool.block_table().cpu(), [4] * 3, lengths, 0.2, tree)
    ref.within(got, want, bound)
    bt = pool.block_table().cpu()
    k, v = pool.read(1, lengths)
    rows = [pages.read(*ref.slots(bt[b], torch.arange(n))) for b, n in enumerate(lengths)]
    assert torch.equal(k.cpu(), torch.cat([r[0] for r in rows]).to(torch.bfloat16))
    assert torch.equal(v.cpu(), torch.cat([r[1] for r in rows]).to(torch.bfloat16))
    k, v = pool.gather(1, 2, 50)
    assert torch.equal(v.cpu(), rows[2][1][:50].transpose(0, 1).to(torch.bfloat16))
    assert bool((pool.k_pages.view(torch.uint8)[0] == 0).all())  # the other layer


def test_recorded_steps(cuda_device):
    """A decode and a verify step recorded into graphs and replayed in turn, lengths equal; what a
    recording cannot do raises."""
    dev = cuda_device
    h, kv, d = 14, 2, 64
    pool = KV8Cache(kv, d, batch=2, capacity_tokens=200, device=dev, seed=2)
    k, v = _rows((200, kv, d), 1).to(dev), _rows((200, kv, d), 2).to(dev)
    pool.prefill(0, k, v, [100, 100])
    pool.reserve_all(120)
    steps = []
    for s in (1, 5):
        steps.append((_rows((2, s, h, d), 10 + s).to(dev), _rows((2, s, kv, d), 20 + s).to(dev), _rows((2, s, kv, d), 30 + s).to(dev)))

    def run(i):
        return pool.append_attend(0, *steps[i], [100, 100], q_token_major=True)

    graphs = []
    side = torch.cuda.Stream()
    for i in range(2):
        want = run(i)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = run(i)
        graphs.append((graph, out, want))
    with pytest.raises(SdvError):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            pool.append_attend(0, *(x[:, :3] for x in steps[1]), [100, 100], q_token_major=True)  # no row table of it yet
    for turn in range(3):
        for i, (graph, out, want) in enumerate(graphs):
            announce(f"kv8 recorded step {i}, replay {turn}")
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
            pool.attend(0, steps[0][0], q_token_major=True, lengths=[100, 100])


def test_pool_on_two_streams(cuda_device):
    """Calls of different counts on two streams, ordered by events: each stream's tables are its own."""
    dev = cuda_device
    h, kv, d = 12, 2, 128
    pool = KV8Cache(kv, d, batch=2, capacity_tokens=400, device=dev, seed=3)
    pages = _mirror(pool)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    lengths, outs = [0, 0], []
    announce("kv8 pool on two streams")
    for turn, counts in enumerate([[120, 60], [1, 5], [40, 1], [1, 5], [3, 3]]):
        st = streams[turn % 2]
        st.wait_stream(streams[1 - turn % 2])
        st.wait_stream(torch.cuda.current_stream())
        n = sum(counts)
        k, v, q = _rows((n, kv, d), 40 + turn), _rows((n, kv, d), 50 + turn), _rows((n, h, d), 60 + turn)
        dk, dv, dq = k.to(dev), v.to(dev), q.to(dev)
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            got = pool.append_attend(0, dq, dk, dv, counts=counts)
        torch.cuda.synchronize()
        _write(pages, pool, lengths, counts, k, v)
        lengths = [a + c for a, c in zip(lengths, counts)]
        want, bound = ref.attention(q, pages, pool.block_table().cpu(), counts, lengths)
        ref.within(got, want, bound)


# ------------------------------------------------------------------------------ the pack
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_pack_layer(cuda_device, fmt):
    """One attention layer under the pack (its output projection the identity, which BF16 carries
    exactly) through prefill, decode, verify, a trim, a repair step: the operator's bound on every
    call, and the bytes that are read back."""
    dev = cuda_device
    H, KV, D = 12, 2, 128
    layer = oeng.SelfAttention(H * D, H, KV, D).to(torch.bfloat16)
    g = _gen(31)
    with torch.no_grad():
        for proj in (layer.q_proj, layer.k_proj, layer.v_proj):
            proj.weight.copy_(torch.randn(proj.weight.shape, generator=g) / 40)
        layer.o_proj.weight.copy_(torch.eye(H * D))
    layer = layer.to(dev)
    layer.kv_format = "v_fp8"
    patch.install("kv8", oeng, kv_format=fmt, capacity_tokens=48, seed=7)
    try:
        cache, keys, values, t0 = None, [], [], 0
        for step, s in enumerate((77, 1, 5, 1, 1)):
            if step == 3:  # two of the five verified tokens stay
                cache, t0 = sc.trim_cache([cache], t0 - 3)[0], t0 - 3
            x = _rows((1, s, H * D), 70 + step).to(dev)
            cos, sin = oeng.Build_Rope_cache(D, s, 1e6, dev, torch.bfloat16, t0)
            announce(f"kv8 pack layer {fmt}, call {step}")
            with torch.inference_mode():
                got, cache = layer(x, cos, sin, cache)
                q = oeng.apply_rope(layer.q_proj(x).view(1, s, H, D).transpose(1, 2), cos, sin)
                k = oeng.apply_rope(layer.k_proj(x).view(1, s, KV, D).transpose(1, 2), cos, sin)
                v = layer.v_proj(x).view(1, s, KV, D)
            keys = torch.cat([keys[:t0], k[0].transpose(0, 1).cpu()]) if step else k[0].transpose(0, 1).cpu()
            values = torch.cat([values[:t0], v[0].cpu()]) if step else v[0].cpu()
            t0 += s
            bt = ref.table([-(-t0 // 16)], 8)
            pages = ref.Pages(8, KV, D, fmt)
            pages.write(*ref.slots(bt[0], torch.arange(t0)), keys, values)
            want, bound = ref.attention(q[0].transpose(0, 1).cpu(), pages, bt, [s], [t0])
            ref.within(got[0].view(s, H, D), want, bound)
        assert sc.cache_length([cache]) == t0 == 77 + 1 + 2 + 1 + 1
        full = cache["pages"].materialize(t0)
        k, v = pages.read(*ref.slots(bt[0], torch.arange(t0)))
        assert torch.equal(full["k"][0].cpu(), k.transpose(0, 1).to(torch.bfloat16))
        assert torch.equal(full["v"][0].cpu(), v.transpose(0, 1).to(torch.bfloat16))
        patch.install("fp8v", oeng)
        with pytest.raises(SdvError, match="another pack"):
            layer(x, cos, sin, cache)
    finally:
        patch.restore()


def test_pack_speculative_decoding(cuda_device):
    """The SpecDec loop with target and draft on the kv8 pack: the draft has the target's weights, so
    most proposals are accepted."""
    announce("kv8 pack speculative decoding")
    target = oeng.tiny_model(11, device=cuda_device)
    draft = oeng.tiny_model(11, device=cuda_device)
    prompt = torch.randint(0, 512, (1, 60), generator=_gen(5))
    patch.install("kv8", oeng, kv_format="int8", capacity_tokens=48, seed=9)
    try:
        got = oeng.spec_decode_greedy(target, draft, prompt, 40, k=4, target_kv="v_fp8", draft_kv="v_fp8")
    finally:
        patch.restore()
    st = got["stats"]
    assert all(isinstance(layer["pages"].pool, KV8Cache) for layer in got["target_cache"])
    assert len(got["gen"]) >= 40 and st["accepted"] >= st["proposed"] // 2


def test_other_caches_are_as_they_were(cuda_device):
    """The v_fp8 pool beside a kv8 pool on one device and stream: neither's workspace is the other's."""
    dev = cuda_device
    h, kv, d = 12, 2, 128
    old, new = PagedKVCache(kv, d, capacity_tokens=600, device=dev, seed=1), KV8Cache(kv, d, capacity_tokens=600, device=dev, seed=1)
    k, v, q = _rows((1, 500, kv, d), 1).to(dev), _rows((1, 500, kv, d), 2).to(dev), _rows((1, h, 1, d), 3).to(dev)
    old.append(0, k, v)
    first = old.attend(0, q)
    new.append(0, k, v)
    a = new.attend(0, q)
    announce("v_fp8 and kv8 calls in turn")
    for _ in range(3):
        assert torch.equal(old.attend(0, q), first) and torch.equal(new.attend(0, q), a)
    assert ops.workspace_status(ops.workspace(dev, 1)) == (0, False)
    rel = float((a.float() - first.float()).norm() / first.float().norm())
    assert rel < 0.05  # both near the BF16 result: K in E4M3FN moves scores by some 2% of their size
