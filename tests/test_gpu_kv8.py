"""The 8-bit KV cache on the GPU against plain torch in 64 bits (tests/kv8_reference.py)."""
from __future__ import annotations

import math

import pytest
import torch

import kv8_reference as ref
from conftest import announce
from specdec_amd._native import SdvError
from specdec_amd.kernels import ops

pytestmark = pytest.mark.gpu
HEADS = {"target": (12, 2, 128), "draft": (14, 2, 64), "mha": (4, 4, 128), "mqa": (20, 1, 64)}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rows(shape, g, outliers=8.0):
    x = torch.randn(shape, generator=g)
    x[..., 3] *= outliers
    return x.to(torch.bfloat16)


def _ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _cu(new, dev):
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return _ints(cu, dev)


def _filled(kv, d, fmt, lens, seed, spare=3):
    """(pages, table) whose sequences hold random tokens."""
    g = _gen(seed)
    counts = [-(-max(t, 0) // 16) for t in lens]
    nb = sum(counts) + spare
    bt = ref.table(counts, nb, seed)
    pages = ref.Pages(nb, kv, d, fmt)
    for b, t in enumerate(lens):
        if t > 0:
            pages.write(*ref.slots(bt[b], torch.arange(t)), _rows((t, kv, d), g), _rows((t, kv, d), g, 20.0))
    return pages, bt


def _attend(dev, heads, fmt, lens, new, seed=1, tree=None, scale=None, pages=None, bt=None, extra=0, **kw):
    h, kv, d = heads
    if pages is None:
        pages, bt = _filled(kv, d, fmt, lens, seed)
    total = sum(new)
    q = torch.randn((total + extra, h, d), generator=_gen(seed + 7)).to(torch.bfloat16)
    got = ops.kv8_attention(q.to(dev), *pages.to(dev), bt.to(dev), _cu(new, dev), _ints(lens, dev), max(max(new), 1),
                            max(max(lens), 1), scale=scale, tree_mask=None if tree is None else tree.to(dev), **kw)
    torch.cuda.synchronize()
    want, bound = ref.attention(q[:total], pages, bt, new, lens, scale, tree)
    return got, want, bound


# ------------------------------------------------------------------------------ write
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("heads", ["target", "draft", "mha"])
@pytest.mark.parametrize("new,lens", [
    ([1], [1]), ([1], [17]), ([16], [16]), ([16], [32]), ([15], [47]), ([33], [50]), ([300], [1000]),
    ([1, 1, 1, 1], [5, 16, 17, 333]), ([0, 3, 0, 20, 1], [9, 3, 0, 25, 40]), ([100, 2, 77], [100, 50, 90])])
def test_append(cuda_device, fmt, heads, new, lens):
    announce(f"kv8 append {fmt} {heads} {new} {lens}")
    dev = cuda_device
    _, kv, d = HEADS[heads]
    pages, bt = _filled(kv, d, fmt, [t - n for t, n in zip(lens, new)], 3)
    counts = [-(-t // 16) for t in lens]
    nb = sum(counts) + 5
    bt = ref.table(counts, nb, 11)
    pages = ref.Pages(nb, kv, d, fmt)
    g = _gen(sum(new))
    total = sum(new)
    k, v = _rows((total + 2, kv, d), g), _rows((total + 2, kv, d), g)  # two rows behind the last sequence
    if total > 4:
        k[1], v[2, 0], v[3] = 0.0, 0.0, 1e-30  # rows of zeros, and one below the fast route's range
        v[4, :, 0] = 2.0 ** -133               # the smallest BF16
    kp, vp, sc = pages.to(dev)
    ops.kv8_append(k.to(dev), v.to(dev), kp, vp, sc, bt.to(dev), _cu(new, dev), _ints(lens, dev))
    torch.cuda.synchronize()
    at = 0
    for b, (n, t) in enumerate(zip(new, lens)):
        if n:
            pages.write(*ref.slots(bt[b], torch.arange(t - n, t)), k[at:at + n], v[at:at + n])
        at += n
    assert torch.equal(kp.view(torch.uint8).cpu(), pages.k)
    assert torch.equal(vp.view(torch.uint8).cpu(), pages.v)
    assert torch.equal(sc.view(torch.int32).cpu()[~torch.isnan(pages.s)], pages.s.view(torch.int32)[~torch.isnan(pages.s)])
    assert torch.equal(torch.isnan(sc).cpu(), torch.isnan(pages.s))


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_append_rows_that_are_not_finite(cuda_device, fmt):
    """Scale NaN and codes 0 for a row with an infinity or a NaN; its neighbours as ever."""
    dev = cuda_device
    pages, bt = ref.Pages(2, 2, 128, fmt), ref.table([2], 2)
    k, v = _rows((20, 2, 128), _gen(1)), _rows((20, 2, 128), _gen(2))
    k[3, 1, 7], k[4, 0, 0], v[3, 0, 127], v[17, 1, 64] = math.inf, math.nan, -math.inf, math.nan
    kp, vp, sc = pages.to(dev)
    announce(f"kv8 append of rows that are not finite {fmt}")
    ops.kv8_append(k.to(dev), v.to(dev), kp, vp, sc, bt.to(dev), _cu([20], dev), _ints([20], dev))
    torch.cuda.synchronize()
    pages.write(*ref.slots(bt[0], torch.arange(20)), k, v)
    assert torch.equal(kp.view(torch.uint8).cpu(), pages.k) and torch.equal(vp.view(torch.uint8).cpu(), pages.v)
    assert torch.equal(torch.isnan(sc).cpu(), torch.isnan(pages.s))


def test_append_takes_projection_parts_and_skips_what_has_no_slot(cuda_device):
    """k and v as parts of one (rows, H + 2 KV, D) tensor; lengths below the row count, blocks that
    the table does not name, and lengths given as one number."""
    dev = cuda_device
    h, kv, d = HEADS["target"]
    qkv = _rows((40, h + 2 * kv, d), _gen(5))
    k, v = qkv[:, h:h + kv], qkv[:, h + kv:]
    new, lens = [10, 20, 10], [4, 60, 30]  # the first has six rows before position 0
    bt = ref.table([1, 4, 2], 9)
    bt[1, 3] = 9    # behind the pool
    bt[2, 1] = -1
    pages = ref.Pages(9, kv, d, "fp8")
    kp, vp, sc = pages.to(dev)
    announce("kv8 append of projection parts")
    dq = qkv.to(dev)
    ops.kv8_append(dq[:, h:h + kv], dq[:, h + kv:], kp, vp, sc, bt.to(dev), _cu(new, dev), _ints(lens, dev))
    torch.cuda.synchronize()
    pages.write(*ref.slots(bt[0], torch.arange(0, 4)), k[6:10], v[6:10])
    pages.write(*ref.slots(bt[1], torch.arange(40, 48)), k[10:18], v[10:18])
    # sequence 2: positions 20..29 lie in block 1, which the table does not name
    assert torch.equal(kp.view(torch.uint8).cpu(), pages.k) and torch.equal(vp.view(torch.uint8).cpu(), pages.v)
    kp2, vp2, sc2 = ref.Pages(9, kv, d, "fp8").to(dev)
    ops.kv8_append(dq[:10, h:h + kv], dq[:10, h + kv:], kp2, vp2, sc2, bt[:1].to(dev), _cu([10], dev), None, 4)
    torch.cuda.synchronize()
    one = ref.Pages(9, kv, d, "fp8")
    one.write(*ref.slots(bt[0], torch.arange(0, 4)), k[6:10], v[6:10])
    assert torch.equal(kp2.view(torch.uint8).cpu(), one.k)


# ------------------------------------------------------------------------------ read-back
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("heads", ["target", "draft"])
@pytest.mark.parametrize("starts,counts", [([0], [1]), ([5], [40]), ([16], [16]), ([0, 100, 7], [300, 0, 33])])
def test_gather(cuda_device, fmt, heads, starts, counts):
    """bf16(code * scale), one fp32 product and one rounding: equal to the bit."""
    dev = cuda_device
    _, kv, d = HEADS[heads]
    pages, bt = _filled(kv, d, fmt, [s + n for s, n in zip(starts, counts)], 4)
    total = sum(counts)
    announce(f"kv8 gather {fmt} {heads} {starts} {counts}")
    wide = torch.full((total + 2, 3 * kv, d), 7.0, dtype=torch.bfloat16, device=dev)
    k, v = ops.kv8_gather(*pages.to(dev), bt.to(dev), _cu(counts, dev), _ints(starts, dev), total + 2, k_out=wide[:, :kv],
                          v_out=wide[:, 2 * kv:])
    plain = ops.kv8_gather(*pages.to(dev), bt.to(dev), _cu(counts, dev), _ints(starts, dev), total)
    torch.cuda.synchronize()
    rows = [pages.read(*ref.slots(bt[b], torch.arange(s, s + n))) for b, (s, n) in enumerate(zip(starts, counts)) if n]
    for got, alone, want in ((k, plain[0], torch.cat([r[0] for r in rows])), (v, plain[1], torch.cat([r[1] for r in rows]))):
        want = want.to(torch.bfloat16)
        assert torch.equal(got[:total].cpu().view(torch.int16), want.view(torch.int16))
        assert torch.equal(alone.cpu().view(torch.int16), want.view(torch.int16))
    assert bool((wide[total:] == 7.0).all()) and bool((wide[:, kv:2 * kv] == 7.0).all())


def test_gather_positions_in_no_block(cuda_device):
    dev = cuda_device
    pages, bt = _filled(2, 128, "int8", [40], 6)
    bt = bt.clone()
    bt[0, 1] = pages.s.shape[0]
    announce("kv8 gather of positions in no block")
    k, v = ops.kv8_gather(*pages.to(dev), bt.to(dev), _cu([60], dev), _ints([-4], dev), 60)
    torch.cuda.synchronize()
    want = torch.zeros((60, 2, 128))
    for lo, hi in ((0, 16), (32, 40)):
        want[lo + 4:hi + 4] = pages.read(*ref.slots(bt[0], torch.arange(lo, hi)))[1]
    # positions 40..47 lie in the last block but were never written: whatever is there
    keep = [i for i in range(60) if not 44 <= i < 52]
    assert torch.equal(v.cpu()[keep].view(torch.int16), want.to(torch.bfloat16)[keep].view(torch.int16))
    assert bool((k.cpu()[:4] == 0).all()) and bool((k.cpu()[20:36] == 0).all()) and bool((k.cpu()[52:] == 0).all())


# ------------------------------------------------------------------------------ attention
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("heads", list(HEADS))
@pytest.mark.parametrize("new,lens", [
    ([1], [1]), ([1], [16]), ([1], [17]), ([1], [64]), ([1], [65]), ([1], [2047]), ([2], [2]), ([5], [5]), ([5], [700]),
    ([5], [1025]), ([1] * 6, [1, 15, 130, 64, 999, 33]), ([1, 5, 0, 3], [40, 5, 12, 513]), ([40], [40]), ([70], [333]),
    ([130, 1, 1], [130, 300, 65])])
def test_attention(cuda_device, fmt, heads, new, lens):
    announce(f"kv8 attention {fmt} {heads} {new} {lens}")
    got, want, bound = _attend(cuda_device, HEADS[heads], fmt, lens, new)
    ref.within(got, want, bound)


@pytest.mark.parametrize("heads,new,lens", [("target", [1], [20011]), ("draft", [300], [5000]), ("target", [257], [4097])])
def test_attention_long(cuda_device, heads, new, lens):
    announce(f"kv8 attention {heads} {new} {lens}")
    got, want, bound = _attend(cuda_device, HEADS[heads], "fp8", lens, new)
    ref.within(got, want, bound)


def test_attention_many_sequences(cuda_device):
    """More sequences than a workgroup has threads, some without rows."""
    new = [(i * 7) % 4 for i in range(600)]
    lens = [n + (i * 13) % 90 for i, n in enumerate(new)]
    announce("kv8 attention of 600 sequences")
    got, want, bound = _attend(cuda_device, (4, 2, 64), "int8", lens, new)
    ref.within(got, want, bound)


@pytest.mark.parametrize("new,lens", [([3, 10, 1], [2, 4, 0]), ([64], [10]), ([1, 2], [0, 0])])
def test_attention_rows_that_see_nothing(cuda_device, new, lens):
    """A length below the row count: the rows before position 0 see nothing and are 0."""
    announce(f"kv8 attention of rows before position 0 {new} {lens}")
    got, want, bound = _attend(cuda_device, HEADS["target"], "fp8", lens, new)
    ref.within(got, want, bound)
    assert bool((want[0] == 0).all())


def _random_tree(new, seed):
    g = _gen(seed)
    words = []
    for n in new:
        own = []
        for i in range(n):
            parent = int(torch.randint(-1, i, (1,), generator=g)) if i else -1
            own.append((own[parent] if parent >= 0 else 0) | 1 << i)
        words += [w - (1 << 64) if w >> 63 else w for w in own]
    return torch.tensor(words, dtype=torch.int64)


@pytest.mark.parametrize("heads", ["target", "draft"])
@pytest.mark.parametrize("new,lens", [([1], [1]), ([7], [7]), ([24], [500]), ([64], [64]), ([64, 3, 20], [1000, 70, 33])])
def test_attention_tree(cuda_device, heads, new, lens):
    tree = _random_tree(new, sum(new))
    announce(f"kv8 attention tree {heads} {new} {lens}")
    got, want, bound = _attend(cuda_device, HEADS[heads], "fp8", lens, new, tree=tree)
    ref.within(got, want, bound)


def test_attention_tree_masks_of_any_bits(cuda_device):
    """A chain's mask gives the causal result; a mask of nothing without a context gives 0."""
    dev, heads = cuda_device, HEADS["target"]
    new, lens = [9, 4], [120, 4]
    chain = torch.tensor([(2 << i) - 1 for n in new for i in range(n)], dtype=torch.int64)
    announce("kv8 attention tree of a chain")
    a, want, bound = _attend(dev, heads, "int8", lens, new, tree=chain)
    b, _, _ = _attend(dev, heads, "int8", lens, new)
    ref.within(a, want, bound)
    ref.within(b, want, bound)
    none = chain.clone()
    none[9:] = 0
    got, want, bound = _attend(dev, heads, "int8", lens, new, tree=none)
    ref.within(got, want, bound)
    assert bool((got[9:] == 0).all())


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("new", [1, 5, 40])
def test_attention_nan_and_masks(cuda_device, fmt, new):
    """Tokens that hold an infinity or a NaN reach the rows that see them and no others."""
    dev = cuda_device
    h, kv, d = HEADS["target"]
    T = 150 + new
    g = _gen(21)
    bt = ref.table([-(-T // 16)], 14)
    pages = ref.Pages(14, kv, d, fmt)
    k, v = _rows((T, kv, d), g), _rows((T, kv, d), g)
    if new > 2:
        k[T - 2, 0, 5], v[T - 3, 1, 9] = math.inf, math.nan  # new tokens: later rows alone see them
    else:
        v[77, 1, 9] = -math.inf
    pages.write(*ref.slots(bt[0], torch.arange(T)), k, v)
    announce(f"kv8 attention over tokens that are not finite {fmt} {new}")
    got, want, bound = _attend(dev, (h, kv, d), fmt, [T], [new], pages=pages, bt=bt)
    assert bool(torch.isnan(want).any()) and bool(torch.isfinite(want).any())
    ref.within(got, want, bound)


@pytest.mark.parametrize("new", [1, 30])
def test_attention_blocks_that_the_table_does_not_name(cuda_device, new):
    dev = cuda_device
    pages, bt = _filled(2, 128, "fp8", [300], 8)
    bt = bt.clone()
    bt[0, 2], bt[0, 7], bt[0, 18] = -1, 10 ** 6, -5
    announce(f"kv8 attention over blocks that are not there {new}")
    got, want, bound = _attend(dev, HEADS["target"], "fp8", [300], [new], pages=pages, bt=bt)
    ref.within(got, want, bound)
    # a length that passes the table
    got, want, bound = _attend(dev, HEADS["target"], "fp8", [400], [new], pages=pages, bt=bt)
    ref.within(got, want, bound)


def test_attention_strides_scale_and_rows_behind(cuda_device):
    """q as a part of a projection, out as a part of a wider tensor, a scale of its own, lengths above
    max_seq_len, rows behind the last sequence left as they were."""
    dev = cuda_device
    h, kv, d = HEADS["draft"]
    pages, bt = _filled(kv, d, "int8", [90, 31], 9)
    new, lens = [3, 2], [90, 31]
    qkv = torch.randn((8, h + 2 * kv, d), generator=_gen(3)).to(torch.bfloat16)
    wide = torch.full((8, h + 3, d), 5.0, dtype=torch.bfloat16, device=dev)
    announce("kv8 attention strided")
    got = ops.kv8_attention(qkv.to(dev)[:, :h], *pages.to(dev), bt.to(dev), _cu(new, dev), _ints([90, 500], dev), 3, 90, scale=0.3,
                            out=wide[:, 1:h + 1])
    torch.cuda.synchronize()
    want, bound = ref.attention(qkv[:5, :h], pages, bt, new, [90, 90], 0.3)
    ref.within(got[:3], want[:3], bound[:3])
    assert bool((wide[5:] == 5.0).all()) and bool((wide[:, 0] == 5.0).all()) and bool((wide[:, h + 1:] == 5.0).all())
    # equal lengths given as one number, an odd view of q
    q = torch.randn((1, h, 2 * d), generator=_gen(4)).to(torch.bfloat16)[:, :, ::2]
    one = ops.kv8_attention(q.to(dev), *pages.to(dev), bt[:1].to(dev), _cu([1], dev), None, 1, 90)
    want, bound = ref.attention(q, pages, bt[:1], [1], [90])
    ref.within(one, want, bound)


def test_attention_scores_far_apart(cuda_device):
    """Scores of several hundred, the largest among the last keys: the running maximum moves late."""
    dev = cuda_device
    h, kv, d = HEADS["target"]
    T = 900
    g = _gen(17)
    k, v = _rows((T, kv, d), g), _rows((T, kv, d), g)
    k = (k.float() * torch.linspace(0.1, 20.0, T)[:, None, None]).to(torch.bfloat16)
    bt = ref.table([57], 60)
    for fmt in ("fp8", "int8"):
        pages = ref.Pages(60, kv, d, fmt)
        pages.write(*ref.slots(bt[0], torch.arange(T)), k, v)
        for new in (1, 5, 50):
            announce(f"kv8 attention of scores far apart {fmt} {new}")
            got, want, bound = _attend(dev, (h, kv, d), fmt, [T], [new], pages=pages, bt=bt)
            ref.within(got, want, bound)


def test_attention_repeats_to_the_bit(cuda_device):
    new, lens = [1, 33, 5, 1], [4000, 700, 2050, 31]
    announce("kv8 attention twice")
    a, _, _ = _attend(cuda_device, HEADS["target"], "fp8", lens, new)
    b, _, _ = _attend(cuda_device, HEADS["target"], "fp8", lens, new)
    assert torch.equal(a.view(torch.int16), b.view(torch.int16))


# ------------------------------------------------------------------------------ together
def test_write_attend_read_over_steps(cuda_device):
    """A prompt, single tokens and verify blocks written and attended to in turn, then read back."""
    dev = cuda_device
    h, kv, d = HEADS["target"]
    fmt = "int8"
    bt = ref.table([20, 12, 8], 41)
    pages = ref.Pages(41, kv, d, fmt)
    kp, vp, sc = pages.to(dev)
    lens, g = [0, 0, 0], _gen(33)
    for new in ([200, 37, 1], [1, 1, 1], [5, 5, 5], [0, 90, 7], [1, 0, 60]):
        lens = [t + n for t, n in zip(lens, new)]
        qkv = _rows((sum(new), h + 2 * kv, d), g, 2.0)
        dq = qkv.to(dev)
        announce(f"kv8 step {new} {lens}")
        ops.kv8_append(dq[:, h:h + kv], dq[:, h + kv:], kp, vp, sc, bt.to(dev), _cu(new, dev), _ints(lens, dev))
        got = ops.kv8_attention(dq[:, :h], kp, vp, sc, bt.to(dev), _cu(new, dev), _ints(lens, dev), max(new), max(lens))
        torch.cuda.synchronize()
        at = 0
        for b, (n, t) in enumerate(zip(new, lens)):
            if n:
                pages.write(*ref.slots(bt[b], torch.arange(t - n, t)), qkv[at:at + n, h:h + kv], qkv[at:at + n, h + kv:])
            at += n
        want, bound = ref.attention(qkv[:, :h], pages, bt, new, lens)
        ref.within(got, want, bound)
    k, v = ops.kv8_gather(kp, vp, sc, bt.to(dev), _cu(lens, dev), _ints([0, 0, 0], dev), sum(lens))
    rows = [pages.read(*ref.slots(bt[b], torch.arange(t))) for b, t in enumerate(lens)]
    assert torch.equal(k.cpu().view(torch.int16), torch.cat([r[0] for r in rows]).to(torch.bfloat16).view(torch.int16))
    assert torch.equal(v.cpu().view(torch.int16), torch.cat([r[1] for r in rows]).to(torch.bfloat16).view(torch.int16))


def test_graphs_and_streams(cuda_device):
    """Two graphs recorded on one stream and replayed side by side on others, with eager calls
    between them: each has its own workspace."""
    dev = cuda_device
    h, kv, d = HEADS["target"]
    new, lens = [5, 1, 40], [900, 333, 64]
    pages, bt = _filled(kv, d, "fp8", lens, 5)
    dp, dbt, cu, ln = pages.to(dev), bt.to(dev), _cu(new, dev), _ints(lens, dev)
    qs = [torch.randn((46, h, d), generator=_gen(i)).to(torch.bfloat16).to(dev) for i in range(2)]
    eager = [ops.kv8_attention(q, *dp, dbt, cu, ln, 40, 900) for q in qs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    side = torch.cuda.Stream()
    for q in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(ops.kv8_attention(q, *dp, dbt, cu, ln, 40, 900))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(3):
        announce(f"kv8 graphs, replay {turn}")
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
        ops.kv8_attention(qs[0], *dp, dbt, cu, ln, 40, 900)
        torch.cuda.synchronize()
        for o, e in zip(outs, eager):
            assert torch.equal(o.view(torch.int16), e.view(torch.int16))


def test_refusals_on_device_tensors(cuda_device):
    dev = cuda_device
    pages, bt = _filled(2, 128, "fp8", [40], 2)
    kp, vp, sc = pages.to(dev)
    bt, cu, ln = bt.to(dev), _cu([1], dev), _ints([40], dev)
    q = torch.zeros((1, 12, 128), dtype=torch.bfloat16, device=dev)
    good = dict(q=q, k_pages=kp, v_pages=vp, scales=sc, block_table=bt, cu_rows=cu, seq_lens=ln, max_q_len=1, max_seq_len=40)
    ops.kv8_attention(**good)
    for bad in (dict(q=q.float()), dict(q=q.cpu()), dict(q=q[:, :11]), dict(q=q[0]), dict(v_pages=vp.view(torch.int8)),
                dict(k_pages=kp.view(torch.uint8)), dict(scales=sc.double()), dict(block_table=bt.long()), dict(cu_rows=cu[:1]),
                dict(seq_lens=ln.long()), dict(max_q_len=0), dict(max_seq_len=0), dict(tree_mask=torch.zeros(2, dtype=torch.int64, device=dev)),
                dict(tree_mask=torch.zeros(1, dtype=torch.int64, device=dev), max_q_len=65), dict(out=q.float()),
                dict(out=q[:, :6]), dict(workspace_tensor=torch.zeros(16, dtype=torch.uint8, device=dev)), dict(max_seq_len=2 ** 31 - 1),
                dict(k_pages=kp[:, :, :, :, :, :8]), dict(q=None)):
        with pytest.raises(SdvError):
            ops.kv8_attention(**{**good, **bad})
    with pytest.raises(SdvError):
        ops.kv8_append(q[:, :2], q[:, :2], kp, vp, sc, bt, cu, None)
    with pytest.raises(SdvError):
        ops.kv8_append(q[:, :2], q[:, :1], kp, vp, sc, bt, cu, ln)
    with pytest.raises(SdvError):
        ops.kv8_gather(kp, vp, sc, bt, cu, ln, -1)
    with pytest.raises(SdvError):
        ops.kv8_gather(kp, vp, sc, bt, cu, ln, 1, k_out=q[:, :4:2])
    none = q[:0]
    assert ops.kv8_attention(none, kp, vp, sc, bt, _cu([0], dev), ln, 1, 40).shape == (0, 12, 128)
    ops.kv8_append(none[:, :2], none[:, :2], kp, vp, sc, bt, _cu([0], dev), ln)
    assert ops.kv8_gather(kp, vp, sc, bt, _cu([0], dev), ln, 0)[0].shape == (0, 2, 128)
