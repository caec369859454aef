"""Rotary positions on the GPU against complex products in 64 bits.

A cos or sin in fp32 is off by at most 2^-21: the angle, at most half a turn after its reduction, by 2^-25 turns or
2^-22 radians (2^-23 more of a turn for positions near 2^31, not used here), and sincospi by four units of 2^-24.  A rotated
value, two products and a sum, is then off by (|x| + |y|) (2^-21 + 2^-22) at most before its rounding to BF16 (half a step, 2^-8
of it)."""
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
FP32 = 2.0 ** -21 + 2.0 ** -22


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rows(shape, seed):
    x = torch.randn(shape, generator=_gen(seed))
    x[..., 3] *= 8.0
    return x.to(torch.bfloat16)


def _ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _turned(x, positions, inv_freq, interleaved, scale=1.0, inverse=False):
    """(rotated rows, |x| + |y| of each value's pair) in 64 bits."""
    r = 2 * inv_freq.numel()
    x = x.double()
    out, size = x.clone(), torch.zeros_like(x)
    even, odd = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    t = torch.outer(torch.as_tensor(positions).double(), inv_freq) * (-1 if inverse else 1)
    w = torch.complex(x[..., even], x[..., odd]) * torch.polar(torch.full_like(t, scale), t)[:, None]
    out[..., even], out[..., odd] = w.real, w.imag
    size[..., even] = size[..., odd] = (x[..., even].abs() + x[..., odd].abs()) * scale
    return out, size


def _check(got, want, size):
    bound = ref.U * want.abs() + (1 + ref.U) * FP32 * size
    return ref.within(got, want, bound)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,rotary", [("target", 128), ("target", 64), ("target", 16), ("draft", 64), ("draft", 48), ("mha", 96), ("mqa", 32)])
@pytest.mark.parametrize("rows", [1, 7, 33, 1000])
def test_rope(cuda_device, heads, rotary, rows, interleaved):
    announce(f"rope {heads} {rotary} {rows} {interleaved}")
    h, kv, d = HEADS[heads]
    x = _rows((rows, h + 2 * kv, d), rows)
    pos = torch.randint(-5000, 1 << 20, (rows,), generator=_gen(rows + 1)).tolist()
    pos[0] = 0
    inv, scale = ops.rope_frequencies(d, rotary_dim=rotary, device="cpu")
    y = x.to(cuda_device)
    q, k = ops.rope(y[:, :h], y[:, h:h + kv], _ints(pos, cuda_device), inv.to(cuda_device), interleaved=interleaved)
    torch.cuda.synchronize()
    assert q.is_contiguous() and k.is_contiguous()
    assert torch.equal(q[0].cpu(), x[0, :h]) and torch.equal(k[0].cpu(), x[0, h:h + kv])  # position 0
    assert torch.equal(q[..., rotary:].cpu(), x[:, :h, rotary:])
    _check(q, *_turned(x[:, :h], pos, inv, interleaved))
    _check(k, *_turned(x[:, h:h + kv], pos, inv, interleaved))
    assert torch.equal(y.cpu(), x)


def test_rope_passes_what_it_does_not_turn_bit_for_bit(cuda_device):
    """Infinities and NaN of the other dimensions, and of other pairs, reach nothing."""
    x = _rows((5, 4, 128), 1)
    x[:, :, 40] = math.nan
    x[:, :, 100] = math.inf
    inv = ops.rope_frequencies(128, rotary_dim=32, device=cuda_device)[0]
    q, none = ops.rope(x.to(cuda_device), None, _ints([1, 2, 3, 4, 5], cuda_device), inv)
    assert none is None
    assert torch.equal(q[..., 32:].cpu().view(torch.int16), x[..., 32:].view(torch.int16))
    assert bool(torch.isfinite(q[..., :32]).all())


@pytest.mark.parametrize("scaling", [{"type": "linear", "factor": 4.0}, {"type": "ntk", "factor": 8.0},
                                     {"type": "yarn", "factor": 4.0, "original": 8192}])
def test_scaled_contexts(cuda_device, scaling):
    x, pos = _rows((64, 6, 128), 4), list(range(100000, 100064))
    inv, scale = ops.rope_frequencies(128, scaling=scaling, device="cpu")
    announce(f"rope {scaling}")
    q, _ = ops.rope(x.to(cuda_device), None, _ints(pos, cuda_device), inv.to(cuda_device), scale=scale)
    _check(q, *_turned(x, pos, inv, False, scale))


@pytest.mark.parametrize("interleaved", [False, True])
def test_inverse_is_the_transpose(cuda_device, interleaved):
    """<rope(x), y> = <x, inverse(y)>: against the definition, against differences of the forward pass, and back again."""
    dev, h, d = cuda_device, 3, 64
    x, y, pos = _rows((9, h, d), 5), _rows((9, h, d), 6), list(range(3, 12))
    inv, _ = ops.rope_frequencies(d, rotary_dim=32, device="cpu")
    g, _ = ops.rope(y.to(dev), None, _ints(pos, dev), inv.to(dev), interleaved=interleaved, scale=1.25, inverse=True)
    want, size = _turned(y, pos, inv, interleaved, 1.25, True)
    _check(g, want, size)
    # the map is linear: its gradient is differences of it along each dimension (in 64 bits, by the definition above)
    basis = torch.eye(d).view(d, 1, d).expand(d, 1, d)
    for p in (3, 7):
        cols, _ = _turned(basis.to(torch.bfloat16), [p] * d, inv, interleaved, 1.25)  # row i: the image of dimension i
        grad = y[p - 3].double() @ cols[:, 0].t()
        assert torch.allclose(grad, want[p - 3], atol=1e-9)
    back, _ = ops.rope(ops.rope(x.to(dev), None, _ints(pos, dev), inv.to(dev), interleaved=interleaved)[0], None, _ints(pos, dev),
                       inv.to(dev), interleaved=interleaved, inverse=True)
    _, size = _turned(x, pos, inv, interleaved)
    ref.within(back, x.double(), 2 * ref.U * size + 4 * FP32 * size + ref.U * x.double().abs())


def test_in_place_and_given_outputs(cuda_device):
    dev, (h, kv, d) = cuda_device, HEADS["target"]
    x = _rows((40, h + 2 * kv, d), 8).to(dev)
    pos, inv = _ints(list(range(40)), dev), ops.rope_frequencies(d, device=dev)[0]
    want = ops.rope(x[:, :h], x[:, h:h + kv], pos, inv)
    out = torch.full((40, h + kv, d), 7.0, dtype=torch.bfloat16, device=dev)
    got = ops.rope(x[:, :h], x[:, h:h + kv], pos, inv, q_out=out[:, :h], k_out=out[:, h:])
    assert got[0].data_ptr() == out.data_ptr() and torch.equal(out, torch.cat(want, 1))
    y = x.clone()
    ops.rope(y[:, :h], y[:, h:h + kv], pos, inv, q_out=y[:, :h], k_out=y[:, h:h + kv])
    assert torch.equal(y, torch.cat((*want, x[:, h + kv:]), 1))
    # rows that the kernel cannot take as they lie are copied
    odd = torch.zeros((40, h * d + 3), dtype=torch.bfloat16, device=dev)[:, 3:].view(40, h, d)
    odd.copy_(x[:, :h])
    assert torch.equal(ops.rope(odd, None, pos, inv)[0], want[0])
    assert torch.equal(ops.rope(x[:, :h].transpose(0, 1).contiguous().transpose(0, 1), None, pos, inv)[0], want[0])
    empty = ops.rope(x[:0, :h], x[:0, h:h + kv], pos[:0], inv)
    assert empty[0].shape == (0, h, d) and empty[1].shape == (0, kv, d)


def test_rope_on_another_stream_and_recorded(cuda_device):
    dev = cuda_device
    x = _rows((16, 4, 64), 9).to(dev)
    pos, inv = _ints(list(range(16)), dev), ops.rope_frequencies(64, device=dev)[0]
    want, _ = ops.rope(x, None, pos, inv)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, _ = ops.rope(x, None, pos, inv)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got, _ = ops.rope(x, None, pos, inv)
    for shift in (5, 70000, 0):
        pos.add_(shift)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, ops.rope(x, None, pos, inv)[0])


# ------------------------------------------------------------------------------ a step's rows
def _cu(new, dev):
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return _ints(cu, dev)


def _read(kp, vp, sc, table, sizes, fmt):
    """fp64 K and scales of the sequences' last tokens."""
    t = ref.TYPES[fmt]
    kp, sc = kp.cpu().view(torch.uint8), sc.cpu()
    ks, ss = [], []
    for b, (n, T) in enumerate(sizes):
        blk, off = ref.slots(table[b], torch.arange(T - n, T))
        ks.append(kp[blk, :, off // 4, :, off % 4].reshape(n, kp.shape[1], kp.shape[3] * 16).contiguous().view(t).double())
        ss.append(sc[blk, :, 0, off].double())
    return torch.cat(ks), torch.cat(ss)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("heads,rotary,interleaved", [("target", 128, False), ("target", 64, True), ("draft", 64, False), ("draft", 32, True),
                                                      ("mha", 96, False), ("mqa", 16, False)])
@pytest.mark.parametrize("new,lens", [([1], [1]), ([1], [17]), ([16], [32]), ([15], [47]), ([300], [1000]), ([1, 1, 1, 1], [5, 16, 17, 333]),
                                      ([0, 3, 0, 20, 1], [9, 3, 0, 25, 40]), ([5, 9, 8, 24], [2000, 13, 8, 100])])
def test_rope_append(cuda_device, fmt, heads, rotary, interleaved, new, lens):
    announce(f"kv8 rope append {fmt} {heads} {rotary} {interleaved} {new} {lens}")
    dev, (h, kv, d) = cuda_device, HEADS[heads]
    total, counts = sum(new), [-(-t // 16) for t in lens]
    nb = sum(counts) + 5
    table = ref.table(counts, nb, 11)
    pages = ref.Pages(nb, kv, d, fmt)
    x = _rows((total + 2, h + 2 * kv, d), total)  # two rows behind the last sequence
    if total > 4:
        x[1, h:], x[2, h:] = 0.0, 2.0 ** -130
    inv, _ = ops.rope_frequencies(d, rotary_dim=rotary, device="cpu")
    kp, vp, sc = pages.to(dev)
    y = x.to(dev)
    q_out = torch.full((total + 2, h, d), 7.0, dtype=torch.bfloat16, device=dev)
    for out in (None, q_out):
        q = ops.kv8_rope_append(y[:, :h], y[:, h:h + kv], y[:, h + kv:], kp, vp, sc, table.to(dev), _cu(new, dev), _ints(lens, dev), 0,
                                inv.to(dev), interleaved=interleaved, q_out=out)
    torch.cuda.synchronize()
    pos = [p for n, t in zip(new, lens) for p in range(t - n, t)]
    assert bool((q_out[total:] == 7.0).all())
    assert torch.equal(q[:total], ops.rope(y[:total, :h], None, _ints(pos, dev), inv.to(dev), interleaved=interleaved)[0])
    # V as kv8_append writes it, K as fp32 rotation and quantization would, to one code where a rounding falls otherwise
    at = 0
    for b, (n, t) in enumerate(zip(new, lens)):
        if n:
            pages.write(*ref.slots(table[b], torch.arange(t - n, t)), x[at:at + n, h:h + kv], x[at:at + n, h + kv:])
        at += n
    assert torch.equal(vp.view(torch.uint8).cpu(), pages.v)
    untouched = torch.isnan(pages.s[:, :, 0])
    assert torch.equal(torch.isnan(sc.cpu()), torch.isnan(pages.s)) and torch.equal(sc.cpu()[:, :, 1][~untouched], pages.s[:, :, 1][~untouched])
    keep = kp.view(torch.uint8).cpu().permute(0, 1, 2, 4, 3, 5).reshape(nb, kv, 16, d)[untouched]
    assert bool((keep == 0x7F).all())
    want, size = _turned(x[:total, h:h + kv], pos, inv, interleaved)
    codes, scales = _read(kp, vp, sc, table, list(zip(new, lens)), fmt)
    off = (FP32 * size).amax(-1)
    top = want.abs().amax(-1)
    Q = ref.LARGEST[fmt]
    s = torch.where(top == 0, torch.ones_like(top), top / Q)
    # a scale in fp32: the maximum's error and the division's (2^-24, or half of the smallest number)
    assert bool(((scales - s).abs() <= off / Q + 2.0 ** -23 * s + 2.0 ** -149).all())
    # a code's value: half a step of it (E4M3FN: 2^-4 of the value, 2^-10 of the scale below its normal numbers) from value / scale
    ratio = want / scales[..., None]
    half = torch.maximum(ratio.abs() * 2.0 ** -4, torch.tensor(2.0 ** -10)) if fmt == "fp8" else torch.tensor(0.5)
    err = (off / scales)[..., None] * 1.1 + ratio.abs() * 2.0 ** -22
    edge = (ratio.abs() - Q).clamp(min=0)  # past the largest code: at most it
    assert bool(((codes - ratio).abs() <= half * (1 + 2.0 ** -20) + err * 1.1 + edge).all())


def test_positions_of_a_tree(cuda_device):
    """positions turn the rows, the slots stay: the same as a rotation by those and a write of what it gives, to K's rounding."""
    dev, (h, kv, d) = cuda_device, HEADS["target"]
    new, lens = [24, 7], [500, 1023]
    counts = [-(-t // 16) for t in lens]
    table = ref.table(counts, sum(counts) + 2, 3).to(dev)
    x = _rows((31, h + 2 * kv, d), 31).to(dev)
    g = torch.Generator().manual_seed(2)
    pos = torch.cat([t - n + torch.randint(0, 5, (n,), generator=g) for n, t in zip(new, lens)]).to(torch.int32).to(dev)
    inv = ops.rope_frequencies(d, device=dev)[0]
    a, b = (ref.Pages(sum(counts) + 2, kv, d, "int8").to(dev) for _ in range(2))
    rest = (table, _cu(new, dev), _ints(lens, dev))
    q = ops.kv8_rope_append(x[:, :h], x[:, h:h + kv], x[:, h + kv:], *a, *rest, 0, inv, positions=pos)
    q2, k2 = ops.rope(x[:, :h], x[:, h:h + kv], pos, inv)
    ops.kv8_append(k2, x[:, h + kv:], *b, *rest)
    assert torch.equal(q, q2) and torch.equal(a[1], b[1]) and torch.equal(torch.isnan(a[2]), torch.isnan(b[2]))
    starts = _ints([t - n for n, t in zip(new, lens)], dev)
    ka, _ = ops.kv8_gather(*a, table, rest[1], starts, 31)
    kb, _ = ops.kv8_gather(*b, table, rest[1], starts, 31)
    # two roundings to BF16 (before and after), and a code's step where they move one: s = max / 127
    step = k2.double().abs().amax(-1, keepdim=True) / 127 * (1 + ref.U)
    assert bool(((ka.double() - kb.double()).abs() <= step + 2 * ref.U * kb.double().abs() + step * ref.U).all())


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_rows_that_are_not_finite_or_have_no_slot(cuda_device, fmt):
    dev = cuda_device
    h, kv, d = 4, 2, 64
    announce(f"kv8 rope append of rows that are not finite, lengths below the row counts {fmt}")
    x = _rows((20, h + 2 * kv, d), 7)
    x[3, h, 7], x[4, h + 1, 0], x[5, h + kv, 5] = math.inf, math.nan, -math.inf
    new, lens = [6, 10, 4], [6, 4, 40]  # the second's first six rows are at -6 .. -1
    table = ref.table([1, 1, 3], 6, 1)
    table[2, 2] = 99  # no such block: positions 32 .. 39
    inv = ops.rope_frequencies(d, device=dev)[0]
    kp, vp, sc = ref.Pages(6, kv, d, fmt).to(dev)
    y = x.to(dev)
    q = ops.kv8_rope_append(y[:, :h], y[:, h:h + kv], y[:, h + kv:], kp, vp, sc, table.to(dev), _cu(new, dev), _ints(lens, dev), 0, inv)
    pos = list(range(6)) + list(range(-6, 4)) + list(range(36, 40))
    assert torch.equal(q, ops.rope(y[:, :h], None, _ints(pos, dev), inv)[0])
    one = table[0, 0]
    got = sc.cpu()[one]
    assert bool(torch.isnan(got[0, 0, 3])) and bool(torch.isnan(got[1, 0, 4])) and bool(torch.isnan(got[0, 1, 5]))
    assert bool(torch.isfinite(got[1, 0, [0, 1, 2, 3, 5]]).all()) and bool(torch.isfinite(got[0, 0, [0, 1, 2, 4, 5]]).all())
    codes = kp.view(torch.uint8).cpu()[one, 0].permute(0, 2, 1, 3).reshape(16, d)
    assert bool((codes[3] == 0).all()) and bool((codes[6:] == 0x7F).all())
    assert bool(torch.isnan(sc.cpu()[table[2, 0]]).all()) and bool(torch.isfinite(sc.cpu()[table[1, 0], :, :, :4]).all())


def test_one_length_for_all_in_a_graph(cuda_device):
    """seq_lens None: a recorded step follows the rows it is given."""
    dev, (h, kv, d) = cuda_device, HEADS["draft"]
    table = ref.table([4, 4], 9, 1).to(dev)
    inv = ops.rope_frequencies(d, device=dev)[0]
    pages = ref.Pages(9, kv, d, "fp8").to(dev)
    x, cu = _rows((6, h + 2 * kv, d), 3).to(dev), _cu([3, 3], dev)
    call = lambda p: ops.kv8_rope_append(x[:, :h], x[:, h:h + kv], x[:, h + kv:], *p, table, cu, None, 50, inv)  # noqa: E731
    call(pages)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = call(pages)
    for seed in (4, 5, 6):
        x.copy_(_rows((6, h + 2 * kv, d), seed))
        graph.replay()
        torch.cuda.synchronize()
        other = ref.Pages(9, kv, d, "fp8").to(dev)
        assert torch.equal(q, call(other))
        for a, b in zip(pages, other):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_refusals(cuda_device):
    dev, (h, kv, d) = cuda_device, HEADS["draft"]
    x, pos, inv = _rows((6, h + kv, d), 3).to(dev), _ints(list(range(6)), dev), ops.rope_frequencies(d, device=dev)[0]
    q, k = x[:, :h], x[:, h:]
    for bad in (dict(q=q.float()), dict(k=k[:5]), dict(positions=pos.long()), dict(positions=pos[:5]), dict(positions=pos.cpu()),
                dict(q=q[:, :0]), dict(inv_freq=inv.float()), dict(inv_freq=inv[:5]), dict(inv_freq=torch.cat((inv, inv))), dict(inv_freq=inv[:0]), dict(q=q[..., :32]),
                dict(q_out=q[:5]), dict(k=None, k_out=k.clone()), dict(q_out=torch.empty((6, h, d + 1), dtype=torch.bfloat16, device=dev)[..., :d])):
        args = dict(q=q, k=k, positions=pos, inv_freq=inv)
        args.update(bad)
        with pytest.raises(SdvError):
            ops.rope(**args)
    pages = ref.Pages(4, kv, d, "fp8").to(dev)
    rest = dict(q=q, k_new=k, v_new=k, k_pages=pages[0], v_pages=pages[1], scales=pages[2], block_table=ref.table([2], 4).to(dev),
                cu_rows=_cu([6], dev), seq_lens=None, max_seq_len=9, inv_freq=inv)
    for bad in (dict(q=q[:5]), dict(v_new=k[:5]), dict(max_seq_len=0), dict(inv_freq=inv.float()), dict(positions=pos[:4]), dict(k_new=q),
                dict(cu_rows=_cu([3, 3], dev)), dict(q_out=k)):
        with pytest.raises(SdvError):
            ops.kv8_rope_append(**{**rest, **bad})
