"""Gradients of rotary positions: against the formula in 64 bits (with the bound of tests/test_gpu_rope.py: a gradient is a result
rotated back) and against differences."""
from __future__ import annotations

import pytest
import torch

import kv8_reference as ref
from conftest import announce
from specdec_amd._native import SdvError
from specdec_amd.kernels import ops
from test_gpu_rope import FP32, HEADS, _check, _ints, _rows, _turned

pytestmark = pytest.mark.gpu


def _leaves(heads, n, dev, seed=1):
    h, kv, d = HEADS[heads]
    return [_rows((n, c, d), seed + i).to(dev).requires_grad_() for i, c in enumerate((h, kv))], ops.rope_frequencies(d, device=dev)[0]


@pytest.mark.parametrize("heads,rotary", [("target", 128), ("draft", 32), ("mqa", 64)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("n", [1, 37])
def test_the_transposed_map(cuda_device, heads, rotary, interleaved, inverse, n):
    dev = cuda_device
    (q, k), _ = _leaves(heads, n, dev)
    inv, _ = ops.rope_frequencies(q.shape[-1], rotary_dim=rotary, device=dev)
    pos = torch.arange(7, 7 + 1000 * n, 1000, dtype=torch.int32, device=dev)
    how = dict(interleaved=interleaved, scale=1.25, inverse=inverse)
    announce(f"rope gradients {heads} {rotary} {how} {n}")
    outs = ops.rope(q, k, pos, inv, **how)
    with torch.no_grad():
        plain = ops.rope(q, k, pos, inv, **how)
    assert all(torch.equal(x, y) and x.requires_grad and not y.requires_grad for x, y in zip(outs, plain))
    up = [_rows(x.shape, 11 + i).to(dev) for i, x in enumerate(outs)]
    got = torch.autograd.grad(outs, (q, k), up)
    for g, w in zip(got, up):
        # the cotangent passes where dimensions do
        want, size = _turned(w.cpu(), pos.cpu(), inv.cpu(), interleaved, 1.25, not inverse)
        _check(g, want, size)
        if rotary < q.shape[-1]:
            assert torch.equal(g[..., rotary:], w[..., rotary:])


@pytest.mark.parametrize("interleaved", [False, True])
def test_against_differences(cuda_device, interleaved):
    """L = sum w rope(q): L(q + e) - L(q - e) is 2 <grad, e>, but for each value's rounding.  q and e are small whole numbers, so
    that q + e and q - e are exact, and w is close to the rotated e, so that the difference is large."""
    dev, n = cuda_device, 21
    g = torch.Generator().manual_seed(5)
    q = torch.randint(-8, 9, (n, 4, 64), generator=g).to(torch.bfloat16).to(dev).requires_grad_()
    e = torch.randint(-1, 2, (n, 4, 64), generator=g).to(torch.bfloat16).to(dev)
    inv, _ = ops.rope_frequencies(64, device=dev)
    pos = _ints(list(range(100, 100 + n)), dev)
    turn = lambda x: ops.rope(x, None, pos, inv, interleaved=interleaved)[0]  # noqa: E731
    w = turn(e)
    announce(f"rope differences {interleaved}")
    out = turn(q)
    (grad,) = torch.autograd.grad(out, q, w)
    ends = [turn(q.detach() + s * e) for s in (1, -1)]
    far = [x.detach().double() for x in ends]
    difference = float((w.double() * (far[0] - far[1])).sum())
    want = 2 * float((grad.double() * e.double()).sum())
    fp32 = (1 + ref.U) * FP32 * 18.0  # of |x| + |y| up to 18
    bound = float((w.double().abs() * (ref.U * (far[0].abs() + far[1].abs()) / (1 - ref.U) + 2 * fp32)).sum())
    bound += 2 * float((e.double().abs() * (ref.U * grad.double().abs() / (1 - ref.U) + fp32)).sum())
    assert bound < 0.1 * abs(want) and abs(difference - want) <= bound


def test_one_of_the_two(cuda_device):
    """Only one result is used, or only one input needs a gradient; none, no rows, and sums' broadcast cotangents."""
    dev = cuda_device
    (q, k), inv = _leaves("target", 9, dev)
    pos = _ints(list(range(9)), dev)
    ones = ops.rope(torch.ones_like(q), torch.ones_like(k), pos, inv, inverse=True)
    announce("rope gradients of one")
    a, b = ops.rope(q, k, pos, inv)
    got = torch.autograd.grad(b.sum(), (q, k), allow_unused=True, retain_graph=True)
    assert got[0] is None and torch.equal(got[1], ones[1])
    assert torch.equal(torch.autograd.grad(a.sum(), q, retain_graph=True)[0], ones[0])
    both = torch.autograd.grad(a.sum() + b.sum(), (q, k))
    assert torch.equal(both[0], ones[0]) and torch.equal(both[1], ones[1])
    a, b = ops.rope(q, None, pos, inv)
    assert b is None and torch.equal(torch.autograd.grad(a.sum(), q)[0], ones[0])
    a, b = ops.rope(q.detach(), k, pos, inv)
    assert torch.equal(torch.autograd.grad(b.sum() + a.sum(), k)[0], ones[1])
    a, b = ops.rope(q[:0], k[:0], pos[:0], inv)
    (a.sum() + b.sum()).backward()
    assert not bool(q.grad.any()) and not bool(k.grad.any())
    out = torch.empty_like(q)
    assert ops.rope(q, None, pos, inv, q_out=out)[0] is out and not out.requires_grad
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        a, _ = ops.rope(q, None, pos, inv)
        pos.add_(1)
        a.sum().backward()


def test_a_gradient_of_a_gradient(cuda_device):
    dev = cuda_device
    (q, _), inv = _leaves("draft", 5, dev)
    pos = _ints([3, 1, 4, 1, 5], dev)
    up = _rows(q.shape, 7).to(dev).requires_grad_()
    (g,) = torch.autograd.grad(ops.rope(q, None, pos, inv)[0], q, up, create_graph=True)
    v = _rows(q.shape, 8).to(dev)
    announce("a gradient of rope's gradient")
    assert torch.equal(torch.autograd.grad(g, up, v)[0], ops.rope(v, None, pos, inv)[0])


@pytest.mark.parametrize("compiled", [False, True])
def test_the_torch_operator(cuda_device, compiled):
    dev = cuda_device
    (q, k), inv = _leaves("target", 12, dev)
    pos = _ints(list(range(50, 62)), dev)
    up = [_rows(x.shape, 11 + i).to(dev) for i, x in enumerate((q, k))]
    turn = lambda q, k: torch.ops.sdv.rope(q, k, pos, inv, True, 0.5)  # noqa: E731
    if compiled:
        turn = torch.compile(turn, fullgraph=True, backend="aot_eager")
    announce(f"gradients of sdv::rope {compiled}")
    got = torch.autograd.grad(turn(q, k), (q, k), up)
    want = torch.autograd.grad(ops.rope(q, k, pos, inv, interleaved=True, scale=0.5), (q, k), up)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    if not compiled:
        torch.library.opcheck(torch.ops.sdv.rope.default, (q, k, pos, inv, True, 0.5))


@pytest.mark.parametrize("library", [False, True])
def test_a_recorded_gradient(cuda_device, library):
    """Of rows that the recording makes: every replay gives the eager gradients of the inputs of the time."""
    dev = cuda_device
    (x, y), inv = _leaves("target", 33, dev)
    pos = _ints(list(range(33)), dev)
    up = [_rows(t.shape, 11 + i).to(dev) for i, t in enumerate((x, y))]
    turn = (lambda q, k: torch.ops.sdv.rope(q, k, pos, inv, False, 2.0)) if library else (lambda q, k: ops.rope(q, k, pos, inv, scale=2.0))

    def step(x, y):
        q, k = x * 2, y * 2
        a, b = turn(q, k)
        return [a, b, *torch.autograd.grad((a, b), (q, k), up)]
    fresh = lambda: [t.detach().clone().requires_grad_() for t in (x, y)]  # noqa: E731
    announce(f"rope's gradient: warm-up {library}")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*fresh())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = [t.detach() for t in step(x, y)]
    for turn_ in range(4):
        with torch.no_grad():
            for i, t in enumerate((x, y, *up)):
                t.copy_(_rows(t.shape, 30 + 5 * turn_ + i))
            pos.add_(100)
        announce(f"rope's gradient: replay {turn_} {library}")
        graph.replay()
        want = step(*fresh())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("library", [False, True])
def test_a_leafs_gradient_is_not_recorded(cuda_device, library):
    dev = cuda_device
    (q, k), inv = _leaves("draft", 5, dev)
    pos = _ints([3, 1, 4, 1, 5], dev)
    turn = torch.ops.sdv.rope if library else ops.rope
    up = [torch.ones_like(q), torch.ones_like(k)]
    announce(f"a leaf's gradient in a recording {library}")
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(SdvError, match="leaves"):
        with torch.cuda.graph(graph):
            outs = turn(q, k, pos, inv)
            torch.autograd.grad(outs, (q, k), up)
    got = torch.autograd.grad(turn(q, k, pos, inv), (q, k), up)
    assert torch.equal(got[0], ops.rope(up[0], None, pos, inv, inverse=True)[0])
