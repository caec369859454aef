"""How exactly kv8 attention's kernel for few rows holds the operands of its product with V: the probability
times V's scale in two BF16 numbers, 2^-16 of it.  The bound of kv8_reference allows one of them, 2^-8,
to every kernel; here V comes in pairs that all but cancel, so that the output's own rounding hides nothing."""
from __future__ import annotations

import pytest
import torch

import kv8_reference as ref
from conftest import announce

HEADS = {"target": (12, 2, 128), "draft": (14, 2, 64)}
SHAPES = [([1], [2]), ([1], [17]), ([2], [300]), ([5], [64]), ([1, 1, 2], [40, 5, 2500]), ([5, 4], [1000, 6])]


def _case(heads, fmt, new, lens):
    """(q, pages, table) of a V whose odd tokens are the even ones' negatives but for one step in sixteen."""
    h, kv, d = HEADS[heads]
    g = torch.Generator().manual_seed(sum(lens))
    counts = [-(-t // 16) for t in lens]
    bt = ref.table(counts, sum(counts) + 2, 3)
    pages = ref.Pages(sum(counts) + 2, kv, d, fmt)
    for b, t in enumerate(lens):
        k = torch.randn((t, kv, d), generator=g)
        v = torch.randn((t, kv, d), generator=g) + 2.0
        v[1::2] = -v[0::2][: t // 2] * (1 + torch.randn((t // 2, kv, d), generator=g) / 16)
        pages.write(*ref.slots(bt[b], torch.arange(t)), k.to(torch.bfloat16), v.to(torch.bfloat16))
    q = (torch.randn((sum(new), h, d), generator=g) / 16).to(torch.bfloat16)
    return q, pages, bt


def _evaluate(q, pages, bt, new, lens, bits=None):
    """(out, bound) float64 of the definition, and how far the kernel may lie from it: U of the output, and
    of sum p |v| / l

    * 2^-16 for the operands, 2^-24 for their product in fp32 before that, and 2^-24 each for the roundings of a sum over T keys
      and of the factors that bring its parts together (T + 32 of them at most);
    * 2 dx for the scores' error dx: D + 4 roundings of values up to sum |q c|, scaled, and 2^-20 for the exponential.

    bits: round the operand p s to that many BF16 numbers, as a kernel might."""
    total, H, D = q.shape
    G = H // pages.kv
    out, bound, at = torch.zeros((total, H, D), dtype=torch.float64), torch.zeros((total, H, D), dtype=torch.float64), 0
    for b, (n, t) in enumerate(zip(new, lens)):
        kc, vc, ks, vs = pages.codes(*ref.slots(bt[b], torch.arange(t)))
        seen = torch.arange(t) <= t - n + torch.arange(n).unsqueeze(1)
        for h in range(H):
            x, c, s = q[at:at + n, h].double(), kc[:, h // G], ks[:, h // G] * D ** -0.5
            y = (x @ c.t()) * s
            p = torch.exp(y - y.masked_fill(~seen, -torch.inf).amax(-1, keepdim=True)) * seen
            l, e = p.sum(-1, keepdim=True), p * vs[:, h // G]
            if bits is not None:
                left, e = e, torch.zeros_like(e)
                for _ in range(bits):
                    part = left.to(torch.bfloat16).double()
                    e, left = e + part, left - part
            v = vc[:, h // G]
            size = (((x.abs() @ c.abs().t()) * s) * seen).amax(-1, keepdim=True)
            dx = (D + 4) * 2.0 ** -24 * size + 2.0 ** -20
            o, most = (e @ v) / l, ((p * vs[:, h // G]) @ v.abs()) / l
            out[at:at + n, h] = o
            bound[at:at + n, h] = ref.U * o.abs() + (1 + ref.U) * (2.0 ** -16 + (t + 33) * 2.0 ** -24 + 2 * dx) * most
        at += n
    return out, bound


@pytest.mark.gpu
@pytest.mark.parametrize("new,lens", SHAPES)
@pytest.mark.parametrize("heads,fmt", [("target", "fp8"), ("target", "int8"), ("draft", "fp8"), ("draft", "int8")])
def test_few_rows(cuda_device, heads, fmt, new, lens):
    from specdec_amd.kernels import ops

    dev = cuda_device
    q, pages, bt = _case(heads, fmt, new, lens)
    cu = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32, device=dev)
    announce(f"kv8 attention, V that all but cancels {heads} {fmt} {new} {lens}")
    got = ops.kv8_attention(q.to(dev), *pages.to(dev), bt.to(dev), cu, torch.tensor(lens, dtype=torch.int32, device=dev), max(new), max(lens))
    torch.cuda.synchronize()
    ref.within(got, *_evaluate(q, pages, bt, new, lens))


@pytest.mark.parametrize("new,lens", SHAPES)
@pytest.mark.parametrize("heads,fmt", [("target", "fp8"), ("draft", "int8")])
def test_the_bound_tells_one_operand_from_two(heads, fmt, new, lens):
    """The definition with the operand rounded to two BF16 numbers and the output to BF16 keeps the bound; rounded to
    one it does not."""
    q, pages, bt = _case(heads, fmt, new, lens)
    want, bound = _evaluate(q, pages, bt, new, lens)
    full, wide = ref.attention(q, pages, bt, new, lens)
    assert torch.allclose(full, want, rtol=1e-9, atol=1e-12)
    ref.within(_evaluate(q, pages, bt, new, lens, 2)[0].to(torch.bfloat16), want, bound)
    one = _evaluate(q, pages, bt, new, lens, 1)[0].to(torch.bfloat16)
    ref.within(one, want, wide)  # the general bound does not tell
    with pytest.raises(AssertionError):
        ref.within(one, want, bound)
