"""The 8-bit KV cache in plain torch on the CPU: quantizer, pages, read-back, attention in 64 bits."""
from __future__ import annotations

import math

import torch

BLOCK = 16
TYPES = {"fp8": torch.float8_e4m3fn, "int8": torch.int8}
LARGEST = {"fp8": 448.0, "int8": 127.0}
U = 2.0 ** -8  # half a step of BF16, relative


def quantize(x: torch.Tensor, fmt: str):
    """(codes, fp32 scales) of BF16 rows (..., D): IEEE divisions, a row that is not finite NaN and 0."""
    x = x.float()
    m = x.abs().amax(-1, keepdim=True)
    s = m / torch.full_like(m, LARGEST[fmt])
    s = torch.where(s == 0, torch.ones_like(s), s)
    finite = torch.isfinite(m)
    y = torch.where(finite, x / s, torch.zeros_like(x))
    code = y.to(TYPES[fmt]) if fmt == "fp8" else torch.round(y).to(TYPES[fmt])
    return code, torch.where(finite, s, torch.full_like(s, math.nan)).squeeze(-1)


class Pages:
    """Pages of one layer, on the CPU; every byte that nothing wrote is 0x7F (NaN in E4M3FN) and
    every such scale NaN, as recycled memory may hold."""

    def __init__(self, num_blocks: int, kv: int, d: int, fmt: str):
        self.kv, self.d, self.fmt = kv, d, fmt
        self.k = torch.full((num_blocks, kv, 4, d // 16, 4, 16), 0x7F, dtype=torch.uint8)
        self.v = torch.full((num_blocks, kv, d, BLOCK), 0x7F, dtype=torch.uint8)
        self.s = torch.full((num_blocks, kv, 2, BLOCK), math.nan)

    def write(self, blk, off, k, v):
        """BF16 rows (n, KV, D) into slots (blk, off) (index tensors)."""
        n = k.shape[0]
        for part, x in enumerate((k, v)):
            code, s = quantize(x, self.fmt)
            code = code.contiguous().view(torch.uint8)
            if part == 0:
                self.k[blk, :, off // 4, :, off % 4] = code.view(n, self.kv, self.d // 16, 16)
            else:
                self.v[blk, :, :, off] = code
            self.s[blk, :, part, off] = s

    def to(self, dev):
        t = TYPES[self.fmt]
        return self.k.to(dev).view(t), self.v.to(dev).view(t), self.s.to(dev)

    def read(self, blk, off):
        """fp32 K and V (n, KV, D) of slots, code * scale rounded to fp32."""
        t, n = TYPES[self.fmt], len(blk)
        k = self.k[blk, :, off // 4, :, off % 4].reshape(n, self.kv, self.d).contiguous().view(t).float()
        v = self.v[blk, :, :, off].contiguous().view(t).float()
        return k * self.s[blk, :, 0, off].unsqueeze(-1), v * self.s[blk, :, 1, off].unsqueeze(-1)

    def codes(self, blk, off):
        """float64 codes and scales (k, v, ks, vs) of slots."""
        t, n = TYPES[self.fmt], len(blk)
        k = self.k[blk, :, off // 4, :, off % 4].reshape(n, self.kv, self.d).contiguous().view(t).double()
        v = self.v[blk, :, :, off].contiguous().view(t).double()
        return k, v, self.s[blk, :, 0, off].double(), self.s[blk, :, 1, off].double()


def table(counts, num_blocks, seed=0):
    """int32 block table of sequences with `counts` blocks at random places; -1 behind them."""
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(num_blocks, generator=g).tolist()
    width = max(1, max(counts))
    rows, at = [], 0
    for c in counts:
        rows.append(order[at:at + c] + [-1] * (width - c))
        at += c
    return torch.tensor(rows, dtype=torch.int32)


def slots(row, positions):
    positions = torch.as_tensor(positions)
    return row[positions // BLOCK].long(), positions % BLOCK


def attention(q, pages, bt, new, lens, scale=None, tree=None):
    """(out, bound) float64 (total, H, D) of BF16 q (total, H, D): the definition in 64 bits, and how
    far a result may lie from it that

    * forms q.c in fp32 from exact products (D + 4 roundings of values up to sum |q c|, the scales' and
      the exponent's own among them), which moves a score by dx and its exponential by as much,
      relatively, in the numerator and in the sum;
    * rounds each exponential times V's scale to BF16 once (U, of sum p |v|), sums in fp32; or, in the
      kernel for many rows, the exponentials p (1 for the largest, so that their sum l is at least 1)
      as 2^7 p and V as 2^b v / 2^E to FP16, 2^E at most the largest V scale s of the keys and b at
      least 5.  Where FP16 is normal that is 2^-11 each of a term, less than U; where it is not,
      half of its smallest step, 2^-25: 2^-32 of p, which makes 2^-32 sum |v| / l, and 2^-30 s of v,
      which makes 2^-30 s, since the p / l sum to 1;
    * rounds the output to BF16 (U, of the output).

    Blocks that the table does not name, and rows that see nothing, as the operator has them.  NaN
    where the row sees a NaN.
    """
    total, H, D = q.shape
    kv, G = pages.kv, H // pages.kv
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros((total, H, D), dtype=torch.float64)
    bound = torch.zeros_like(out)
    nb, at = pages.s.shape[0], 0
    for b, (n, T) in enumerate(zip(new, lens)):
        ctx = T - n
        if n == 0:
            continue
        if T > 0:
            pos = torch.arange(T)
            row = torch.full((-(-T // BLOCK),), -1, dtype=torch.int64)
            have = min(len(row), bt.shape[1])
            row[:have] = bt[b, :have].long()
            named = ((row >= 0) & (row < nb))[pos // BLOCK]
            kc, vc, ks, vs = pages.codes(row.clamp(0, nb - 1)[pos // BLOCK], pos % BLOCK)
            i = torch.arange(n).unsqueeze(1)
            if tree is None:
                seen = pos <= ctx + i
            else:
                j = pos - ctx
                word = tree[at:at + n].unsqueeze(1)
                seen = (pos < ctx) | ((j >= 0) & (j < 64) & ((word >> j.clamp(0, 63)) & 1 == 1))
            seen = seen & named
            x = q[at:at + n].double()
            for h in range(H):
                c, sk = kc[:, h // G], ks[:, h // G] * scale
                y = (x[:, h] @ c.nan_to_num().t()) * sk
                y = torch.where(seen, y, torch.full_like(y, -math.inf))
                m = y.nan_to_num(nan=-math.inf, posinf=math.inf).amax(-1, keepdim=True)
                p = torch.exp(y - torch.where(torch.isinf(m) & (m < 0), torch.zeros_like(m), m))
                v = (vc[:, h // G].nan_to_num() * vs[:, h // G].unsqueeze(-1))
                # what a row does not see does not reach it: a NaN there is left out of the product
                bad = torch.isnan(v).any(-1)
                v0 = torch.where(bad.unsqueeze(-1), torch.zeros_like(v), v)
                l = p.sum(-1, keepdim=True)
                o = (p @ v0) / l
                hit = (seen & bad).any(-1, keepdim=True)
                o = torch.where(hit, torch.full_like(o, math.nan), o)
                none = ~seen.any(-1, keepdim=True)
                o = torch.where(none, torch.zeros_like(o), o)
                size = ((x[:, h].abs() @ c.nan_to_num().abs().t()) * sk.abs()).nan_to_num()
                dx = (D + 4) * 2.0 ** -24 * torch.where(seen, size, torch.zeros_like(size)).amax(-1, keepdim=True) + 2.0 ** -20
                out[at:at + n, h] = o
                tiny = seen.double() @ v0.abs() * 2.0 ** -32 / l
                largest = torch.where(named & ~bad, vs[:, h // G], torch.zeros_like(vs[:, 0])).nan_to_num().max()
                bound[at:at + n, h] = U * o.abs() + (1 + U) * ((U + 2 * dx) * (p @ v0.abs()) / l + tiny + 2.0 ** -30 * largest)
        at += n
    return out, bound


def within(got, want, bound):
    """Largest (error / bound), NaN where and only where `want` has one; bound 0 asks for equality."""
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN in the wrong places"
    ok = ~torch.isnan(want)
    err, b = (got - want).abs()[ok], bound[ok].nan_to_num()
    assert bool((err <= b + 1e-300).all()), f"error {err.max():.3e} where {b[err.argmax()]:.3e} is allowed"
    return float((err / b.clamp(min=1e-300)).max()) if err.numel() else 0.0
