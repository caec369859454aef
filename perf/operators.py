"""The 8-bit KV cache's operators, as cases to time and to check.

A case is a dict of plain values; "kind" says which operator it goes through:

* ``write``   ``ops.kv8_append``: the new tokens' K and V quantized and written into the pages;
* ``read``    ``ops.kv8_gather``: a stretch of every sequence read back into packed BF16 rows;
* ``attend``  ``ops.kv8_attention``: every sequence's new tokens over its paged context -- single
              tokens, verify blocks, trees of drafted tokens, prompt chunks, or all in one batch.

"lo" and "hi" bound the context lengths (the new tokens among them), "new_lo" and "new_hi" the new
tokens (for ``read`` the rows read back) of each sequence; "mixed" gives every sequence but the
first a single new token.  "fmt" is the pages' type.  Head shapes are the Qwen2.5 ones the rest of
the repository uses (12/2/128 and 14/2/64).

The plain form is torch operations in 32 bits over the same pages.  Page layout, per block and KV
head: K codes [4][D/16][4][16] (token 4p+r, dimension 16c+j at [p][c][r][j]), V codes [D][16],
scales [2][16] (K's, then V's).
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

_TARGET = {"heads": 12, "kv": 2, "dim": 128}
_DRAFT = {"heads": 14, "kv": 2, "dim": 64}
_BLOCK = 16
_TYPES = {"fp8": torch.float8_e4m3fn, "int8": torch.int8}
_LARGEST = {"fp8": 448.0, "int8": 127.0}


def _case(name, kind, shape, fmt, batch, context, new, tree=False, mixed=False):
    return {"name": name, "kind": kind, **shape, "fmt": fmt, "batch": batch, "lo": context[0], "hi": context[1], "new_lo": new[0],
            "new_hi": new[1], "tree": tree, "mixed": mixed, "lengths": 41}


def listed():
    return [
        # a decode step of a serving batch writes its 32 new tokens: the smallest write
        _case("write_tokens32", "write", _TARGET, "fp8", 32, (2048, 32768), (1, 1)),
        # the last 2048-token chunk of an 8K prompt written into one layer
        _case("write_chunk2048", "write", _TARGET, "fp8", 1, (8192, 8192), (2048, 2048)),
        # whole and continued prompts of a batch, packed, none of them page-aligned, draft heads
        _case("write_ragged_int8", "write", _DRAFT, "int8", 8, (4001, 8191), (100, 4000)),
        # one 8K sequence read back, as a tool that wants the cache's tensors does
        _case("read_8192", "read", _TARGET, "fp8", 1, (8192, 8192), (8192, 8192)),
        # a batch of contexts read back to move them to another cache
        _case("read_batch_int8", "read", _TARGET, "int8", 16, (2048, 16384), (1999, 16001)),
        # single-token decode over a short context: what one call costs when there is little to read
        _case("decode_1x2048", "attend", _TARGET, "fp8", 1, (2048, 2048), (1, 1)),
        # the draft model's decode, at a length that is no multiple of a page
        _case("draft_1x8191_int8", "attend", _DRAFT, "int8", 1, (8191, 8191), (1, 1)),
        # decode of a serving batch: 32 sequences of 2K to 32K tokens
        _case("batch32_ragged", "attend", _TARGET, "fp8", 32, (2048, 32768), (1, 1)),
        # the target verifies trees of 24 drafted tokens for four sequences
        _case("tree_4x8192", "attend", _TARGET, "fp8", 4, (4096, 8192), (24, 24), tree=True),
        # the speculative verify step of a batch: five rows each
        _case("verify_8x4096_int8", "attend", _TARGET, "int8", 8, (1000, 4096), (5, 5)),
        # the last 2048-token chunk of an 8K prompt, one layer of the target: the largest
        _case("chunk_2048x8192", "attend", _TARGET, "fp8", 1, (8192, 8192), (2048, 2048)),
        # a serving step of the draft: one prompt chunk of 777 tokens among 15 decoding sequences
        _case("mixed_777_int8", "attend", _DRAFT, "int8", 16, (1500, 5000), (777, 777), mixed=True),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over the logarithm, odd ones among them."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 100)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(["write", "read", "attend", "attend", "attend"])
        case = {"kind": kind, **rng.choice([_TARGET, _DRAFT]), "fmt": rng.choice(["fp8", "int8"]), "batch": rng.choice([1, 1, _log(rng, 2, 48)]),
                "tree": False, "mixed": False, "lengths": rng.randrange(1 << 20)}
        if kind == "attend":
            what = rng.choice(["decode", "verify", "tree", "chunk", "mixed"])
            if what == "decode":
                new = (1, 1)
            elif what == "verify":
                new = (rng.randint(2, 8),) * 2 if rng.random() < 0.5 else (1, rng.randint(3, 16))
            elif what == "tree":
                new = (_log(rng, 2, 64),) * 2
            else:
                new = (_log(rng, 17, 2048),) * 2
                case["mixed"] = what == "mixed"
            case["tree"] = what == "tree"
        else:
            lo = _log(rng, 1, 4096)
            new = (lo, _log(rng, lo, 8192))
        lo = _log(rng, max(16, new[1]), max(32768, new[1]))
        case.update(lo=lo, hi=_log(rng, lo, max(32768, lo)), new_lo=new[0], new_hi=new[1])
        if _cost(case) <= most:
            return case


# ---------------------------------------------------------------------------- sizes
def _lengths(case):
    """(context length, new tokens) of every sequence; the first has the longest context."""
    rng = random.Random(case["lengths"])
    out = []
    for b in range(case["batch"]):
        t = case["hi"] if b == 0 else rng.randint(case["lo"], case["hi"])
        n = 1 if case["mixed"] and b else rng.randint(case["new_lo"], case["new_hi"])
        out.append((t, min(n, t)))
    return out


def work(case):
    h, kv, d = case["heads"], case["kv"], case["dim"]
    page, plain = kv * (2 * d + 8), kv * 4 * d  # bytes of a token's codes and scales, and of its BF16 K and V
    nbytes = flops = 0
    for t, n in _lengths(case):
        if case["kind"] == "attend":
            nbytes += t * page + 4 * n * h * d + 4 * -(-t // _BLOCK)
            flops += 4 * h * d * (n * (t - n) + n * (n + 1) // 2)
        else:
            nbytes += n * (page + plain) + 4 * (-(-n // _BLOCK) + 1)
    return {"bytes": nbytes, "flops": flops}


# ---------------------------------------------------------------------------- inputs
def _values(shape, g, outliers):
    """N(0, 1) in BF16; 1% of the (KV head, dimension) channels `outliers` times as large."""
    x = torch.randn(shape, generator=g, device="cuda")
    channels = shape[-2] * shape[-1]
    factor = torch.ones(channels, device="cuda")
    factor[torch.randperm(channels, generator=g, device="cuda")[: max(1, round(0.01 * channels))]] = outliers
    return (x * factor.reshape(shape[-2:])).to(torch.bfloat16)


def _quantize(x, fmt):
    """(codes, fp32 scales) of BF16 rows (..., D): max|x| / 448 or / 127, 1 for a row of zeros."""
    x = x.float()
    m = x.abs().amax(-1, keepdim=True)
    scale = m / torch.full_like(m, _LARGEST[fmt])
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    code = (x / scale).to(_TYPES[fmt]) if fmt == "fp8" else torch.round(x / scale).to(_TYPES[fmt])
    return code, scale.squeeze(-1)


def _store(state, blk, off, k, v):
    """BF16 rows (n, KV, D) quantized into slots (blk, off) of the pages."""
    kp, vp, sc = state["k_pages"].view(torch.uint8), state["v_pages"].view(torch.uint8), state["scales"]
    n, kv, d = k.shape
    kc, ks = _quantize(k, state["fmt"])
    vc, vs = _quantize(v, state["fmt"])
    kp[blk, :, off // 4, :, off % 4] = kc.view(torch.uint8).view(n, kv, d // 16, 16)
    vp[blk, :, :, off] = vc.view(torch.uint8)
    sc[blk, :, 0, off] = ks
    sc[blk, :, 1, off] = vs


def _tree(n, rng):
    """Visibility of a random tree of n drafted tokens: bit j of word i says that token i sees token j."""
    words = []
    for i in range(n):
        words.append((words[rng.randint(max(0, i - 4), i - 1)] if i else 0) | 1 << i)
    return [w - (1 << 64) if w >> 63 else w for w in words]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind, h, kv, d, fmt = case["kind"], case["heads"], case["kv"], case["dim"], case["fmt"]
    sizes = _lengths(case)
    lens, new = [t for t, _ in sizes], [n for _, n in sizes]
    counts = [-(-t // _BLOCK) for t in lens]
    nb = sum(counts) + 8
    # a pool whose blocks lie scattered, and a table of every sequence's
    order = torch.randperm(nb, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(counts)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = order[at:at + c]
        at += c
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    state = {"kind": kind, "fmt": fmt, "table": table, "cu": ints(starts), "lens": ints(lens), "max_new": max(new), "max_len": max(lens),
             "total": starts[-1], "host": (lens, new),
             "k_pages": torch.zeros((nb, kv, 4, d // 16, 4, 16), dtype=torch.uint8, device="cuda").view(_TYPES[fmt]),
             "v_pages": torch.zeros((nb, kv, d, _BLOCK), dtype=torch.uint8, device="cuda").view(_TYPES[fmt]),
             "scales": torch.ones((nb, kv, 2, _BLOCK), dtype=torch.float32, device="cuda")}
    # the new tokens' rows as a projection leaves them: q, k and v of a token side by side
    rows = torch.empty((starts[-1], h + 2 * kv, d), dtype=torch.bfloat16, device="cuda")
    rows[:, h:h + kv] = _values((starts[-1], kv, d), g, 8.0)
    rows[:, h + kv:] = _values((starts[-1], kv, d), g, 20.0)
    if kind == "write":
        zero = torch.randperm(starts[-1], generator=g, device="cuda")[: starts[-1] // 1000]
        rows[zero, h:] = 0.0  # padding rows
        state.update(k=rows[:, h:h + kv], v=rows[:, h + kv:])
        return state
    for b, t in enumerate(lens):
        pos = torch.arange(t, device="cuda")
        _store(state, table[b].long()[pos // _BLOCK], pos % _BLOCK, _values((t, kv, d), g, 8.0), _values((t, kv, d), g, 20.0))
    if kind == "read":
        state["starts"] = ints([t - n for t, n in sizes])
        return state
    rows[:, :h] = torch.randn((starts[-1], h, d), generator=g, device="cuda").to(torch.bfloat16)
    state["q"] = rows[:, :h]
    state["tree"] = None
    if case["tree"]:
        rng = random.Random(seed)
        state["tree"] = torch.tensor([w for n in new for w in _tree(n, rng)], dtype=torch.int64, device="cuda")
    return state


# ---------------------------------------------------------------------------- the plain forms
def _positions(state, starts):
    """(block, offset) of every packed row: row i of sequence b is position starts[b] + i."""
    rows = torch.arange(state["total"], dtype=torch.int32, device="cuda")
    b = torch.searchsorted(state["cu"][1:], rows, right=True)
    pos = (starts[b] + rows - state["cu"][b]).long()
    return state["table"][b, pos // _BLOCK].long(), pos % _BLOCK


def _load(state, blk, off):
    """Dequantized fp32 K and V (n, KV, D) of the slots (blk, off)."""
    kind = _TYPES[state["fmt"]]
    kp, vp, sc = state["k_pages"].view(torch.uint8), state["v_pages"].view(torch.uint8), state["scales"]
    n, kv, d = blk.shape[0], vp.shape[1], vp.shape[2]
    k = kp[blk, :, off // 4, :, off % 4].reshape(n, kv, d).view(kind).float() * sc[blk, :, 0, off].unsqueeze(-1)
    v = vp[blk, :, :, off].contiguous().view(kind).float() * sc[blk, :, 1, off].unsqueeze(-1)
    return k, v


def _plain(state):
    if state["kind"] == "write":
        blk, off = _positions(state, state["lens"] - (state["cu"][1:] - state["cu"][:-1]))
        _store(state, blk, off, state["k"], state["v"])
        return {"k_pages": state["k_pages"], "v_pages": state["v_pages"], "scales": state["scales"]}
    if state["kind"] == "read":
        k, v = _load(state, *_positions(state, state["starts"]))
        return {"k": k.to(torch.bfloat16), "v": v.to(torch.bfloat16)}
    q = state["q"]
    h, d = q.shape[1:]
    out, at = [], 0
    for b, (t, n) in enumerate(zip(*state["host"])):
        pos = torch.arange(t, device="cuda")
        k, v = _load(state, state["table"][b].long()[pos // _BLOCK], pos % _BLOCK)
        kv = k.shape[1]
        x = q[at:at + n].float().view(n, kv, h // kv, d).permute(1, 2, 0, 3).reshape(kv, -1, d)  # rows: (head, token)
        k, v = k.permute(1, 2, 0).contiguous(), v.transpose(0, 1).contiguous()
        row = torch.arange(n, device="cuda")
        if state["tree"] is None:
            unseen = pos > t - n + row.unsqueeze(1)
        else:
            bit = (pos - (t - n)).clamp(min=0)
            unseen = (pos >= t - n) & ((state["tree"][at:at + n].unsqueeze(1) >> bit.clamp(max=63)) & 1 == 0)
        y = torch.empty_like(x)
        for i in range(kv):
            s = (x[i] @ k[i]).view(-1, n, t) / math.sqrt(d)
            s = s.masked_fill(unseen, -math.inf)
            p = torch.exp(s - s.amax(-1, keepdim=True))
            y[i] = ((p / p.sum(-1, keepdim=True)).view(-1, t) @ v[i])
        out.append(y.view(h, n, d).transpose(0, 1))
        at += n
    return torch.cat(out).to(torch.bfloat16)


# ---------------------------------------------------------------------------- one pass
_ops = None


def _library():
    global _ops
    if _ops is None:
        package = str(Path(__file__).resolve().parents[1] / "specdec-context-scaling_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        from specdec_amd.kernels import ops

        _ops = ops
    return _ops


def _framework(state):
    ops = _library()
    pages = (state["k_pages"], state["v_pages"], state["scales"])
    if state["kind"] == "write":
        ops.kv8_append(state["k"], state["v"], *pages, state["table"], state["cu"], state["lens"])
        return {"k_pages": pages[0], "v_pages": pages[1], "scales": pages[2]}
    if state["kind"] == "read":
        k, v = ops.kv8_gather(*pages, state["table"], state["cu"], state["starts"], state["total"])
        return {"k": k, "v": v}
    return ops.kv8_attention(state["q"], *pages, state["table"], state["cu"], state["lens"], state["max_new"], state["max_len"],
                             tree_mask=state["tree"])


def run(state):
    return _framework(state) if own else _plain(state)


# ---------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    x = prepare(case, seed)
    lens, new = x["host"]
    kv, d, fmt = case["kv"], case["dim"], case["fmt"]
    if case["kind"] == "write":
        scales, at = x["scales"].double(), 0
        for b, (t, n) in enumerate(zip(lens, new)):
            for j in range(n):
                p = t - n + j
                if p % _BLOCK and j:
                    continue
                block, m = int(x["table"][b, p // _BLOCK]), min(n - j, _BLOCK - p % _BLOCK)
                for part, rows in enumerate((x["k"], x["v"])):
                    s = rows[at + j:at + j + m].double().abs().max(-1).values / _LARGEST[fmt]
                    scales[block, :, part, p % _BLOCK:p % _BLOCK + m] = torch.where(s == 0, 1.0, s).t()
            at += n
        return {"k_pages": None, "v_pages": None, "scales": scales}  # codes are defined to the bit

    def dequantized(b, lo, hi):
        """Positions lo..hi-1 of sequence b: K and V (KV, n, D)."""
        blocks = x["table"][b, lo // _BLOCK:-(-hi // _BLOCK)].long()
        cut = slice(lo % _BLOCK, lo % _BLOCK + hi - lo)
        s = x["scales"][blocks].double().permute(1, 2, 0, 3).reshape(kv, 2, -1)[:, :, cut]
        kc = x["k_pages"].view(torch.uint8)[blocks].permute(1, 0, 2, 4, 3, 5).reshape(kv, -1, d)[:, cut].contiguous().view(_TYPES[fmt])
        vc = x["v_pages"].view(torch.uint8)[blocks].permute(1, 0, 3, 2).reshape(kv, -1, d)[:, cut].contiguous().view(_TYPES[fmt])
        return kc.double() * s[:, 0, :, None], vc.double() * s[:, 1, :, None]

    if case["kind"] == "read":
        pairs = [dequantized(b, t - n, t) for b, (t, n) in enumerate(zip(lens, new))]
        return {"k": torch.cat([k.transpose(0, 1) for k, _ in pairs]), "v": torch.cat([v.transpose(0, 1) for _, v in pairs])}
    out, at = torch.empty(x["q"].shape, dtype=torch.float64, device="cuda"), 0
    group = case["heads"] // kv
    for b, (t, n) in enumerate(zip(lens, new)):
        k, v = dequantized(b, 0, t)
        seen = torch.ones((n, t), dtype=torch.bool, device="cuda")
        if x["tree"] is None:
            seen[:, t - n:] = torch.ones((n, n), dtype=torch.bool, device="cuda").tril()
        else:
            words = x["tree"][at:at + n].tolist()
            seen[:, t - n:] = torch.tensor([[w >> j & 1 for j in range(n)] for w in words], dtype=torch.bool, device="cuda")
        for head in range(case["heads"]):
            scores = x["q"][at:at + n, head].double() @ k[head // group].t().contiguous() / math.sqrt(d)
            out[at:at + n, head] = torch.softmax(scores.masked_fill(~seen, -math.inf), -1) @ v[head // group].contiguous()
        at += n
    return out
