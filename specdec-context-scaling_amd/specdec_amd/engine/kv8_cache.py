"""Paged KV cache with K and V in 8 bits: the pool, allocator and block tables of
:class:`PagedKVCache` over the kv8 operators (``ops.kv8_append``, ``kv8_attention``,
``kv8_gather``).

    k_pages  (L, num_blocks, KV, 4, D/16, 4, 16)  float8_e4m3fn or int8
    v_pages  (L, num_blocks, KV, D, 16)           the same type, dimension-major per page
    scales   (L, num_blocks, KV, 2, 16)           fp32: K's 16 tokens, then V's

2 (D + 4) bytes per token and KV head, 528 of 776 per token and layer of the v_fp8 cache at 2 x 128.
No counterpart in the reference, whose caches keep K in BF16 or scale groups of 32 dimensions
(specdec/engine/model_self.py:300-320, 689-706).

Every call may give each sequence its own number of rows (``counts``): a step that decodes some
sequences, verifies drafted blocks or trees of others and takes a chunk of a third one's prompt is
one write and one attention per layer.

Recording into a HIP graph: with equal counts and lengths a recorded ``append_attend`` reads nothing
from the host but the row table, which an earlier call with the same counts has made; what it cannot
do inside a recording (add blocks, grow the pool, new tables) raises.  Pages and tables that a recording
used stay alive as long as the pool; once the pool has grown the graph has to be recorded again,
since what it writes does not reach the new pages.
"""
from __future__ import annotations

import torch

from .._native import SdvError
from ..kernels import ops
from .paged_cache import BLOCK, LayerPages, PagedKVCache, _no_recording, _recording, shape_carrier

FORMATS = {"fp8": torch.float8_e4m3fn, "int8": torch.int8}


class KV8Cache(PagedKVCache):
    """Page pool for ``num_layers`` layers and ``batch`` sequences, K and V in ``kv_format`` codes
    ("fp8" or "int8")."""

    def __init__(self, kv_heads: int, head_dim: int, *, kv_format: str = "fp8", num_layers: int = 1, batch: int = 1,
                 num_blocks: int | None = None, capacity_tokens: int = 256, device="cuda", seed: int | None = None,
                 growable: bool = True):
        if kv_format not in FORMATS:
            raise ValueError(f"kv_format must be one of {sorted(FORMATS)} (got {kv_format!r})")
        self.kv_format = kv_format
        super().__init__(kv_heads, head_dim, num_layers=num_layers, batch=batch, num_blocks=num_blocks,
                         capacity_tokens=capacity_tokens, device=device, seed=seed, growable=growable)
        self._cu: tuple | None = None     # ((counts, stream), device row table) of the last call
        self._lens: tuple | None = None   # ((lengths, stream), device array) of the last call
        self._served = (None, None)       # block table and K pages that _streams stands for
        self._streams: set = set()        # streams that the allocator knows to use them

    # ------------------------------------------------------------------ storage
    def _new_pages(self, nb: int):
        L, KV, D, t = self.num_layers, self.kv_heads, self.head_dim, FORMATS[self.kv_format]
        k = torch.zeros((L, nb, KV, 4, D // 16, 4, BLOCK), dtype=torch.uint8, device=self.device).view(t)
        v = torch.zeros((L, nb, KV, D, BLOCK), dtype=torch.uint8, device=self.device).view(t)
        s = torch.ones((L, nb, KV, 2, BLOCK), dtype=torch.float32, device=self.device)
        return k, v, s

    def _grow(self, min_blocks: int) -> None:
        _no_recording(self.device, "the page pool would grow")
        self._note_stream()  # the old pages are read on this stream, then dropped
        super()._grow(min_blocks)
        self._served = (None, None)

    @property
    def scales(self) -> torch.Tensor:
        return self.v_scales  # the pool's third page tensor: here K's scales as well

    def reserve_all(self, n_tokens: int, q_heads: int | None = None, q_len: int | None = None) -> None:
        """Page blocks and the device block table for the first n_tokens positions of every sequence,
        before recording a step up to them.  q_heads and q_len size nothing here: a call's workspace is
        its own, and a recording's is made with it."""
        for b in range(self.batch):
            self.reserve(b, n_tokens)
        self.block_table()

    # ------------------------------------------------------------------ tables
    # The row table and lengths of the last call are kept, for the stream that they were made on (a table
    # that is replaced goes back to that stream's memory).  Their contents never change, so a recorded
    # call may take those of an earlier call on any stream; it holds them.
    def _table(self, what: str, kept, values: tuple, build):
        """((values, stream), int32 tensor): the kept one where it serves, else a new one from the host."""
        recording = _recording(self.device)
        stream = ops._stream(self.device) if self.device.type == "cuda" else 0
        if kept is not None and kept[0][0] == values and (recording or kept[0][1] == stream):
            return kept
        _no_recording(self.device, f"{what} would be copied from the host")
        return (values, stream), torch.tensor(build(), dtype=torch.int32).to(self.device)

    def _rows(self, counts):
        """(counts, device row table (batch + 1,)) of `counts` rows per sequence."""
        counts = tuple(int(c) for c in counts)
        if len(counts) != self.batch or min(counts) < 0:
            raise ValueError(f"counts {counts} for a batch of {self.batch}")
        self._cu = self._table("a row table", self._cu, counts, lambda: [sum(counts[:b]) for b in range(self.batch + 1)])
        return counts, self._hold(self._cu[1])

    def _lengths(self, lengths):
        """(device lengths or None, longest): None where all are equal and not 0 (the operators take one
        length for all from 1 on)."""
        if len(lengths) != self.batch or min(lengths) < 0:
            raise ValueError(f"lengths {lengths} for a batch of {self.batch}")
        longest = max(lengths)
        if longest > 0 and all(n == longest for n in lengths):
            return None, longest
        self._lens = self._table("sequence lengths", self._lens, tuple(lengths), lambda: list(lengths))
        return self._hold(self._lens[1]), longest

    def _note_stream(self) -> None:
        """The block table and the pages are one for all streams, and go back to the memory of the stream
        that made them when they are replaced.  The allocator is told of every other stream that uses them,
        whose kernels it then waits for."""
        if self.device.type != "cuda":
            return
        if self._served[0] is not self._bt or self._served[1] is not self.k_pages:
            self._served, self._streams = (self._bt, self.k_pages), set()
        stream = ops._stream(self.device)
        if stream not in self._streams:
            self._streams.add(stream)
            on = torch.cuda.current_stream(self.device)
            for t in (self._bt, self.k_pages, self.v_pages, self.v_scales):
                if t is not None:
                    t.record_stream(on)

    def _operands(self, layer: int):
        """(K pages, V pages, scales, block table) of a call on the current stream."""
        table = self.block_table()
        if _recording(self.device):
            self._hold(table)
            self._hold_pages()
        else:
            self._note_stream()
        return (*self.layer(layer), table)

    # ------------------------------------------------------------------ kernels
    def write(self, layer: int, k_new: torch.Tensor, v_new: torch.Tensor, counts, starts=None) -> None:
        """Append counts[b] tokens to each sequence of one layer: k_new/v_new BF16 (sum(counts), KV, D),
        sequence after sequence.  Positions start at ``starts`` (default: the current lengths); the
        lengths become start + count."""
        starts = list(self.lengths) if starts is None else [int(s) for s in starts]
        counts, cu = self._rows(counts)
        ends = [s + c for s, c in zip(starts, counts)]
        if len(starts) != self.batch or min(starts) < 0:
            raise ValueError(f"starts {starts} for a batch of {self.batch}")
        if k_new.shape[0] != sum(counts):
            raise SdvError(f"k_new {tuple(k_new.shape)} does not hold {sum(counts)} rows")
        for b in range(self.batch):
            self.reserve(b, ends[b])
        if max(ends) > 0:
            lens, longest = self._lengths(ends)
            ops.kv8_append(k_new, v_new, *self._operands(layer), cu, lens, longest)
        self.lengths[:] = ends

    def append(self, layer: int, k_new: torch.Tensor, v_new: torch.Tensor, starts: list[int] | None = None):
        """write() of S tokens per sequence: k_new/v_new BF16 (B, S, KV, D)."""
        B, S = k_new.shape[:2]
        shape = (B * S, self.kv_heads, self.head_dim)
        self.write(layer, k_new.reshape(shape), v_new.reshape(shape), (S,) * B, starts)

    def prefill(self, layer: int, k_new: torch.Tensor, v_new: torch.Tensor, lengths: list[int],
                slots: torch.Tensor | None = None) -> torch.Tensor | None:
        """Whole prompts of different lengths: write() from position 0.  Slots come from the block table on
        the device: `slots`, which PagedKVCache's layers hand on, is returned as it came and not read."""
        self.write(layer, k_new, v_new, lengths, [0] * self.batch)
        return slots

    def attend(self, layer: int, q: torch.Tensor, *, counts=None, q_token_major: bool = False, lengths=None,
               scale: float | None = None, tree_mask: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of every sequence's last tokens over this layer's pages at the current lengths.

        q BF16 (sum(counts), H, D) with ``counts`` rows per sequence; without counts (B, H, S, D), or
        (B, S, H, D) with q_token_major, S rows of every sequence.  Returns out shaped like q.
        tree_mask (int64, one word a row): see ops.kv8_attention."""
        lengths = list(self.lengths) if lengths is None else [int(n) for n in lengths]
        rows, shape = q, None
        if counts is None:
            if q.dim() != 4 or q.shape[0] != self.batch:
                raise SdvError(f"q {tuple(q.shape)} is not (B = {self.batch}, H, S, D); with rows of different counts pass counts")
            rows = q if q_token_major else q.transpose(1, 2)
            shape = rows.shape
            counts = (shape[1],) * self.batch
            rows = rows.reshape(-1, *shape[2:])
        counts, cu = self._rows(counts)
        if rows.dim() != 3 or rows.shape[0] != sum(counts):
            raise SdvError(f"q {tuple(q.shape)} does not hold {sum(counts)} rows")
        if out is not None and out.shape != q.shape:
            raise SdvError(f"out {tuple(out.shape)} != q {tuple(q.shape)}")
        direct = out if shape is None else None
        lens, longest = self._lengths(lengths)
        got = ops.kv8_attention(rows, *self._operands(layer), cu, lens, max(1, *counts), max(1, longest), scale=scale,
                                tree_mask=tree_mask, out=direct)
        if shape is not None:
            got = got.view(shape)
            got = got if q_token_major else got.transpose(1, 2).contiguous()
            if out is not None:
                got = out.copy_(got)
        return got

    def append_attend(self, layer: int, q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, starts: list[int] | None = None, *,
                      counts=None, q_token_major: bool = False, scale: float | None = None, tree_mask: torch.Tensor | None = None,
                      out: torch.Tensor | None = None) -> torch.Tensor:
        """The layer's new tokens written, then attention over the context that includes them: k_new and
        v_new as for write() with ``counts``, else (B, S, KV, D); q as for attend()."""
        if counts is None:
            self.append(layer, k_new, v_new, starts)
        else:
            self.write(layer, k_new, v_new, counts, starts)
        return self.attend(layer, q, counts=counts, q_token_major=q_token_major, scale=scale, tree_mask=tree_mask, out=out)

    def read(self, layer: int, counts, starts=None):
        """(k, v) BF16 (sum(counts), KV, D): counts[b] tokens of each sequence from position starts[b]
        (default 0), dequantized."""
        counts, cu = self._rows(counts)
        starts = [0] * self.batch if starts is None else [int(s) for s in starts]
        if len(starts) != self.batch or any(s < 0 or s + c > n for s, c, n in zip(starts, counts, self.lengths)):
            raise ValueError(f"positions {starts} + {counts} outside the sequences' {self.lengths} tokens")
        _no_recording(self.device, "positions would be copied from the host")
        at = torch.tensor(starts, dtype=torch.int32).to(self.device)
        return ops.kv8_gather(*self._operands(layer), cu, at, sum(counts))

    def gather(self, layer: int, seq: int, n: int | None = None):
        """(k, v) BF16 (KV, T, D) of a sequence's first n tokens (default: all), dequantized."""
        n = self.lengths[seq] if n is None else n
        k, v = self.read(layer, [n if b == seq else 0 for b in range(self.batch)])
        return k.transpose(0, 1), v.transpose(0, 1)

    # ------------------------------------------------------------------ accounting
    def logical_bytes_per_token_layer(self) -> int:
        """K and V codes and an fp32 scale each: 528 B for KV=2, D=128."""
        return self.kv_heads * 2 * (self.head_dim + 4)

    def footprint(self) -> dict:
        tok = sum(self.lengths)
        kv8 = tok * self.num_layers * self.logical_bytes_per_token_layer()
        bf16 = tok * self.num_layers * self.kv_heads * 4 * self.head_dim
        scales = tok * self.num_layers * self.kv_heads * 8
        return {"tokens": tok, "kv8_bytes": kv8, "bf16_bytes": bf16, "saved_frac": 1 - kv8 / max(bf16, 1),
                "scale_frac_of_kv8": scales / max(kv8, 1),
                "pool_bytes": self.k_pages.numel() + self.v_pages.numel() + self.scales.numel() * 4}


class KV8LayerPages(LayerPages):
    """Handle of one engine layer's kv8 pages, carried in its cache dict under "pages"."""

    def layer_dict(self, length: int) -> dict:
        """{"fmt", "k", "k_scale", "v", "v_scale", "pages"} for a logical length of `length` tokens.  "fmt"
        is the engine's name of the switch that selects the paged packs."""
        p = self.pool
        B, KV, D, dev, t = p.batch, p.kv_heads, p.head_dim, p.device, FORMATS[p.kv_format]
        codes, scale = shape_carrier((B, KV, length, D), t, dev), shape_carrier((B, KV, length, 1), torch.float32, dev)
        return {"fmt": "v_fp8", "k": codes, "k_scale": scale, "v": codes, "v_scale": scale, "pages": self}

    def materialize(self, length: int) -> dict:
        """Dequantized copies {"k", "v"} BF16 (B, KV, T, D): the engine's BF16 cache format."""
        p = self.pool
        k, v = p.read(self.layer, [length] * p.batch)
        shape = (p.batch, length, p.kv_heads, p.head_dim)
        return {"k": k.view(shape).transpose(1, 2).contiguous(), "v": v.view(shape).transpose(1, 2).contiguous()}
