"""Torch-facing operators of the FP8-V path (mirror of specdec/kernels/ops.py).

torch is plumbing here: tensors provide device memory and the current HIP stream; every
computation runs in libsdv's gfx950 kernels through the C ABI (include/sdv.h).  Argument
problems raise ``RuntimeError`` (:class:`specdec_amd.SdvError`), the way the reference
op's TORCH_CHECKs do (specdec/kernels/cuda/attention.cu:245-262); an unknown backend raises
``ValueError`` as in specdec/kernels/ops.py:76.

Operators
---------
``quant_append``      kernel 1: V -> FP8 (per token and KV head max-abs/448 scale) plus the
                      BF16 K copy, written into page slots.
``paged_attention``   kernels 2/3: GQA decode / k+1-row verify over BF16 K + FP8 V pages.
``attention``         the reference op's signature ``attention(q, k, v, backend)``
                      (ops.py:67-76) over a contiguous v_fp8 cache: k BF16 (B,KV,T,D) and
                      v given as the (payload, scale) pair the engine stores.
                      One kernel packs the cache into pages first.
``kv8_append``        the 8-bit cache: new tokens' K and V quantized (fp8 or int8) into pages.
``kv8_gather``        the 8-bit cache read back into packed BF16 rows.
``kv8_attention``     ragged query rows (single tokens, verify blocks or trees, prompt chunks,
                      or all in one batch) over the 8-bit cache.
``kv8_shared_attention``  the same for sequences that begin with the same pages, read once for all.
``rope``              rotary positions of packed query and key rows (``rope_frequencies``: what it turns by).
``kv8_rope_append``   a step's rows in one launch: q rotated, K rotated and quantized, V quantized.
``copy_blocks``       whole page blocks of every layer copied, within a pool of either cache or to another.
``kv8_keep``          the 8-bit cache: an accepted path's tokens moved together, in every layer.
``fp8_encode``        elementwise fp32 -> E4M3FN on the device.
"""
from __future__ import annotations

import ctypes
import functools
import math
import os
import weakref

import torch

from .. import _native
from .._native import SdvError

BLOCK = _native.BLOCK_SIZE
_SCALE_MODES = {"div": _native.SCALE_DIV, "rcp": _native.SCALE_RCP}
_BACKENDS = ("hip", "cuda")  # "cuda" is what reference call sites pass (patch.py:107)

_WORKSPACES: dict = {}
# Cached workspaces replaced by larger ones that a call recorded into a HIP graph used (the
# graph still points at them).  A replacement is at least twice the size of the buffer it
# replaces, so these hold at most as many bytes as the current workspace of their stream.
_RETIRED: list = []
_RECORDED = weakref.WeakSet()  # cached workspaces handed to a call while its stream was recording
_READY: dict = {}  # id(tensor) -> weakref of workspaces whose sync prefix is known to be zero
# SDV_CHECK_SYNC=1: every paged_attention call reads its workspace's failure count afterwards
# and raises SdvError when a single-launch wait expired (synchronises; a debugging aid)
_CHECK_SYNC = os.environ.get("SDV_CHECK_SYNC", "0") not in ("", "0")


def _fail(msg: str):
    raise SdvError(msg, _native.SDV_ERR_SHAPE)


# The eager engine calls these operators once per layer and step, so their host cost is part of
# every decoded token: pointers go to ctypes as plain ints (the argtypes are c_void_p), the
# current stream comes from torch's raw query when it has one, and workspace sizes are cached.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(dev: torch.device) -> int:
    if _raw_stream is not None:
        return _raw_stream(dev.index if dev.index is not None else torch.cuda.current_device())
    return torch.cuda.current_stream(dev).cuda_stream


def _p(t):
    return t.data_ptr() if t is not None else None


def _need(t, name, dtypes, dev=None, ndim=None):
    if not isinstance(t, torch.Tensor):
        _fail(f"{name} must be a tensor")
    if not t.is_cuda:
        _fail(f"{name} must be on a HIP device (got {t.device})")
    if dev is not None and t.device != dev:
        _fail(f"{name} is on {t.device}, expected {dev}")
    if t.dtype not in dtypes:
        _fail(f"{name} must have dtype in {dtypes} (got {t.dtype})")
    if not t.is_contiguous():
        _fail(f"{name} must be contiguous")
    if ndim is not None and t.dim() not in ndim:
        _fail(f"{name} must have {ndim} dims (got {tuple(t.shape)})")


def _pages_dims(k_pages, v_pages, v_scales, layered: bool):
    lead = 1 if layered else 0
    if k_pages.dim() != 5 + lead or v_pages.dim() != 4 + lead or v_scales.dim() != 3 + lead:
        _fail(f"page tensors must be (..., num_blocks, KV, D/8, 16, 8) / (..., num_blocks, KV, D, 16) / "
              f"(..., num_blocks, KV, 16); got {tuple(k_pages.shape)}, {tuple(v_pages.shape)}, "
              f"{tuple(v_scales.shape)}")
    nb, kv, dc, blk, eight = k_pages.shape[lead:]
    d = dc * 8
    if blk != BLOCK or eight != 8 or tuple(v_pages.shape[lead:]) != (nb, kv, d, BLOCK) or \
            tuple(v_scales.shape[lead:]) != (nb, kv, BLOCK):
        _fail(f"page shapes disagree: k {tuple(k_pages.shape)}, v {tuple(v_pages.shape)}, s {tuple(v_scales.shape)}")
    if layered and not (k_pages.shape[0] == v_pages.shape[0] == v_scales.shape[0]):
        _fail("page tensors disagree on the layer count")
    return nb, kv, d


def _plain_pages(q, k_pages, v_pages, v_scales, block_table, seq_lens):
    """(blocks, KV heads, head_dim) when every tensor of a paged_attention call is what _need and
    _pages_dims ask for, tested in one pass (the engine calls it per layer and token); else None."""
    try:
        dev, ks = q.device, k_pages.shape
        lead = len(q.shape) - 4
        if lead not in (0, 1) or len(ks) != 5 + lead:
            return None
        nb, kv, dc, blk, eight = ks[lead:]
        front = ks[:lead + 2]
        if (blk == BLOCK and eight == 8 and v_pages.shape == (*front, dc * 8, BLOCK) and v_scales.shape == (*front, BLOCK)
                and q.is_cuda and k_pages.device == dev and v_pages.device == dev and v_scales.device == dev
                and block_table.device == dev and q.dtype is torch.bfloat16 and k_pages.dtype is torch.bfloat16
                and v_pages.dtype is torch.uint8 and v_scales.dtype is torch.float32 and block_table.dtype is torch.int32
                and len(block_table.shape) == 2 and q.is_contiguous() and k_pages.is_contiguous() and v_pages.is_contiguous()
                and v_scales.is_contiguous() and block_table.is_contiguous()
                and (seq_lens is None or (seq_lens.device == dev and seq_lens.dtype is torch.int32
                                          and len(seq_lens.shape) == 1 and seq_lens.is_contiguous()))):
            return nb, kv, dc * 8
    except AttributeError:  # not a tensor
        pass
    return None


def new_workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    """A fresh uint8 workspace of at least nbytes whose synchronisation prefix is zeroed
    (sdv_attention_workspace_init on the current stream)."""
    dev = torch.device(device)
    ws = torch.empty(max(int(nbytes), _native.SYNC_BYTES), dtype=torch.uint8, device=dev)
    _init_workspace(ws)
    return ws


def _init_workspace(ws: torch.Tensor) -> None:
    _native.check(_native.load().sdv_attention_workspace_init(_p(ws), ws.numel(), _stream(ws.device)),
                  "sdv_attention_workspace_init")
    key = id(ws)
    _READY[key] = weakref.ref(ws, lambda _r, key=key: _READY.pop(key, None))


def workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    """A cached uint8 workspace of at least nbytes on (device, current stream).

    A cached buffer that is too small is replaced by one at least twice its size.  The old
    buffer is freed, unless a call recorded into a HIP graph used it: the graph still points
    at it, so it is kept alive (at most the current buffer's size in all, by the doubling).
    Callers that record graphs should rather pass their own buffer (``workspace_tensor``)
    and keep it for the graph's lifetime.
    """
    dev = torch.device(device)
    key = (dev, _stream(dev))
    ws = _WORKSPACES.get(key)
    if ws is None or ws.numel() < nbytes:
        grow = 0
        if ws is not None:
            grow = 2 * ws.numel()
            if ws in _RECORDED:
                _RETIRED.append(ws)
        ws = new_workspace(dev, max(nbytes, grow, 1 << 20))
        _WORKSPACES[key] = ws
    if torch.cuda.is_current_stream_capturing():
        _RECORDED.add(ws)
    return ws


def single_launch_workgroups(num_layers: int, batch: int, q_heads: int, kv_heads: int, q_len: int, head_dim: int,
                             max_seq_len: int) -> int:
    """Workgroups of the single-launch kernel for these sizes on the current device, or 0
    when paged_attention takes the three-launch path."""
    return int(_native.load().sdv_attention_single_launch(num_layers, batch, q_heads, kv_heads, q_len, head_dim,
                                                           max_seq_len))


def _ws_args(ws: torch.Tensor | None):
    """(pointer, bytes, stream) of a workspace; None: the current device's no-allocation scratch
    (the workspace of sdv_paged_attention_noalloc), which the library names by a NULL pointer."""
    if ws is None:
        return None, 0, _stream(torch.device("cuda", torch.cuda.current_device()))
    return _p(ws), ws.numel(), _stream(ws.device)


def workspace_status(ws: torch.Tensor | None = None) -> tuple[int, bool]:
    """(failures, poisoned) of a workspace (sdv_attention_workspace_status; synchronises the
    current stream): failures = expired waits and refused calls of the single-launch path
    since the workspace was initialised; poisoned = graph-recorded calls are being refused
    until reset_workspace().  ws None: the no-allocation entry point's scratch on the current
    device."""
    fail, poison = ctypes.c_uint32(0), ctypes.c_uint32(0)
    ptr, n, st = _ws_args(ws)
    _native.check(_native.load().sdv_attention_workspace_status(ptr, n, ctypes.byref(fail), ctypes.byref(poison), st),
                  "sdv_attention_workspace_status")
    return int(fail.value), bool(poison.value)


def sync_errors(ws: torch.Tensor | None = None) -> int:
    """Expired waits and refused calls of the single-launch path recorded in a workspace
    (synchronises)."""
    return workspace_status(ws)[0]


def check_workspace(ws: torch.Tensor | None = None) -> None:
    """Raise SdvError when a single-launch call on this workspace could not complete (its
    outputs hold NaN where it failed); the reference raises every error (model_self.py:331-332).
    ws None: the no-allocation entry point's scratch on the current device."""
    fail, poison = workspace_status(ws)
    if fail or poison:
        raise SdvError(f"single-launch attention: {fail} wait(s) expired or call(s) refused on this workspace"
                       f"{' (graph-recorded calls poisoned)' if poison else ''}; outputs of the failed calls are NaN. "
                       f"Call ops.reset_workspace() before recording new graphs on it", _native.SDV_ERR_HIP)


def reset_workspace(ws: torch.Tensor | None = None) -> None:
    """Zero a workspace's synchronisation area (clears the failure count and the graph poison).
    ws None: the no-allocation entry point's scratch on the current device."""
    if ws is not None:
        _init_workspace(ws)
        return
    ptr, n, st = _ws_args(None)
    _native.check(_native.load().sdv_attention_workspace_init(ptr, n, st), "sdv_attention_workspace_init")


def set_wait_limit(polls: int) -> None:
    """Bound of the single launch's cross-workgroup waits for later calls (0: the default);
    tests use a tiny bound to drive the failure path."""
    _native.check(_native.load().sdv_attention_set_wait_limit(int(polls)), "sdv_attention_set_wait_limit")


@functools.lru_cache(maxsize=256)
def attention_workspace_bytes(num_layers: int, batch: int, q_heads: int, kv_heads: int, q_len: int,
                              head_dim: int, max_seq_len: int) -> int:
    n = _native.load().sdv_attention_workspace_size(num_layers, batch, q_heads, kv_heads, q_len,
                                                    head_dim, max_seq_len)
    if n == 0:
        _fail(f"unsupported attention sizes L={num_layers} B={batch} H={q_heads} KV={kv_heads} "
              f"S={q_len} D={head_dim} T={max_seq_len}")
    return int(n)


def quant_append(v_new: torch.Tensor, slot_mapping: torch.Tensor, k_pages: torch.Tensor,
                 v_pages: torch.Tensor, v_scales: torch.Tensor, k_new: torch.Tensor | None = None,
                 *, scale_mode: str = "div", tile_starts: torch.Tensor | None = None) -> None:
    """Quantize V to FP8 and write V (and BF16 K when given) into page slots, in place.

    v_new/k_new: BF16 (n_tokens, KV, D), or (L, n_tokens, KV, D) with layered pages.
    slot_mapping: int32 (n_tokens,), slot = block * 16 + offset, negative = skip.
    Pages: k (…, num_blocks, KV, D/8, 16, 8) BF16; v (…, num_blocks, KV, D, 16) uint8 or
    float8_e4m3fn; scales (…, num_blocks, KV, 16) fp32.
    tile_starts: optional int32 (n_tiles + 1,) on the device: tile i is rows
    [tile_starts[i], min(tile_starts[i] + 16, tile_starts[i+1])) (see varlen_tile_starts).
    """
    lib = _native.load()
    _need(v_new, "v_new", (torch.bfloat16,), ndim=(3, 4))
    dev = v_new.device
    layered = v_new.dim() == 4
    _need(k_pages, "k_pages", (torch.bfloat16,), dev)
    _need(v_pages, "v_pages", (torch.uint8, torch.float8_e4m3fn), dev)
    _need(v_scales, "v_scales", (torch.float32,), dev)
    _need(slot_mapping, "slot_mapping", (torch.int32,), dev, ndim=(1,))
    nb, kv, d = _pages_dims(k_pages, v_pages, v_scales, layered)
    L = v_new.shape[0] if layered else 1
    n_tokens = v_new.shape[-3]
    if tuple(v_new.shape[-2:]) != (kv, d) or slot_mapping.shape[0] != n_tokens:
        _fail(f"v_new {tuple(v_new.shape)} / slot_mapping {tuple(slot_mapping.shape)} do not match "
              f"pages (KV={kv}, D={d})")
    if layered and k_pages.shape[0] != L:
        _fail(f"v_new has {L} layers, pages have {k_pages.shape[0]}")
    if k_new is not None:
        _need(k_new, "k_new", (torch.bfloat16,), dev)
        if k_new.shape != v_new.shape:
            _fail(f"k_new {tuple(k_new.shape)} != v_new {tuple(v_new.shape)}")
    if scale_mode not in _SCALE_MODES:
        raise ValueError(f"scale_mode must be one of {sorted(_SCALE_MODES)}")
    # the kernel moves 16-byte pieces of each row; a view starting mid-row is copied first
    if v_new.data_ptr() % 16:
        v_new = v_new.clone()
    if k_new is not None and k_new.data_ptr() % 16:
        k_new = k_new.clone()
    per = lambda t: t[0].numel() if layered else 0  # noqa: E731  (elements per layer)
    if tile_starts is None:
        st = lib.sdv_quant_append(_p(v_new), _p(k_new), _p(slot_mapping), n_tokens, kv, d, d, L,
                                  per(v_new), _p(k_pages), _p(v_pages), _p(v_scales), nb,
                                  per(k_pages), per(v_pages), per(v_scales), _SCALE_MODES[scale_mode],
                                  _stream(dev))
        _native.check(st, "sdv_quant_append")
        return
    _need(tile_starts, "tile_starts", (torch.int32,), dev, ndim=(1,))
    if tile_starts.shape[0] < 1:
        _fail("tile_starts needs n_tiles + 1 entries")
    st = lib.sdv_quant_append_tiles(_p(v_new), _p(k_new), _p(slot_mapping), n_tokens, kv, d, d, L,
                                    per(v_new), _p(k_pages), _p(v_pages), _p(v_scales), nb,
                                    per(k_pages), per(v_pages), per(v_scales), _SCALE_MODES[scale_mode],
                                    _p(tile_starts), tile_starts.shape[0] - 1, _stream(dev))
    _native.check(st, "sdv_quant_append_tiles")


def varlen_slots(block_table: torch.Tensor, lengths: list[int], tiles: bool = True):
    """(slots, tile_starts) of whole prompts packed back to back: the slot of every row, from the
    block table int32 (B, max_blocks), and varlen_tile_starts(lengths) as a tensor (None without
    ``tiles``), in one kernel on the current stream (sdv_varlen_slots)."""
    _need(block_table, "block_table", (torch.int32,), ndim=(2,))
    n = len(lengths)
    if n > block_table.shape[0]:
        _fail(f"{n} lengths for a block table of {block_table.shape[0]} sequences")
    dev = block_table.device
    slots = torch.empty(sum(lengths), dtype=torch.int32, device=dev)
    table = torch.empty(sum(-(-x // BLOCK) for x in lengths) + 1, dtype=torch.int32, device=dev) if tiles else None
    if slots.numel() == 0:
        return slots, table.zero_() if tiles else None
    _native.check(_native.load().sdv_varlen_slots(_p(block_table), block_table.shape[1], (ctypes.c_int32 * n)(*lengths), n,
                                                  _p(slots), _p(table), _stream(dev)), "sdv_varlen_slots")
    return slots, table


def varlen_tile_starts(lengths: list[int], starts: list[int] | None = None) -> list[int]:
    """Tile table for a packed varlen input of sequences with `lengths` tokens whose first token
    lands at position `starts[b]` of its sequence (0: a whole prompt): tiles break where a page
    block begins, so every whole block is one tile.  n_tiles + 1 entries; the last is the
    total row count."""
    starts = starts or [0] * len(lengths)
    out, row = [], 0
    for n, p0 in zip(lengths, starts):
        if n < 0 or p0 < 0:
            raise ValueError("negative length or start position")
        i = 0
        while i < n:
            step = min(n - i, 16 - (p0 + i) % 16)
            out.append(row + i)
            i += step
        row += n
    out.append(row)
    return out


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, v_scales: torch.Tensor,
                    block_table: torch.Tensor, seq_lens: torch.Tensor, max_seq_len: int, *,
                    q_token_major: bool = False, out: torch.Tensor | None = None,
                    workspace_tensor: torch.Tensor | None = None,
                    phases: int = _native.PHASE_ALL,
                    append: tuple[torch.Tensor, torch.Tensor, torch.Tensor] | None = None,
                    scale_mode: str = "div") -> torch.Tensor:
    """GQA attention of q over paged BF16 K / FP8 V.

    q: BF16 (B, H, S, D) (or (B, S, H, D) with q_token_major=True); a leading layer dimension
    (L, ...) processes L layers in one launch with layered pages (L, num_blocks, ...).
    block_table int32 (B, max_blocks); seq_lens int32 (B,) = context length including the S
    new tokens, each <= max_seq_len, or None: every sequence has max_seq_len tokens (nothing
    to copy to the device, so the call can be recorded into a HIP graph).  Returns out shaped
    like q (BF16).
    ``phases`` (profiling) runs a subset of the three launches; see sdv_paged_attention_phases.
    ``append`` = (k_new, v_new, slot_mapping): first write the S new tokens of every sequence
    into the pages (as quant_append with ``scale_mode`` would; k_new/v_new BF16 (B*S, KV, D),
    or (L, B*S, KV, D) with layers, token b*S + i at position seq_lens[b] - S + i), in the same
    call (sdv_paged_attention_append); slot_mapping None takes each token's slot from the block
    table on the device.
    """
    lib = _native.load()
    dims = _plain_pages(q, k_pages, v_pages, v_scales, block_table, seq_lens)
    if dims is None:  # something unusual, or wrong: one check at a time says what
        _need(q, "q", (torch.bfloat16,), ndim=(4, 5))
        dev = q.device
        _need(k_pages, "k_pages", (torch.bfloat16,), dev)
        _need(v_pages, "v_pages", (torch.uint8, torch.float8_e4m3fn), dev)
        _need(v_scales, "v_scales", (torch.float32,), dev)
        _need(block_table, "block_table", (torch.int32,), dev, ndim=(2,))
        if seq_lens is not None:
            _need(seq_lens, "seq_lens", (torch.int32,), dev, ndim=(1,))
        dims = _pages_dims(k_pages, v_pages, v_scales, q.dim() == 5)
    nb, kv, d = dims
    dev = q.device
    layered = q.dim() == 5
    L = q.shape[0] if layered else 1
    if layered and k_pages.shape[0] != L:
        _fail(f"q has {L} layers, pages have {k_pages.shape[0]}")
    if q_token_major:
        B, S, H, Dq = q.shape[-4:]
    else:
        B, H, S, Dq = q.shape[-4:]
    if Dq != d or H % kv:
        _fail(f"q {tuple(q.shape)} does not match pages (KV={kv}, D={d})")
    if block_table.shape[0] != B or (seq_lens is not None and seq_lens.shape[0] != B):
        _fail(f"block_table {tuple(block_table.shape)} / seq_lens "
              f"{None if seq_lens is None else tuple(seq_lens.shape)} need batch {B}")
    max_seq_len = int(max_seq_len)
    if max_seq_len <= 0 or block_table.shape[1] * BLOCK < max_seq_len:
        _fail(f"max_seq_len {max_seq_len} must be in [1, 16 * max_blocks = {block_table.shape[1] * BLOCK}]")
    if out is None:
        out = torch.empty_like(q)
    else:
        _need(out, "out", (torch.bfloat16,), dev)
        if out.shape != q.shape:
            _fail(f"out {tuple(out.shape)} != q {tuple(q.shape)}")
    nbytes = attention_workspace_bytes(L, B, H, kv, S, d, max_seq_len)
    if workspace_tensor is None:
        workspace_tensor = workspace(dev, nbytes)
    else:
        _need(workspace_tensor, "workspace_tensor", (torch.uint8,), dev)
        if workspace_tensor.numel() < nbytes:
            _fail(f"workspace_tensor holds {workspace_tensor.numel()} bytes, {nbytes} needed")
        ref = _READY.get(id(workspace_tensor))
        if ref is None or ref() is not workspace_tensor:  # a caller's own buffer: zero its sync prefix once
            _init_workspace(workspace_tensor)
    per = lambda t: t[0].numel()  # noqa: E731
    k_ls, v_ls, s_ls = (per(k_pages), per(v_pages), per(v_scales)) if layered else (0, 0, 0)
    args = (_p(q), _p(k_pages), _p(v_pages), _p(v_scales), nb, k_ls, v_ls, s_ls,
            _p(block_table), block_table.shape[1], _p(seq_lens), L, B, H, kv, S, d, max_seq_len,
            int(bool(q_token_major)), _p(workspace_tensor), workspace_tensor.numel(), _p(out), _stream(dev))
    if append is not None:
        if phases != _native.PHASE_ALL:
            raise ValueError("append runs with the whole call (phases=PHASE_ALL)")
        if scale_mode not in _SCALE_MODES:
            raise ValueError(f"scale_mode must be one of {sorted(_SCALE_MODES)}")
        k_new, v_new, slots = append
        want = ((L,) if layered else ()) + (B * S, kv, d)
        for name, t in (("k_new", k_new), ("v_new", v_new)):
            _need(t, name, (torch.bfloat16,), dev)
            if tuple(t.shape) != want:
                _fail(f"{name} {tuple(t.shape)} != {want}")
        if slots is not None:
            _need(slots, "slot_mapping", (torch.int32,), dev, ndim=(1,))
            if slots.shape[0] != B * S:
                _fail(f"slot_mapping {tuple(slots.shape)} needs {B * S} entries")
        if k_new.data_ptr() % 16:
            k_new = k_new.clone()
        if v_new.data_ptr() % 16:
            v_new = v_new.clone()
        st = lib.sdv_paged_attention_append(*args[:-1], _p(k_new), _p(v_new), _p(slots), per(v_new) if layered else 0,
                                            _SCALE_MODES[scale_mode], args[-1])
        _native.check(st, "sdv_paged_attention_append")
        if _CHECK_SYNC:
            check_workspace(workspace_tensor)
        return out
    if phases == _native.PHASE_ALL:
        st = lib.sdv_paged_attention(*args)
    else:
        st = lib.sdv_paged_attention_phases(*args, int(phases))
    _native.check(st, "sdv_paged_attention")
    if _CHECK_SYNC:
        check_workspace(workspace_tensor)
    return out


def _plain(t, dtype, dev, shape) -> bool:
    """A contiguous device tensor of this type and shape whose first byte is 16-byte aligned."""
    return (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype is dtype and t.device == dev and t.shape == shape
            and t.is_contiguous() and t.data_ptr() % 16 == 0)


def append_attend_pages(q, k_new, v_new, pages, block_table, max_seq_len, B, S, H, KV, D, token_major, ws, scale_mode):
    """paged_attention(..., append=(k_new, v_new, None)) of one layer of a pool whose page
    addresses the caller has (`pages`: K, V, scales, blocks), every sequence max_seq_len tokens
    long; k_new/v_new (B, S, KV, D).  None when an argument is not the plain tensor that the fixed
    arguments of the call stand for: paged_attention then takes it, or says what is wrong."""
    dev = q.device
    if pages is None or scale_mode not in _SCALE_MODES or H % KV or \
            not _plain(q, torch.bfloat16, dev, (B, S, H, D) if token_major else (B, H, S, D)) or \
            not _plain(k_new, torch.bfloat16, dev, (B, S, KV, D)) or not _plain(v_new, torch.bfloat16, dev, (B, S, KV, D)) or \
            not (block_table.device == dev and block_table.dtype is torch.int32 and block_table.is_contiguous()) or \
            block_table.shape[0] != B or max_seq_len <= 0 or block_table.shape[1] * BLOCK < max_seq_len or ws.device != dev:
        return None
    out = torch.empty_like(q)
    kp, vp, sp, nb = pages
    st = _native.load().sdv_paged_attention_append(
        q.data_ptr(), kp, vp, sp, nb, 0, 0, 0, block_table.data_ptr(), block_table.shape[1], None, 1, B, H, KV, S, D,
        max_seq_len, int(token_major), ws.data_ptr(), ws.numel(), out.data_ptr(), k_new.data_ptr(), v_new.data_ptr(), None, 0,
        _SCALE_MODES[scale_mode], _stream(dev))
    if st:
        _native.check(st, "sdv_paged_attention_append")
    if _CHECK_SYNC:
        check_workspace(ws)
    return out


def quant_append_pages(v_new, k_new, slots, pages, tile_starts, KV, D, scale_mode, stream) -> bool:
    """quant_append of one layer of a pool whose page addresses the caller has; False (nothing
    done) when an argument is not the plain tensor that the call's fixed arguments stand for.
    `stream` is the current one of v_new's device (where `pages` is not None, the pool's)."""
    if pages is None or not isinstance(v_new, torch.Tensor) or v_new.dim() != 3 or scale_mode not in _SCALE_MODES:
        return False
    dev, n = v_new.device, v_new.shape[0]
    if not _plain(v_new, torch.bfloat16, dev, (n, KV, D)) or not _plain(k_new, torch.bfloat16, dev, (n, KV, D)) or \
            not _plain(slots, torch.int32, dev, (n,)) or tile_starts.device != dev:
        return False
    kp, vp, sp, nb = pages
    st = _native.load().sdv_quant_append_tiles(
        v_new.data_ptr(), k_new.data_ptr(), slots.data_ptr(), n, KV, D, D, 1, 0, kp, vp, sp, nb, 0, 0, 0,
        _SCALE_MODES[scale_mode], tile_starts.data_ptr(), tile_starts.shape[0] - 1, stream)
    if st:
        _native.check(st, "sdv_quant_append_tiles")
    return True


def pack_contiguous(k: torch.Tensor, v_payload: torch.Tensor, v_scale: torch.Tensor):
    """Copy a contiguous v_fp8 cache (B,KV,T,D) into pages (one copy; block b*nbps + j is
    tokens 16j.. of sequence b).  Returns (k_pages, v_pages, v_scales, block_table, seq_lens)."""
    B, KV, T, D = k.shape
    nbps = -(-T // BLOCK)
    Tp = nbps * BLOCK
    pad = Tp - T
    kk = torch.nn.functional.pad(k, (0, 0, 0, pad)) if pad else k
    vv = v_payload.view(torch.uint8)
    vv = torch.nn.functional.pad(vv, (0, 0, 0, pad)) if pad else vv
    ss = v_scale.reshape(B, KV, T)
    ss = torch.nn.functional.pad(ss, (0, pad), value=1.0) if pad else ss
    k_pages = (kk.reshape(B, KV, nbps, BLOCK, D // 8, 8).permute(0, 2, 1, 4, 3, 5)
               .reshape(B * nbps, KV, D // 8, BLOCK, 8).contiguous())
    v_pages = vv.reshape(B, KV, nbps, BLOCK, D).permute(0, 2, 1, 4, 3).reshape(B * nbps, KV, D, BLOCK).contiguous()
    v_scales = ss.reshape(B, KV, nbps, BLOCK).permute(0, 2, 1, 3).reshape(B * nbps, KV, BLOCK).contiguous()
    block_table = torch.arange(B * nbps, dtype=torch.int32, device=k.device).reshape(B, nbps)
    seq_lens = torch.full((B,), T, dtype=torch.int32, device=k.device)
    return k_pages, v_pages, v_scales, block_table, seq_lens


def attention(q: torch.Tensor, k: torch.Tensor, v, backend: str = "hip") -> torch.Tensor:
    """Reference op signature (specdec/kernels/ops.py:67-76) for the v_fp8 cache format.

    q (B,H,S,D) BF16; k (B,KV,T,D) BF16; v = (payload float8_e4m3fn (B,KV,T,D),
    scale fp32 (B,KV,T,1)) exactly as the reference cache stores it.  The FP8 payload is
    dequantized inside the kernel; row i of the S-row block sees keys j <= T - S + i.
    """
    if backend not in _BACKENDS:
        raise ValueError(backend)
    if isinstance(v, torch.Tensor):
        raise SdvError("the FP8-V backend needs v as (payload float8_e4m3fn, scale fp32); "
                       "BF16 V is the reference's 'fp16' cache format, which this library does not serve",
                       _native.SDV_ERR_UNSUPPORTED)
    payload, scale = v
    _need(q, "q", (torch.bfloat16,), ndim=(4,))
    _need(k, "k", (torch.bfloat16,), q.device, ndim=(4,))
    if payload.shape != k.shape or tuple(scale.shape) != tuple(k.shape[:3]) + (1,):
        _fail(f"v payload {tuple(payload.shape)} / scale {tuple(scale.shape)} do not match k {tuple(k.shape)}")
    return torch.ops.sdv.attention(q.contiguous(), k.contiguous(), payload.contiguous(), scale.contiguous())


def _contiguous_attention(q: torch.Tensor, k: torch.Tensor, payload: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """attention() over contiguous tensors: one kernel writes the cache into pages (the bytes
    pack_contiguous gives), and the paged kernels run over them.  The pages, scales and block table
    share one allocation."""
    lib = _native.load()
    _need(q, "q", (torch.bfloat16,), ndim=(4,))
    dev = q.device
    _need(k, "k", (torch.bfloat16,), dev, ndim=(4,))
    if payload.element_size() != 1:
        _fail(f"v payload must hold one byte per element (got {payload.dtype})")
    _need(payload, "v payload", (payload.dtype,), dev)
    _need(scale, "v scale", (torch.float32,), dev)
    (B, H, S, D), (Bk, KV, T, Dk) = q.shape, k.shape
    if Bk != B or Dk != D or KV <= 0 or H % KV:
        _fail(f"q {tuple(q.shape)} does not match k {tuple(k.shape)}")
    if T <= 0:
        _fail(f"k {tuple(k.shape)} holds no tokens")
    nbytes = attention_workspace_bytes(1, B, H, KV, S, D, T)
    # the kernel moves 16-byte pieces of K and 4-byte pieces of V
    if k.data_ptr() % 16:
        k = k.clone()
    if payload.data_ptr() % 4:
        payload = payload.clone()
    nb = -(-T // BLOCK)
    pages = B * nb
    k_bytes, v_bytes, s_bytes = pages * KV * BLOCK * D * 2, pages * KV * BLOCK * D, pages * KV * BLOCK * 4
    buf = torch.empty(k_bytes + v_bytes + s_bytes + pages * 4, dtype=torch.uint8, device=dev)
    kp = buf.data_ptr()
    vp = kp + k_bytes
    sp = vp + v_bytes
    bt = sp + s_bytes
    st = _stream(dev)
    _native.check(lib.sdv_pack_contiguous(_p(k), _p(payload), _p(scale), B, KV, T, D, kp, vp, sp, bt, st),
                  "sdv_pack_contiguous")
    out = torch.empty_like(q)
    ws = workspace(dev, nbytes)
    _native.check(lib.sdv_paged_attention(_p(q), kp, vp, sp, pages, 0, 0, 0, bt, nb, None, 1, B, H, KV, S, D, T, 0,
                                          _p(ws), ws.numel(), _p(out), st), "sdv_paged_attention")
    if _CHECK_SYNC:
        check_workspace(ws)
    return out


def fp8_encode(x: torch.Tensor) -> torch.Tensor:
    """fp32 -> uint8 E4M3FN codes (RNE; NaN beyond 464), computed on the device."""
    _need(x, "x", (torch.float32,))
    out = torch.empty(x.shape, dtype=torch.uint8, device=x.device)
    _native.check(_native.load().sdv_fp8_encode(_p(x), _p(out), x.numel(), _stream(x.device)), "sdv_fp8_encode")
    return out


# ---------------------------------------------------------------------------- the 8-bit KV cache
_KV8_FORMATS = {torch.float8_e4m3fn: _native.KV8_FP8, torch.int8: _native.KV8_INT8}
_get_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _kv8_call(fn, what: str, dev: torch.device, *args) -> None:
    """fn(*args, stream) on dev's current stream, with dev the current device."""
    if dev.index is not None and dev.index != _get_device():
        with torch.cuda.device(dev):
            st = fn(*args, _stream(dev))
    else:
        st = fn(*args, _stream(dev))
    if st:
        _native.check(st, what)


def _kv8_device(k_pages) -> torch.device:
    if not isinstance(k_pages, torch.Tensor):
        _fail("k_pages must be a tensor")
    return k_pages.device


def _kv8_pages(k_pages, v_pages, scales, block_table, dev):
    """(blocks, KV heads, head_dim, format) of a layer's kv8 pages, checked."""
    try:
        nb, kv, four, dc, r, j = k_pages.shape
        shapes = (four, r, j) == (4, 4, 16) and v_pages.shape == (nb, kv, dc * 16, BLOCK) and scales.shape == (nb, kv, 2, BLOCK)
        fmt = _KV8_FORMATS.get(k_pages.dtype)
        if (shapes and fmt is not None and v_pages.dtype is k_pages.dtype and scales.dtype is torch.float32
                and block_table.dtype is torch.int32 and block_table.dim() == 2 and dev.type == "cuda" and k_pages.device == dev
                and v_pages.device == dev and scales.device == dev and block_table.device == dev and k_pages.is_contiguous()
                and v_pages.is_contiguous() and scales.is_contiguous() and block_table.is_contiguous()):
            return nb, kv, dc * 16, fmt
    except (AttributeError, ValueError):  # not a tensor, or of another rank
        pass
    types = tuple(_KV8_FORMATS)
    _need(k_pages, "k_pages", types, dev, (6,))
    _need(v_pages, "v_pages", (k_pages.dtype,), dev, (4,))
    _need(scales, "scales", (torch.float32,), dev, (4,))
    _need(block_table, "block_table", (torch.int32,), dev, (2,))
    _fail(f"kv8 pages must be (num_blocks, KV, 4, D/16, 4, 16) / (num_blocks, KV, D, 16) / (num_blocks, KV, 2, 16); got "
          f"{tuple(k_pages.shape)}, {tuple(v_pages.shape)}, {tuple(scales.shape)}")


def _kv8_rows(t, name, dev, heads=None, dim=None, write=False):
    """(tensor, elements between tokens) of packed BF16 rows (total, heads, D).  Rows may lie any
    multiple of 8 elements apart; what else the kernels cannot take as it lies is copied (an output:
    refused)."""
    if not isinstance(t, torch.Tensor):
        _fail(f"{name} must be a tensor")
    if t.dtype is not torch.bfloat16 or t.device != dev or t.dim() != 3:
        _fail(f"{name} must be (rows, heads, D) bfloat16 on {dev} (got {tuple(t.shape)} {t.dtype} on {t.device})")
    n, h, d = t.shape
    if (heads is not None and h != heads) or (dim is not None and d != dim):
        _fail(f"{name} {tuple(t.shape)} does not match {heads} heads of {dim}")
    row, head, one = t.stride()
    if n <= 1:
        row = h * d
    if one == 1 and (head == d or h == 1) and row >= h * d and row % 8 == 0 and t.data_ptr() % 16 == 0:
        return t, row
    if write:
        _fail(f"{name} must have contiguous heads and tokens a multiple of 8 elements apart, 16-byte aligned (strides {t.stride()})")
    return t.clone(memory_format=torch.contiguous_format), h * d


def _kv8_ints(t, name, dev, n, dtype=torch.int32):
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.device == dev and t.shape == (n,) and t.is_contiguous()):
        _need(t, name, (dtype,), dev, (1,))
        _fail(f"{name} {tuple(t.shape)} needs {n} entries")
    return t.data_ptr()


def kv8_append(k_new: torch.Tensor, v_new: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, scales: torch.Tensor,
               block_table: torch.Tensor, cu_rows: torch.Tensor, seq_lens: torch.Tensor | None, max_seq_len: int = 0) -> None:
    """Quantize new tokens' K and V and write them into the 8-bit cache, in place.

    k_new/v_new: BF16 (total, KV, D), the sequences' rows one after another; parts of a wider
    projection output may be passed as they lie.  Pages of one layer: k (num_blocks, KV, 4, D/16, 4,
    16) and v (num_blocks, KV, D, 16), both float8_e4m3fn or int8, scales (num_blocks, KV, 2, 16)
    fp32 (K's, then V's).  block_table int32 (B, max_blocks).  cu_rows int32 (B + 1,): sequence b's
    rows are cu_rows[b] .. cu_rows[b+1] - 1; they are its last positions, seq_lens int32 (B,) being
    the lengths with them, or None: every sequence has max_seq_len tokens.  Rows behind cu_rows[B]
    are not touched; rows whose position the block table does not hold are skipped.  No two rows of a
    call may have the same slot.
    """
    st = _native.binding().append(k_new, v_new, k_pages, v_pages, scales, block_table, cu_rows, seq_lens, max_seq_len)
    if st is not None:
        if st:
            _native.check(st, "sdv_kv8_append")
        return
    # something unusual, or wrong: copied where it may be, else named
    dev = _kv8_device(k_pages)
    nb, kv, d, fmt = _kv8_pages(k_pages, v_pages, scales, block_table, dev)
    k_new, ks = _kv8_rows(k_new, "k_new", dev, kv, d)
    v_new, vs = _kv8_rows(v_new, "v_new", dev, kv, d)
    if k_new.shape[0] != v_new.shape[0]:
        _fail(f"k_new {tuple(k_new.shape)} != v_new {tuple(v_new.shape)}")
    B, mb = block_table.shape
    if seq_lens is None and max_seq_len <= 0:
        _fail("seq_lens None needs max_seq_len")
    cu = _kv8_ints(cu_rows, "cu_rows", dev, B + 1)
    lens = None if seq_lens is None else _kv8_ints(seq_lens, "seq_lens", dev, B)
    if k_new.shape[0] == 0:
        return
    _kv8_call(_native.load().sdv_kv8_append, "sdv_kv8_append", dev, k_new.data_ptr(), v_new.data_ptr(), ks, vs, k_new.shape[0],
              k_pages.data_ptr(), v_pages.data_ptr(), scales.data_ptr(), nb, fmt, block_table.data_ptr(), mb,
              cu, lens, int(max_seq_len), B, kv, d)


def kv8_gather(k_pages: torch.Tensor, v_pages: torch.Tensor, scales: torch.Tensor, block_table: torch.Tensor,
               cu_rows: torch.Tensor, starts: torch.Tensor, total_rows: int, *, k_out: torch.Tensor | None = None,
               v_out: torch.Tensor | None = None):
    """Read the 8-bit cache back: (k, v) BF16 (total_rows, KV, D), each value bf16(code * scale).

    Rows cu_rows[b] .. cu_rows[b+1] - 1 (int32 (B + 1,)) are positions starts[b], starts[b] + 1, ...
    (int32 (B,)) of sequence b; positions that the block table does not hold read as zeros, rows
    behind cu_rows[B] are not written.  k_out/v_out: write there instead (tokens may lie any
    multiple of 8 elements apart).  The other arguments as for kv8_append.
    """
    if k_out is None and v_out is None:
        got = _native.binding().gather(k_pages, v_pages, scales, block_table, cu_rows, starts, total_rows)
        if got is not None:
            if got.__class__ is int:
                _native.check(got, "sdv_kv8_gather")
            return got
    dev = _kv8_device(k_pages)
    nb, kv, d, fmt = _kv8_pages(k_pages, v_pages, scales, block_table, dev)
    total_rows = int(total_rows)
    if total_rows < 0:
        _fail(f"total_rows {total_rows} is negative")
    B, mb = block_table.shape
    outs = []
    for t, name in ((k_out, "k_out"), (v_out, "v_out")):
        if t is None:
            t = torch.empty((total_rows, kv, d), dtype=torch.bfloat16, device=dev)
        outs.append((*_kv8_rows(t, name, dev, kv, d, write=True), name))
        if t.shape[0] != total_rows:
            _fail(f"{name} {tuple(t.shape)} needs {total_rows} rows")
    (k, ks, _), (v, vs, _) = outs
    cu, first = _kv8_ints(cu_rows, "cu_rows", dev, B + 1), _kv8_ints(starts, "starts", dev, B)
    if total_rows == 0:
        return k, v
    _kv8_call(_native.load().sdv_kv8_gather, "sdv_kv8_gather", dev, k_pages.data_ptr(), v_pages.data_ptr(), scales.data_ptr(), nb,
              fmt, block_table.data_ptr(), mb, cu, first, B, total_rows, kv, d, k.data_ptr(), v.data_ptr(), ks, vs)
    return k, v


@functools.lru_cache(maxsize=256)
def kv8_attention_workspace_bytes(batch: int, total_rows: int, q_heads: int, kv_heads: int, head_dim: int, max_q_len: int,
                                  max_seq_len: int) -> int:
    n = _native.load().sdv_kv8_attention_workspace_size(batch, total_rows, q_heads, kv_heads, head_dim, max_q_len, max_seq_len)
    if n == 0:
        _fail(f"unsupported kv8 attention sizes B={batch} rows={total_rows} H={q_heads} KV={kv_heads} D={head_dim} "
              f"max_q_len={max_q_len} max_seq_len={max_seq_len}")
    return int(n)


def kv8_workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    """A fresh workspace for kv8_attention of at least nbytes, its count area zeroed."""
    ws = torch.empty(max(int(nbytes), _native.KV8_SYNC_BYTES), dtype=torch.uint8, device=device)
    ws[:_native.KV8_SYNC_BYTES].zero_()
    return ws


def kv8_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, scales: torch.Tensor, block_table: torch.Tensor,
                  cu_rows: torch.Tensor, seq_lens: torch.Tensor | None, max_q_len: int, max_seq_len: int, *,
                  scale: float | None = None, tree_mask: torch.Tensor | None = None, out: torch.Tensor | None = None,
                  workspace_tensor: torch.Tensor | None = None) -> torch.Tensor:
    """GQA attention of ragged query rows over the 8-bit cache; returns BF16 (total, H, D).

    q BF16 (total, H, D): sequence b's rows are cu_rows[b] .. cu_rows[b+1] - 1, its last positions
    (seq_lens[b] tokens in all, <= max_seq_len; None: max_seq_len for every sequence).  Any row counts
    may stand in one batch; max_q_len is the largest.  A row sees the keys up to its own position;
    with tree_mask (int64 or uint64 (total,), max_q_len <= 64) the context before the new tokens and
    the new tokens j whose bit j of its mask is set.  scale: default 1 / sqrt(D).  A row that sees
    nothing is 0, one whose scores are all -inf (an infinite q) NaN; rows behind cu_rows[B] are not
    written.  out (like q; tokens may lie any multiple of 8 elements apart) and workspace_tensor (uint8, of
    kv8_attention_workspace_bytes; not for calls that may overlap on the device, nor for host threads that
    may be in a call with it at once) are the caller's own.  The pages as for kv8_append.

    A call with more than 32 rows per sequence and KV head (by max_q_len) that is not a short one holds V
    relative to the largest V scale of a row tile's keys, those that a row does not see and rows of zeros (scale 1)
    among them: beside the roundings to 11 bits an output is off by up to 2^-30 of that scale, whatever its own
    size, and by up to 2^-32 of the sum of |V| over its keys, divided by that of their exponentials.
    """
    if workspace_tensor is None:
        got = _native.binding().attention(q, k_pages, v_pages, scales, block_table, cu_rows, seq_lens, max_q_len, max_seq_len, scale,
                                          tree_mask, out)
        if got is not None:
            if got.__class__ is int:
                _native.check(got, "sdv_kv8_attention")
            return got
    dev = _kv8_device(k_pages)
    nb, kv, d, fmt = _kv8_pages(k_pages, v_pages, scales, block_table, dev)
    q, q_row = _kv8_rows(q, "q", dev, None, d)
    total, H = q.shape[:2]
    if H == 0 or H % kv:
        _fail(f"q {tuple(q.shape)} does not match pages (KV={kv}, D={d})")
    B, mb = block_table.shape
    max_q_len, max_seq_len = int(max_q_len), int(max_seq_len)
    cu = _kv8_ints(cu_rows, "cu_rows", dev, B + 1)
    lens = None if seq_lens is None else _kv8_ints(seq_lens, "seq_lens", dev, B)
    tree = None
    if tree_mask is not None:
        if max_q_len > 64:
            _fail(f"a tree mask holds 64 tokens (max_q_len {max_q_len})")
        tree = _kv8_ints(tree_mask, "tree_mask", dev, total, torch.uint64 if tree_mask.dtype is torch.uint64 else torch.int64)
    if out is None:
        out = torch.empty((total, H, d), dtype=torch.bfloat16, device=dev)
        out_row = H * d
    else:
        out, out_row = _kv8_rows(out, "out", dev, H, d, write=True)
        if out.shape[0] != total:
            _fail(f"out {tuple(out.shape)} != q {tuple(q.shape)}")
    nbytes = kv8_attention_workspace_bytes(B, total, H, kv, d, max_q_len, max_seq_len)
    if workspace_tensor is not None:
        _need(workspace_tensor, "workspace_tensor", (torch.uint8,), dev)
        if workspace_tensor.numel() < nbytes:
            _fail(f"workspace_tensor holds {workspace_tensor.numel()} bytes, {nbytes} needed")
        if workspace_tensor.data_ptr() % 256:
            _fail("workspace_tensor must be 256-byte aligned")
        if total:  # it may have held anything since the last call
            workspace_tensor[:_native.KV8_SYNC_BYTES].zero_()
    if total == 0:
        return out
    scale = d ** -0.5 if scale is None else float(scale)
    if workspace_tensor is None:  # again, as a plain case; what still is none (a tensor subclass) has a workspace to itself
        got = _native.binding().attention(q, k_pages, v_pages, scales, block_table, cu_rows, seq_lens, max_q_len, max_seq_len, scale,
                                          tree_mask, out)
        if got is not None:
            if got.__class__ is int:
                _native.check(got, "sdv_kv8_attention")
            return got
        workspace_tensor = kv8_workspace(dev, nbytes)
    _kv8_call(_native.load().sdv_kv8_attention, "sdv_kv8_attention", dev, q.data_ptr(), q_row, k_pages.data_ptr(),
              v_pages.data_ptr(), scales.data_ptr(), nb, fmt, block_table.data_ptr(), mb, cu, lens, tree, B, total, H, kv, d,
              max_q_len, max_seq_len, scale, workspace_tensor.data_ptr(),
              workspace_tensor.numel(), out.data_ptr(), out_row)
    return out


def kv8_shared_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, scales: torch.Tensor, block_table: torch.Tensor,
                         cu_rows: torch.Tensor, seq_lens: torch.Tensor | None, max_q_len: int, max_seq_len: int, cu_groups: torch.Tensor,
                         prefix_lens: torch.Tensor, max_prefix_len: int, *, scale: float | None = None,
                         tree_mask: torch.Tensor | None = None, tile_rows: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
    """kv8_attention for sequences that begin with the same pages, whose shared keys are read and computed once for each group of them.

    cu_groups int32 (groups + 1,): group g is sequences cu_groups[g] .. cu_groups[g+1] - 1; a sequence may be in none.  prefix_lens
    int32 (B,), the same for all of a group and at most each one's context before its new tokens (0 for a sequence in no group): so
    many first tokens, taken down to whole blocks, are blocks that the table names alike for all of the group.  Every row of the group
    sees them all, then its own sequence's keys from there on.  max_prefix_len bounds them.  The other arguments, and the result, are
    kv8_attention's, to its roundings: tiles of 32 rows hold the exponentials in 16 bits and the codes exactly, as it does for few rows,
    those of 128 hold the exponentials, and V with its scale, in FP16, as it does for many.

    tile_rows: rows of the group that a workgroup has at a time, 32 or 128; 0: whichever is faster for one group of these sizes, or
    kv8_attention where that is faster than both (short prefixes, few sequences, more than 64 rows of a sequence and KV head).  With
    few sequences in groups, or prefixes of very different lengths, kv8_attention may be faster than that choice.
    """
    got = _native.binding().shared(q, k_pages, v_pages, scales, block_table, cu_rows, seq_lens, max_q_len, max_seq_len, cu_groups,
                                   prefix_lens, max_prefix_len, scale, tree_mask, tile_rows, out)
    if got is not None:
        if got.__class__ is int:
            _native.check(got, "sdv_kv8_shared_attention")
        return got
    if tile_rows not in (0, 32, 128):
        raise ValueError(f"tile_rows must be 0, 32 or 128 (got {tile_rows})")
    dev = _kv8_device(k_pages)
    nb, kv, d, fmt = _kv8_pages(k_pages, v_pages, scales, block_table, dev)
    q, q_row = _kv8_rows(q, "q", dev, None, d)
    total, H = q.shape[:2]
    if H == 0 or H % kv:
        _fail(f"q {tuple(q.shape)} does not match pages (KV={kv}, D={d})")
    B, mb = block_table.shape
    max_q_len, max_seq_len, max_prefix_len = int(max_q_len), int(max_seq_len), int(max_prefix_len)
    cu = _kv8_ints(cu_rows, "cu_rows", dev, B + 1)
    lens = None if seq_lens is None else _kv8_ints(seq_lens, "seq_lens", dev, B)
    _need(cu_groups, "cu_groups", (torch.int32,), dev, (1,))
    groups = cu_groups.shape[0] - 1
    if not 0 <= groups <= B:
        _fail(f"cu_groups {tuple(cu_groups.shape)} needs 1 to {B + 1} entries")
    prefix = _kv8_ints(prefix_lens, "prefix_lens", dev, B)
    tree = None
    if tree_mask is not None:
        if max_q_len > 64:
            _fail(f"a tree mask holds 64 tokens (max_q_len {max_q_len})")
        tree = _kv8_ints(tree_mask, "tree_mask", dev, total, torch.uint64 if tree_mask.dtype is torch.uint64 else torch.int64)
    if out is None:
        out = torch.empty((total, H, d), dtype=torch.bfloat16, device=dev)
        out_row = H * d
    else:
        out, out_row = _kv8_rows(_same_rows(out, total, "out"), "out", dev, H, d, write=True)
    if not 0 <= max_prefix_len <= mb * BLOCK:
        _fail(f"max_prefix_len {max_prefix_len} outside the table's {mb} blocks")
    lib = _native.load()
    sizes = (B, groups, total, H, kv, d, max_q_len, max_seq_len, max_prefix_len)
    tile = tile_rows or lib.sdv_kv8_shared_attention_tile_rows(*sizes)
    if tile == 0:
        return kv8_attention(q, k_pages, v_pages, scales, block_table, cu_rows, seq_lens, max_q_len, max_seq_len, scale=scale,
                             tree_mask=tree_mask, out=out)
    nbytes = lib.sdv_kv8_shared_attention_workspace_size(*sizes, tile)
    if nbytes == 0:
        _fail(f"unsupported sizes B={B} groups={groups} rows={total} H={H} KV={kv} D={d} max_q_len={max_q_len} "
              f"max_seq_len={max_seq_len} max_prefix_len={max_prefix_len}")
    if total == 0:
        return out
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _kv8_call(lib.sdv_kv8_shared_attention, "sdv_kv8_shared_attention", dev, q.data_ptr(), q_row, k_pages.data_ptr(), v_pages.data_ptr(),
              scales.data_ptr(), nb, fmt, block_table.data_ptr(), mb, cu, lens, tree, cu_groups.data_ptr(), prefix, B, groups, total, H, kv,
              d, max_q_len, max_seq_len, max_prefix_len, tile, d ** -0.5 if scale is None else float(scale), ws.data_ptr(), nbytes,
              out.data_ptr(), out_row)
    return out


# ---------------------------------------------------------------------------- positions and page moves
def rope_frequencies(head_dim: int, base: float = 1000000.0, *, rotary_dim: int | None = None, scaling: dict | None = None,
                     device="cuda") -> tuple[torch.Tensor, float]:
    """(inv_freq, scale) for ``rope`` and ``kv8_rope_append``: float64 (rotary_dim / 2,) radians per position, base^(-2i / rotary_dim)
    for pair i, and what cos and sin are multiplied by.

    scaling stretches a context: {"type": "linear", "factor": f} divides all frequencies by f; {"type": "ntk", "factor": f}
    raises the base so that the slowest pair's is divided by f and the fastest stays; {"type": "yarn", "factor": f,
    "original": n, "slow": 1, "fast": 32} (Peng et al., arXiv:2309.00071) divides those that turn less than `slow` times in n
    positions, leaves those that turn more than `fast` times, goes over between them in proportion to the turns, and has scale
    0.1 ln f + 1.  That is the paper's ramp; models that go over in proportion to the pair's number, between rounded bounds, have other
    frequencies in between.  Any float64 tensor will do: those of a model's own configuration serve as they are.
    """
    r = head_dim if rotary_dim is None else int(rotary_dim)
    if not 0 < r <= head_dim or r % 16:
        raise ValueError(f"rotary_dim must be a multiple of 16 up to {head_dim} (got {r})")
    if base <= 0:
        raise ValueError(f"base must be positive (got {base})")
    scaling = dict(scaling or {"type": "none"})
    kind, factor, scale = scaling.pop("type", None), float(scaling.pop("factor", 1.0)), 1.0
    if factor < 1:
        raise ValueError(f"factor must be at least 1 (got {factor})")
    more = {k: float(scaling.pop(k, v)) for k, v in {"original": 0.0, "slow": 1.0, "fast": 32.0}.items()} if kind == "yarn" else {}
    if scaling:
        raise ValueError(f"scaling {kind!r} does not take {sorted(scaling)}")
    if kind == "ntk":
        base = base * factor ** (r / (r - 2))
    inv = base ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)
    if kind == "linear":
        inv = inv / factor
    elif kind == "yarn":
        if more["original"] <= 0 or not more["slow"] < more["fast"]:
            raise ValueError("yarn needs the original context length, and slow < fast")
        turns = more["original"] * inv / (2 * math.pi)
        stays = ((turns - more["slow"]) / (more["fast"] - more["slow"])).clamp(0, 1)
        inv = inv / factor * (1 - stays) + inv * stays
        scale = 0.1 * math.log(factor) + 1
    elif kind not in ("none", "ntk"):
        raise ValueError(f"scaling type must be linear, ntk or yarn (got {kind!r})")
    return inv.to(device), scale


def _frequencies(inv_freq, dev, d) -> int:
    """The rotated dimensions that inv_freq stands for, checked."""
    _need(inv_freq, "inv_freq", (torch.float64,), dev, (1,))
    n = 2 * inv_freq.shape[0]
    if not 0 < n <= d or n % 16:
        _fail(f"inv_freq {tuple(inv_freq.shape)} stands for {n} dimensions: a multiple of 16 up to {d} is needed")
    return n


def _same_rows(t, n, name):
    if t.shape[0] != n:
        _fail(f"{name} {tuple(t.shape)} needs {n} rows")
    return t


def rope(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor, *, interleaved: bool = False,
         scale: float = 1.0, inverse: bool = False, q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None):
    """Rotary positions: (q, k) rotated, BF16 (rows, heads, D) each (k may be None), D 64 or 128.

    q and k: rows of any stride that is a multiple of 8 elements (parts of a projection's output as they lie).  positions int32
    (rows,).  inv_freq float64 (r/2,), scale: see rope_frequencies.  Of a head's first r dimensions pair i is (i, i + r/2), or
    (2i, 2i + 1) if interleaved: it becomes scale (x cos t - y sin t, x sin t + y cos t), t = position * inv_freq[i], computed
    in fp32 from an angle in 64 bits and rounded once.  inverse: rotated back (the transpose).  Gradients of q and k are those
    of the results rotated back by the same angles, BF16 like them (recorded into a HIP graph only of tensors that the recording
    makes, not of leaves).  q_out and k_out, which may be q and k themselves (no other
    overlap): written there, outside autograd.
    """
    if q_out is None and k_out is None:
        got = _native.binding().rope(q, k, positions, inv_freq, interleaved, scale, inverse)
        if got is not None:
            if got.__class__ is int:
                _native.check(got, "sdv_rope")
            return got
    if not isinstance(q, torch.Tensor):
        _fail("q must be a tensor")
    if q_out is None and k_out is None and torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (q, k)):
        return _Rope.apply(q, k, positions, inv_freq, interleaved, scale, inverse)
    dev = q.device
    if dev.type != "cuda":
        _fail(f"q must be on a HIP device (got {dev})")
    q, qs = _kv8_rows(q, "q", dev)
    n, H, d = q.shape
    if d not in (64, 128):
        _fail(f"head_dim must be 64 or 128 (got {d})")
    if H == 0:
        _fail(f"q {tuple(q.shape)} has no heads")
    r = _frequencies(inv_freq, dev, d)
    pos = _kv8_ints(positions, "positions", dev, n)
    outs = [torch.empty((n, H, d), dtype=torch.bfloat16, device=dev) if q_out is None else q_out]
    outs[0], qos = _kv8_rows(_same_rows(outs[0], n, "q_out"), "q_out", dev, H, d, write=True)
    kp = kop = None
    ks = kos = kh = 0
    if k is not None:
        k, ks = _kv8_rows(k, "k", dev, None, d)
        kh = _same_rows(k, n, "k").shape[1]
        outs.append(torch.empty((n, kh, d), dtype=torch.bfloat16, device=dev) if k_out is None else k_out)
        outs[1], kos = _kv8_rows(_same_rows(outs[1], n, "k_out"), "k_out", dev, kh, d, write=True)
        kp, kop = k.data_ptr(), outs[1].data_ptr()
    elif k_out is not None:
        _fail("k_out without k")
    else:
        outs.append(None)
    if n:
        _kv8_call(_native.load().sdv_rope, "sdv_rope", dev, q.data_ptr(), qs, H, kp, ks, kh, pos, inv_freq.data_ptr(), r,
                  int(bool(interleaved)), float(scale), int(bool(inverse)), n, d, outs[0].data_ptr(), qos, kop, kos)
    return tuple(outs)


def _rope_recorded(ctx) -> None:
    # a leaf's gradient is added up on the stream where the leaf was first used; one that an eager graph still holds would draw
    # that stream into the recording, which torch ends the process over
    if ctx.leaf and torch.cuda.is_current_stream_capturing():
        raise SdvError("the gradient of rope's q or k is being recorded into a HIP graph while they are leaves: record the "
                       "operation that makes them as well (a clone will do)")


def _leaf(*tensors) -> bool:
    return any(t is not None and t.requires_grad and t.is_leaf for t in tensors)


class _Rope(torch.autograd.Function):
    """rope of rows that require grad: a linear map, s times a rotation, whose transpose is s times the inverse rotation."""

    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, interleaved, scale, inverse):
        ctx.save_for_backward(positions, inv_freq)
        ctx.how, ctx.leaf = dict(interleaved=interleaved, scale=scale, inverse=not inverse), _leaf(q, k)
        ctx.set_materialize_grads(False)
        return rope(q, k, positions, inv_freq, interleaved=interleaved, scale=scale, inverse=inverse)

    @staticmethod
    def backward(ctx, gq, gk):
        _rope_recorded(ctx)
        grads = [g if need else None for g, need in zip((gq, gk), ctx.needs_input_grad)]
        given = [g for g in grads if g is not None]
        if given:
            back = iter(rope(given[0], given[1] if len(given) > 1 else None, *ctx.saved_tensors, **ctx.how))
            grads = [None if g is None else next(back) for g in grads]
        return (*grads, None, None, None, None, None)


def kv8_rope_append(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    scales: torch.Tensor, block_table: torch.Tensor, cu_rows: torch.Tensor, seq_lens: torch.Tensor | None,
                    max_seq_len: int, inv_freq: torch.Tensor, *, interleaved: bool = False, scale: float = 1.0,
                    positions: torch.Tensor | None = None, q_out: torch.Tensor | None = None) -> torch.Tensor:
    """A step's rows in one launch: q rotated (returned, BF16 (total, H, D)), k_new rotated and written into the 8-bit cache, v_new written.

    The arguments of kv8_append, and those of rope; positions int32 (total,) where a row's is not the one that it is written
    at (a tree's nodes), else None.  K is quantized as it is rotated, in fp32: its codes are one rounding nearer to the rotated
    values than those of rope and then kv8_append.  q_out: written there, which may be q itself; rows behind cu_rows[B] of it are not.
    Like the cache's other operators outside autograd.
    """
    if q_out is None:
        got = _native.binding().rope_append(q, k_new, v_new, k_pages, v_pages, scales, block_table, cu_rows, seq_lens, max_seq_len, inv_freq,
                                            interleaved, scale, positions)
        if got is not None:
            if got.__class__ is int:
                _native.check(got, "sdv_kv8_rope_append")
            return got
    dev = _kv8_device(k_pages)
    nb, kv, d, fmt = _kv8_pages(k_pages, v_pages, scales, block_table, dev)
    q, qs = _kv8_rows(q, "q", dev, None, d)
    total, H = q.shape[:2]
    k_new, ks = _kv8_rows(k_new, "k_new", dev, kv, d)
    v_new, vs = _kv8_rows(v_new, "v_new", dev, kv, d)
    _same_rows(k_new, total, "k_new")
    _same_rows(v_new, total, "v_new")
    if H == 0:
        _fail(f"q {tuple(q.shape)} has no heads")
    B, mb = block_table.shape
    max_seq_len = int(max_seq_len)
    if seq_lens is None and max_seq_len <= 0:
        _fail("seq_lens None needs max_seq_len")
    cu = _kv8_ints(cu_rows, "cu_rows", dev, B + 1)
    lens = None if seq_lens is None else _kv8_ints(seq_lens, "seq_lens", dev, B)
    pos = None if positions is None else _kv8_ints(positions, "positions", dev, total)
    r = _frequencies(inv_freq, dev, d)
    out = torch.empty((total, H, d), dtype=torch.bfloat16, device=dev) if q_out is None else q_out
    out, os_ = _kv8_rows(_same_rows(out, total, "q_out"), "q_out", dev, H, d, write=True)
    if total == 0:
        return out
    _kv8_call(_native.load().sdv_kv8_rope_append, "sdv_kv8_rope_append", dev, q.data_ptr(), qs, out.data_ptr(), os_, H, k_new.data_ptr(),
              v_new.data_ptr(), ks, vs, total, k_pages.data_ptr(), v_pages.data_ptr(), scales.data_ptr(), nb, fmt, block_table.data_ptr(),
              mb, cu, lens, max_seq_len, B, kv, d, pos, inv_freq.data_ptr(), r, int(bool(interleaved)), float(scale))
    return out


def _blocks_of(k, v, s, what, dev=None):
    """(layers, blocks, bytes of a block of each) of page tensors of either cache, checked."""
    _need(k, f"{what}k_pages", (torch.bfloat16, torch.float8_e4m3fn, torch.int8), dev)
    dev = k.device
    _need(v, f"{what}v_pages", (torch.uint8, torch.float8_e4m3fn, torch.int8), dev, (4, 5))
    _need(s, f"{what}scales", (torch.float32,), dev)
    lead = v.dim() - 4
    front = v.shape[:lead + 2]
    if k.shape[:lead + 2] != front or s.shape[:lead + 2] != front or min(front) <= 0:
        _fail(f"{what}pages disagree: k {tuple(k.shape)}, v {tuple(v.shape)}, scales {tuple(s.shape)}")
    layers, nb = (front[0] if lead else 1), front[lead]
    return layers, nb, [t.numel() // (layers * nb) * t.element_size() for t in (k, v, s)]


def copy_blocks(k_pages: torch.Tensor, v_pages: torch.Tensor, scales: torch.Tensor, src: torch.Tensor, dst: torch.Tensor, *,
                to: tuple[torch.Tensor, torch.Tensor, torch.Tensor] | None = None) -> None:
    """Copy whole page blocks, of one layer or of all at once: block src[i] to block dst[i], int32 (n,) each on the device.

    The page tensors of either cache, ([layers,] num_blocks, KV, ...).  to: the page tensors of another pool with the same layers
    and block shapes, which dst then names the blocks of.  Pairs that name no block are skipped.  No block may be the
    destination of two pairs, or of one and the source of another.
    """
    other = (k_pages, v_pages, scales) if to is None else tuple(to)
    if len(other) != 3:
        _fail("`to` needs K pages, V pages and scales")
    st = _native.binding().copy_blocks(k_pages, v_pages, scales, src, dst, *other)
    if st is not None:
        if st:
            _native.check(st, "sdv_copy_blocks")
        return
    layers, nb, size = _blocks_of(k_pages, v_pages, scales, "")
    dev = k_pages.device
    layers_to, nb_to, size_to = _blocks_of(*other, "to's ", dev)
    lead = v_pages.dim() - 4
    if layers != layers_to or any(x.dtype is not y.dtype or x.dim() != y.dim() or x.shape[lead + 1:] != y.shape[lead + 1:]
                                  for x, y in zip((k_pages, v_pages, scales), other)):
        _fail("`to` has other layers, types or block shapes")
    _need(src, "src", (torch.int32,), dev, (1,))
    n = src.shape[0]
    a, b = _kv8_ints(src, "src", dev, n), _kv8_ints(dst, "dst", dev, n)
    if n:
        _kv8_call(_native.load().sdv_copy_blocks, "sdv_copy_blocks", dev, k_pages.data_ptr(), v_pages.data_ptr(), scales.data_ptr(), nb,
                  *(t.data_ptr() for t in other), nb_to, *size, layers, a, b, n)


def kv8_keep(k_pages: torch.Tensor, v_pages: torch.Tensor, scales: torch.Tensor, block_table: torch.Tensor, cu_kept: torch.Tensor,
             kept: torch.Tensor, starts: torch.Tensor) -> None:
    """Keep some of the 8-bit cache's last tokens and close the gaps between them, in place, in one layer or in all of them.

    The token at position starts[b] + kept[cu_kept[b] + i] of sequence b comes to position starts[b] + i: after the verify of a
    drafted tree, kept are the accepted path's nodes and starts the contexts before it.  int32 on the device: cu_kept (B + 1,),
    kept (total,), starts (B,).  Pages as for kv8_append, or with a leading layer dimension.  Up to 64 tokens of a sequence are
    all read before any is written, whatever their order; of more the entries must ascend.  A token whose source or destination the
    table does not hold stays.  Sequences whose moved tokens share blocks must not be in one call.
    """
    st = _native.binding().keep(k_pages, v_pages, scales, block_table, cu_kept, kept, starts)
    if st is not None:
        if st:
            _native.check(st, "sdv_kv8_keep")
        return
    layers, nb, _ = _blocks_of(k_pages, v_pages, scales, "")
    dev = k_pages.device
    layered = v_pages.dim() == 5
    one = [t[0] if layered else t for t in (k_pages, v_pages, scales)]
    nb, kv, d, _ = _kv8_pages(*one, block_table, dev)
    B, mb = block_table.shape
    _need(kept, "kept", (torch.int32,), dev, (1,))
    cu, first = _kv8_ints(cu_kept, "cu_kept", dev, B + 1), _kv8_ints(starts, "starts", dev, B)
    if kept.shape[0]:
        _kv8_call(_native.load().sdv_kv8_keep, "sdv_kv8_keep", dev, k_pages.data_ptr(), v_pages.data_ptr(), scales.data_ptr(), nb,
                  *(t.numel() for t in one), layers, block_table.data_ptr(), mb, cu, kept.data_ptr(), kept.shape[0], first, B, kv, d)


# ---------------------------------------------------------------------------- torch.library
# The ops as torch custom operators (namespace "sdv"), so torch.compile and fake-tensor tracing
# see them: the real implementations are the functions above (the C ABI through ctypes); the
# fake implementations only produce outputs of the right shape and dtype.  The page tensors of
# the appending ops are declared mutated.
@torch.library.custom_op("sdv::paged_attention", mutates_args=())
def _lib_paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, v_scales: torch.Tensor,
                         block_table: torch.Tensor, seq_lens: torch.Tensor | None, max_seq_len: int,
                         q_token_major: bool = False) -> torch.Tensor:
    return paged_attention(q, k_pages, v_pages, v_scales, block_table, seq_lens, max_seq_len,
                           q_token_major=q_token_major)


@_lib_paged_attention.register_fake
def _(q, k_pages, v_pages, v_scales, block_table, seq_lens, max_seq_len, q_token_major=False):
    return torch.empty_like(q)


@torch.library.custom_op("sdv::attention", mutates_args=())
def _lib_attention(q: torch.Tensor, k: torch.Tensor, v_payload: torch.Tensor, v_scale: torch.Tensor) -> torch.Tensor:
    return _contiguous_attention(q, k, v_payload, v_scale)


@_lib_attention.register_fake
def _(q, k, v_payload, v_scale):
    return torch.empty_like(q)


@torch.library.custom_op("sdv::paged_attention_append", mutates_args=("k_pages", "v_pages", "v_scales"))
def _lib_paged_attention_append(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                                v_scales: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor | None,
                                max_seq_len: int, k_new: torch.Tensor, v_new: torch.Tensor,
                                slot_mapping: torch.Tensor | None, scale_mode: str = "div",
                                q_token_major: bool = False) -> torch.Tensor:
    return paged_attention(q, k_pages, v_pages, v_scales, block_table, seq_lens, max_seq_len,
                           q_token_major=q_token_major, append=(k_new, v_new, slot_mapping), scale_mode=scale_mode)


@_lib_paged_attention_append.register_fake
def _(q, k_pages, v_pages, v_scales, block_table, seq_lens, max_seq_len, k_new, v_new, slot_mapping,
      scale_mode="div", q_token_major=False):
    return torch.empty_like(q)


@torch.library.custom_op("sdv::quant_append", mutates_args=("k_pages", "v_pages", "v_scales"))
def _lib_quant_append(v_new: torch.Tensor, slot_mapping: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                      v_scales: torch.Tensor, k_new: torch.Tensor | None = None, scale_mode: str = "div") -> None:
    quant_append(v_new, slot_mapping, k_pages, v_pages, v_scales, k_new, scale_mode=scale_mode)


@_lib_quant_append.register_fake
def _(v_new, slot_mapping, k_pages, v_pages, v_scales, k_new=None, scale_mode="div"):
    return None


@torch.library.custom_op("sdv::kv8_append", mutates_args=("k_pages", "v_pages", "scales"))
def _lib_kv8_append(k_new: torch.Tensor, v_new: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, scales: torch.Tensor,
                    block_table: torch.Tensor, cu_rows: torch.Tensor, seq_lens: torch.Tensor | None, max_seq_len: int = 0) -> None:
    kv8_append(k_new, v_new, k_pages, v_pages, scales, block_table, cu_rows, seq_lens, max_seq_len)


@_lib_kv8_append.register_fake
def _(k_new, v_new, k_pages, v_pages, scales, block_table, cu_rows, seq_lens, max_seq_len=0):
    return None


@torch.library.custom_op("sdv::kv8_gather", mutates_args=())
def _lib_kv8_gather(k_pages: torch.Tensor, v_pages: torch.Tensor, scales: torch.Tensor, block_table: torch.Tensor,
                    cu_rows: torch.Tensor, starts: torch.Tensor, total_rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    return kv8_gather(k_pages, v_pages, scales, block_table, cu_rows, starts, total_rows)


@_lib_kv8_gather.register_fake
def _(k_pages, v_pages, scales, block_table, cu_rows, starts, total_rows):
    shape = (total_rows, v_pages.shape[1], v_pages.shape[2])
    return tuple(v_pages.new_empty(shape, dtype=torch.bfloat16) for _ in range(2))


@torch.library.custom_op("sdv::kv8_attention", mutates_args=())
def _lib_kv8_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, scales: torch.Tensor,
                       block_table: torch.Tensor, cu_rows: torch.Tensor, seq_lens: torch.Tensor | None, max_q_len: int,
                       max_seq_len: int, scale: float | None = None, tree_mask: torch.Tensor | None = None) -> torch.Tensor:
    return kv8_attention(q, k_pages, v_pages, scales, block_table, cu_rows, seq_lens, max_q_len, max_seq_len, scale=scale,
                         tree_mask=tree_mask)


@_lib_kv8_attention.register_fake
def _(q, k_pages, v_pages, scales, block_table, cu_rows, seq_lens, max_q_len, max_seq_len, scale=None, tree_mask=None):
    return q.new_empty(q.shape)


@torch.library.custom_op("sdv::kv8_shared_attention", mutates_args=())
def _lib_kv8_shared_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, scales: torch.Tensor,
                              block_table: torch.Tensor, cu_rows: torch.Tensor, seq_lens: torch.Tensor | None, max_q_len: int,
                              max_seq_len: int, cu_groups: torch.Tensor, prefix_lens: torch.Tensor, max_prefix_len: int,
                              scale: float | None = None, tree_mask: torch.Tensor | None = None, tile_rows: int = 0) -> torch.Tensor:
    return kv8_shared_attention(q, k_pages, v_pages, scales, block_table, cu_rows, seq_lens, max_q_len, max_seq_len, cu_groups, prefix_lens,
                                max_prefix_len, scale=scale, tree_mask=tree_mask, tile_rows=tile_rows)


@_lib_kv8_shared_attention.register_fake
def _(q, k_pages, v_pages, scales, block_table, cu_rows, seq_lens, max_q_len, max_seq_len, cu_groups, prefix_lens, max_prefix_len,
      scale=None, tree_mask=None, tile_rows=0):
    return q.new_empty(q.shape)


@torch.library.custom_op("sdv::rope", mutates_args=())
def _lib_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, interleaved: bool = False,
              scale: float = 1.0, inverse: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    return rope(q, k, positions, inv_freq, interleaved=interleaved, scale=scale, inverse=inverse)


@_lib_rope.register_fake
def _(q, k, positions, inv_freq, interleaved=False, scale=1.0, inverse=False):
    return q.new_empty(q.shape), k.new_empty(k.shape)


def _rope_keep(ctx, inputs, output):
    ctx.save_for_backward(*inputs[2:4])
    ctx.how, ctx.leaf = inputs[4:], _leaf(*inputs[:2])


def _rope_back(ctx, gq, gk):
    _rope_recorded(ctx)
    interleaved, scale, inverse = ctx.how
    return (*torch.ops.sdv.rope(gq, gk, *ctx.saved_tensors, interleaved, scale, not inverse), None, None, None, None, None)


_lib_rope.register_autograd(_rope_back, setup_context=_rope_keep)


@torch.library.custom_op("sdv::kv8_rope_append", mutates_args=("k_pages", "v_pages", "scales"))
def _lib_kv8_rope_append(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                         scales: torch.Tensor, block_table: torch.Tensor, cu_rows: torch.Tensor, seq_lens: torch.Tensor | None,
                         max_seq_len: int, inv_freq: torch.Tensor, interleaved: bool = False, scale: float = 1.0,
                         positions: torch.Tensor | None = None) -> torch.Tensor:
    return kv8_rope_append(q, k_new, v_new, k_pages, v_pages, scales, block_table, cu_rows, seq_lens, max_seq_len, inv_freq,
                           interleaved=interleaved, scale=scale, positions=positions)


@_lib_kv8_rope_append.register_fake
def _(q, k_new, v_new, k_pages, v_pages, scales, block_table, cu_rows, seq_lens, max_seq_len, inv_freq, interleaved=False, scale=1.0,
      positions=None):
    return q.new_empty(q.shape)


@torch.library.custom_op("sdv::copy_blocks", mutates_args=("k_pages", "v_pages", "scales"))
def _lib_copy_blocks(k_pages: torch.Tensor, v_pages: torch.Tensor, scales: torch.Tensor, src: torch.Tensor, dst: torch.Tensor) -> None:
    copy_blocks(k_pages, v_pages, scales, src, dst)


@_lib_copy_blocks.register_fake
def _(k_pages, v_pages, scales, src, dst):
    return None


@torch.library.custom_op("sdv::kv8_keep", mutates_args=("k_pages", "v_pages", "scales"))
def _lib_kv8_keep(k_pages: torch.Tensor, v_pages: torch.Tensor, scales: torch.Tensor, block_table: torch.Tensor, cu_kept: torch.Tensor,
                  kept: torch.Tensor, starts: torch.Tensor) -> None:
    kv8_keep(k_pages, v_pages, scales, block_table, cu_kept, kept, starts)


@_lib_kv8_keep.register_fake
def _(k_pages, v_pages, scales, block_table, cu_kept, kept, starts):
    return None
