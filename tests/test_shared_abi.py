"""Shared-prefix attention's entry points on the host: refusals before any HIP call, workspace sizes, the rule for tiles; CPU and fake
tensors."""
from __future__ import annotations

import ctypes

import pytest
import torch

from specdec_amd import _native, build
from specdec_amd._native import SdvError
from specdec_amd.kernels import ops

P = ctypes.c_void_p(0x1000)   # aligned, never dereferenced
ODD, HALF = ctypes.c_void_p(0x1008), ctypes.c_void_p(0x1002)
N = None
SIZES = dict(B=8, groups=1, total=8, H=12, KV=2, D=128, rows=1, longest=8192, prefix=4096)


@pytest.fixture(scope="module")
def lib():
    if not _native.LIB_PATH.exists():
        build.build()
    return _native.load()


def _bytes(lib, tile, **kw):
    return lib.sdv_kv8_shared_attention_workspace_size(*{**SIZES, **kw}.values(), tile)


def _rows(lib, **kw):
    return lib.sdv_kv8_shared_attention_tile_rows(*{**SIZES, **kw}.values())


def _call(lib, **kw):
    a = dict(q=P, qs=1536, kp=P, vp=P, sc=P, nb=8, fmt=0, bt=P, mb=512, cu=P, lens=P, tree=N, groups_at=P, prefix_at=P, **SIZES, tile=32,
             scale=1.0, ws=P, bytes=_bytes(lib, kw.get("tile", 32)) if kw.get("tile", 32) in (32, 128) else 1 << 40, out=P, os=1536)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.sdv_kv8_shared_attention(*a.values(), N)


def test_checks(lib):
    for name in ("q", "kp", "vp", "sc", "bt", "cu", "groups_at", "prefix_at", "out"):
        assert _call(lib, **{name: N}) == _native.SDV_ERR_NULL, name
    shape = [dict(B=0), dict(groups=-1), dict(groups=9), dict(total=-1), dict(H=0), dict(KV=0), dict(H=13), dict(rows=0), dict(longest=0), dict(prefix=-1),
             dict(H=1 << 17, KV=1 << 10), dict(nb=0), dict(mb=0), dict(mb=1 << 28), dict(mb=255), dict(qs=1528), dict(os=1528),
             dict(longest=1 << 30), dict(prefix=1 << 28), dict(total=1 << 30)]
    for bad in shape:
        assert _call(lib, **bad) == _native.SDV_ERR_SHAPE, bad
    for bad in (dict(D=96), dict(fmt=2), dict(tile=0), dict(tile=64), dict(tile=-32), dict(tree=P, rows=65)):
        assert _call(lib, **bad) == _native.SDV_ERR_UNSUPPORTED, bad
    for bad in (dict(q=ODD), dict(out=ODD), dict(qs=1540), dict(os=1540), dict(kp=ODD), dict(vp=ODD), dict(sc=ODD), dict(bt=HALF), dict(cu=HALF),
                dict(lens=HALF), dict(tree=HALF), dict(groups_at=HALF), dict(prefix_at=HALF)):
        assert _call(lib, **bad) == _native.SDV_ERR_ALIGN, bad
    for tile in (32, 128):
        n = _bytes(lib, tile)
        for bad in (dict(ws=N), dict(ws=ODD), dict(bytes=n - 1), dict(bytes=0)):
            assert _call(lib, tile=tile, **bad) == _native.SDV_ERR_WORKSPACE, bad
        assert _call(lib, tile=tile, total=0) == _native.SDV_OK     # nothing to do


@pytest.mark.parametrize("tile", [32, 128])
@pytest.mark.parametrize("D", [64, 128])
def test_workspace(lib, tile, D):
    """A table of rows and a part for each tile and workgroup: 32 or 128 rows of a prefix, 16 or 32 of a sequence's, D + 2 floats a row
    at least; never less for more."""
    for total, rows, groups in ((8, 1, 1), (40, 5, 1), (40, 5, 4), (512, 64, 8), (0, 1, 1)):
        n = _bytes(lib, tile, D=D, total=total, rows=rows, groups=groups)
        own = 16 if 6 * rows <= 16 else 32
        assert n >= 4 * (D + 2) * 2 * total * 12, (total, rows, groups)
        assert n >= 4 * (D + 2) * 512 * (tile + own)
        assert n <= _bytes(lib, tile, D=D, total=total + 1, rows=rows, groups=groups)
        assert n <= _bytes(lib, tile, D=D, total=total, rows=rows, groups=min(8, groups + 1))
    assert _bytes(lib, 0) == _bytes(lib, 64) == _bytes(lib, 32, D=96) == _bytes(lib, 32, H=13) == _bytes(lib, 128, longest=1 << 30) == 0
    assert _bytes(lib, 32, longest=100) == _bytes(lib, 32, longest=200000)   # lengths do not size it


def test_the_rule(lib):
    """0: sequence by sequence."""
    assert _rows(lib, B=1, total=1) == 0 and _rows(lib, groups=8) == 0 and _rows(lib, groups=0) == 0  # nothing is read twice
    assert _rows(lib, rows=11, total=88) == 0                                                        # 66 rows of a KV head
    assert _rows(lib, D=96) == 0 and _rows(lib, longest=1 << 30) == 0
    for rows in (1, 5):
        last = 0
        for prefix in (0, 16, 256, 1024, 4096, 16384, 65536, 1 << 18):                               # more to share: never less so
            got = _rows(lib, B=32, total=32 * rows, rows=rows, prefix=prefix, longest=prefix + 100)
            assert got in (0, 32, 128) and got >= last
            last = got
        assert last == 128
    for groups in (1, 2, 4, 31):
        assert _rows(lib, B=32, total=32, groups=groups, prefix=1 << 17, longest=1 << 18) >= _rows(lib, B=32, total=32, groups=groups + 1, prefix=1 << 17,
                                                                                               longest=1 << 18)


def test_tensors_on_the_cpu_are_refused():
    kp, vp, sc = torch.zeros((2, 2, 4, 8, 4, 16), dtype=torch.int8), torch.zeros((2, 2, 128, 16), dtype=torch.int8), torch.ones((2, 2, 2, 16))
    bt, cu, one = torch.zeros((1, 2), dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q = torch.zeros((1, 4, 128), dtype=torch.bfloat16)
    with pytest.raises(SdvError, match="HIP device"):
        ops.kv8_shared_attention(q, kp, vp, sc, bt, cu, one, 1, 1, cu, one, 16)
    with pytest.raises(ValueError, match="tile_rows"):
        ops.kv8_shared_attention(q, kp, vp, sc, bt, cu, one, 1, 1, cu, one, 16, tile_rows=64)
    b = _native.binding()
    assert b.shared(q, kp, vp, sc, bt, cu, one, 1, 1, cu, one, 16, None, None, 0, None) is None
    for bad in ((), (None,) * 16, (1, "x", None, 2.0, [], {}, ()), (0,) * 16, (q,) * 16):
        assert b.shared(*bad) is None
    with pytest.raises(TypeError):
        b.bind_shared(1)
    with pytest.raises(ValueError):
        b.bind_shared(0, 0, 0)


def test_fake_tensors_propagate_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        kp = torch.empty((9, 2, 4, 8, 4, 16), dtype=torch.float8_e4m3fn, device="cuda")
        vp, sc = torch.empty((9, 2, 128, 16), dtype=torch.float8_e4m3fn, device="cuda"), torch.empty((9, 2, 2, 16), device="cuda")
        bt, cu, groups, ids = (torch.empty(n, dtype=torch.int32, device="cuda") for n in ((3, 4), (4,), (2,), (3,)))
        q = torch.empty((7, 12, 128), dtype=torch.bfloat16, device="cuda")
        out = torch.ops.sdv.kv8_shared_attention(q, kp, vp, sc, bt, cu, None, 3, 60, groups, ids, 32)
        assert out.shape == q.shape and out.dtype is torch.bfloat16
    assert "!" not in str(torch.ops.sdv.kv8_shared_attention.default._schema)
