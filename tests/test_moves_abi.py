"""The entry points for positions and page moves refuse bad arguments on the host, before any HIP call; frequencies of
stretched contexts against their definitions; the operators leave CPU tensors alone."""
from __future__ import annotations

import ctypes
import math
import re

import pytest
import torch

from specdec_amd import _native, build
from specdec_amd._native import SdvError
from specdec_amd.kernels import ops

P = ctypes.c_void_p(0x1000)   # aligned, never dereferenced
ODD = ctypes.c_void_p(0x1008)
N = None


@pytest.fixture(scope="module")
def lib():
    if not _native.LIB_PATH.exists():
        build.build()
    return _native.load()


def _rope(lib, **kw):
    a = dict(q=P, qs=1536, H=12, k=P, ks=256, KV=2, pos=P, inv=P, r=128, il=0, scale=1.0, back=0, n=4, D=128, qo=P, qos=1536, ko=P, kos=256)
    a.update(kw)
    return lib.sdv_rope(*a.values(), N)


def _step(lib, **kw):
    a = dict(q=P, qs=1536, qo=P, qos=1536, H=12, k=P, v=P, ks=256, vs=256, n=4, kp=P, vp=P, sc=P, nb=8, fmt=0, bt=P, mb=4, cu=P, ln=P,
             T=0, B=1, KV=2, D=128, pos=N, inv=P, r=128, il=0, scale=1.0)
    a.update(kw)
    return lib.sdv_kv8_rope_append(*a.values(), N)


def _copy(lib, **kw):
    a = dict(k=P, v=P, s=P, nb=8, k2=P, v2=P, s2=P, nb2=8, kb=4096, vb=4096, sb=256, L=2, src=P, dst=P, n=3)
    a.update(kw)
    return lib.sdv_copy_blocks(*a.values(), N)


def _keep(lib, **kw):
    a = dict(kp=P, vp=P, sc=P, nb=8, ks=65536, vs=65536, ss=512, L=2, bt=P, mb=4, cu=P, kept=P, n=3, st=P, B=1, KV=2, D=128)
    a.update(kw)
    return lib.sdv_kv8_keep(*a.values(), N)


def _refused(lib, call, null=(), shape=(), unsupported=(), align=()):
    for name in null:
        assert call(lib, **{name: N}) == _native.SDV_ERR_NULL, name
    for status, cases in ((_native.SDV_ERR_SHAPE, shape), (_native.SDV_ERR_UNSUPPORTED, unsupported), (_native.SDV_ERR_ALIGN, align)):
        for bad in cases:
            assert call(lib, **bad) == status, bad
    assert call(lib, n=0) == _native.SDV_OK  # nothing to do


def test_rope_checks(lib):
    _refused(lib, _rope, ("q", "k", "pos", "inv", "qo", "ko"),
             [dict(r=0), dict(r=8), dict(r=144), dict(il=2), dict(back=2), dict(n=-1), dict(n=1 << 30), dict(H=0), dict(KV=-1), dict(qs=1528),
              dict(kos=128), dict(H=1 << 20, qs=1 << 40)],
             [dict(D=96)], [dict(q=ODD), dict(ko=ODD), dict(qs=1540), dict(ks=260), dict(pos=ctypes.c_void_p(0x1002)),
                            dict(inv=ctypes.c_void_p(0x1004))])
    assert _rope(lib, KV=0, k=N, ko=N, ks=0, kos=0, n=0) == _native.SDV_OK


def test_step_checks(lib):
    _refused(lib, _step, ("q", "qo", "k", "v", "kp", "vp", "sc", "bt", "cu", "inv"),
             [dict(r=24), dict(r=0), dict(r=144), dict(H=0), dict(H=65536, qs=1 << 24, qos=1 << 24), dict(qs=1528), dict(qos=1528), dict(ks=128),
              dict(ln=N), dict(nb=0), dict(B=0), dict(n=-1), dict(mb=1 << 28)],
             [dict(D=96), dict(fmt=2)], [dict(q=ODD), dict(qo=ODD), dict(qs=1540), dict(qos=1540), dict(v=ODD), dict(inv=ctypes.c_void_p(0x1004)),
                                         dict(pos=ctypes.c_void_p(0x1002))])


def test_copy_checks(lib):
    _refused(lib, _copy, ("k", "v", "s", "k2", "v2", "s2", "src", "dst"),
             [dict(nb=0), dict(nb2=0), dict(L=0), dict(L=65536), dict(n=-1), dict(kb=0), dict(vb=1 << 30)], [],
             [dict(kb=4104), dict(sb=8), dict(k=ODD), dict(s2=ODD), dict(src=ctypes.c_void_p(0x1002))])


def test_keep_checks(lib):
    _refused(lib, _keep, ("kp", "vp", "sc", "bt", "cu", "kept", "st"),
             [dict(nb=0), dict(nb=1 << 28), dict(mb=0), dict(mb=1 << 28), dict(B=0), dict(KV=0), dict(L=0), dict(n=-1), dict(ks=32752), dict(vs=0),
              dict(ss=508)],
             [dict(D=96)], [dict(kp=ODD), dict(ks=65544), dict(bt=ctypes.c_void_p(0x1002)), dict(kept=ctypes.c_void_p(0x1002))])
    assert _keep(lib, L=1, ks=0, vs=0, ss=0, n=0) == _native.SDV_OK


def test_frequencies():
    inv, scale = ops.rope_frequencies(128, 10000.0, device="cpu")
    assert scale == 1.0 and inv.dtype is torch.float64
    assert inv.tolist() == pytest.approx([10000.0 ** (-2 * i / 128) for i in range(64)], rel=1e-14)
    part, _ = ops.rope_frequencies(128, 10000.0, rotary_dim=32, device="cpu")
    assert part.tolist() == pytest.approx([10000.0 ** (-i / 16) for i in range(16)], rel=1e-14)
    linear, scale = ops.rope_frequencies(128, 10000.0, scaling={"type": "linear", "factor": 4.0}, device="cpu")
    assert scale == 1.0 and torch.allclose(linear, inv / 4, rtol=1e-14)
    ntk, scale = ops.rope_frequencies(128, 10000.0, scaling={"type": "ntk", "factor": 8.0}, device="cpu")
    assert scale == 1.0 and ntk[0] == 1.0 and float(ntk[-1]) == pytest.approx(float(inv[-1]) / 8, rel=1e-12)
    yarn, scale = ops.rope_frequencies(128, 10000.0, scaling={"type": "yarn", "factor": 4.0, "original": 4096}, device="cpu")
    assert scale == pytest.approx(0.1 * math.log(4) + 1)
    for i in range(64):
        turns = 4096 * float(inv[i]) / (2 * math.pi)
        stays = min(1.0, max(0.0, (turns - 1) / 31))
        assert float(yarn[i]) == pytest.approx(float(inv[i]) * (stays + (1 - stays) / 4), rel=1e-12)
    assert torch.equal(ops.rope_frequencies(64, scaling={"type": "ntk", "factor": 1.0}, device="cpu")[0], ops.rope_frequencies(64, device="cpu")[0])


@pytest.mark.parametrize("bad", [dict(rotary_dim=24), dict(rotary_dim=0), dict(rotary_dim=144), dict(base=0.0), dict(scaling={"type": "x"}),
                                 dict(scaling={"factor": 2.0}), dict(scaling={"type": "linear", "factor": 0.5}),
                                 dict(scaling={"type": "linear", "factor": 2.0, "original": 5}), dict(scaling={"type": "yarn", "factor": 2.0}),
                                 dict(scaling={"type": "yarn", "factor": 2.0, "original": 64, "slow": 9, "fast": 9})])
def test_frequencies_refuse(bad):
    with pytest.raises(ValueError):
        ops.rope_frequencies(128, device="cpu", **bad)


def test_tensors_on_the_cpu_are_refused():
    kp, vp, sc = torch.zeros((2, 2, 4, 8, 4, 16), dtype=torch.int8), torch.zeros((2, 2, 128, 16), dtype=torch.int8), torch.ones((2, 2, 2, 16))
    bt, cu, one = torch.zeros((1, 2), dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    x, inv = torch.zeros((1, 2, 128), dtype=torch.bfloat16), torch.zeros(64, dtype=torch.float64)
    for call in (lambda: ops.rope(x, x, one, inv), lambda: ops.kv8_rope_append(x, x, x, kp, vp, sc, bt, cu, one, 0, inv),
                 lambda: ops.copy_blocks(kp, vp, sc, one, one), lambda: ops.kv8_keep(kp, vp, sc, bt, cu, one, one)):
        with pytest.raises(SdvError, match="HIP device"):
            call()
    b = _native.binding()
    assert b.rope(x, x, one, inv, False, 1.0, False) is None and b.rope_append(x, x, x, kp, vp, sc, bt, cu, one, 0, inv, False, 1.0, None) is None
    assert b.copy_blocks(kp, vp, sc, one, one, kp, vp, sc) is None and b.keep(kp, vp, sc, bt, cu, one, one) is None
    for bad in ((), (None,) * 14, (1, "x", None, 2.0, [], {}, ()), (0,) * 8):
        assert b.rope(*bad) is None and b.rope_append(*bad) is None and b.copy_blocks(*bad) is None and b.keep(*bad) is None
    with pytest.raises(TypeError):
        b.bind_moves(1)
    with pytest.raises(ValueError):
        b.bind_moves(0, 0, 0, 0)


def test_fake_tensors_propagate_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        kp = torch.empty((9, 2, 4, 8, 4, 16), dtype=torch.float8_e4m3fn, device="cuda")
        vp, sc = torch.empty((9, 2, 128, 16), dtype=torch.float8_e4m3fn, device="cuda"), torch.empty((9, 2, 2, 16), device="cuda")
        bt, cu, ids = (torch.empty(n, dtype=torch.int32, device="cuda") for n in ((3, 4), (4,), (3,)))
        q, x = (torch.empty((7, h, 128), dtype=torch.bfloat16, device="cuda") for h in (12, 2))
        pos, inv = torch.empty(7, dtype=torch.int32, device="cuda"), torch.empty(64, dtype=torch.float64, device="cuda")
        a, b = torch.ops.sdv.rope(q, x, pos, inv)
        assert a.shape == q.shape and b.shape == x.shape and a.dtype is torch.bfloat16
        out = torch.ops.sdv.kv8_rope_append(q, x, x, kp, vp, sc, bt, cu, None, 60, inv)
        assert out.shape == q.shape and out.dtype is torch.bfloat16
        assert torch.ops.sdv.copy_blocks(kp, vp, sc, ids, ids) is None and torch.ops.sdv.kv8_keep(kp, vp, sc, bt, cu, ids, ids) is None
    for name in ("kv8_rope_append", "copy_blocks", "kv8_keep"):
        schema = str(getattr(torch.ops.sdv, name).default._schema)
        assert all(re.search(r"Tensor\(a\d+!\) " + part, schema) for part in ("k_pages", "v_pages", "scales")), schema
    assert "!" not in str(torch.ops.sdv.rope.default._schema)
