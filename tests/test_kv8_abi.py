"""The 8-bit cache's entry points refuse bad arguments on the host, before any HIP call; its int8
division route gives the IEEE quotient's codes (an exhaustive walk on the CPU)."""
from __future__ import annotations

import ctypes
import os
import random
import re
import shutil
import subprocess

import pytest
import torch

from conftest import ROOT
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


def _append(lib, **kw):
    a = dict(k=P, v=P, ks=256, vs=256, n=4, kp=P, vp=P, sc=P, nb=8, fmt=0, bt=P, mb=4, cu=P, ln=P, T=0, B=1, KV=2, D=128)
    a.update(kw)
    return lib.sdv_kv8_append(*a.values(), N)


def _gather(lib, **kw):
    a = dict(kp=P, vp=P, sc=P, nb=8, fmt=0, bt=P, mb=4, cu=P, st=P, B=1, n=4, KV=2, D=128, k=P, v=P, ks=256, vs=256)
    a.update(kw)
    return lib.sdv_kv8_gather(*a.values(), N)


def _attend(lib, **kw):
    a = dict(q=P, qs=1536, kp=P, vp=P, sc=P, nb=8, fmt=0, bt=P, mb=4, cu=P, ln=P, tree=N, B=1, n=4, H=12, KV=2, D=128, S=4, T=64,
             scale=0.1, ws=P, wsb=1 << 30, out=P, os=1536)
    a.update(kw)
    return lib.sdv_kv8_attention(*a.values(), N)


@pytest.mark.parametrize("call,null", [(_append, ("k", "v", "kp", "vp", "sc", "bt", "cu")),
                                       (_gather, ("k", "v", "kp", "vp", "sc", "bt", "cu", "st")),
                                       (_attend, ("q", "kp", "vp", "sc", "bt", "cu", "out"))])
def test_shared_checks(lib, call, null):
    for name in null:
        assert call(lib, **{name: N}) == _native.SDV_ERR_NULL, name
    for bad in (dict(n=-1), dict(nb=0), dict(mb=0), dict(mb=1 << 28), dict(B=0), dict(KV=0), dict(n=(1 << 30) + 1)):
        assert call(lib, **bad) == _native.SDV_ERR_SHAPE, bad
    for bad in (dict(D=96), dict(fmt=2), dict(fmt=-1)):
        assert call(lib, **bad) == _native.SDV_ERR_UNSUPPORTED, bad
    for name in ("kp", "vp", "sc"):
        assert call(lib, **{name: ODD}) == _native.SDV_ERR_ALIGN, name
    for name in ("bt", "cu"):
        assert call(lib, **{name: ctypes.c_void_p(0x1002)}) == _native.SDV_ERR_ALIGN, name
    assert call(lib, n=0) == _native.SDV_OK  # nothing to do


def test_append_checks(lib):
    assert _append(lib, ks=255) == _native.SDV_ERR_SHAPE
    assert _append(lib, vs=260) == _native.SDV_ERR_ALIGN
    assert _append(lib, k=ODD) == _native.SDV_ERR_ALIGN
    assert _append(lib, ln=N) == _native.SDV_ERR_SHAPE      # no lengths and no length
    assert _append(lib, KV=65536, ks=1 << 24, vs=1 << 24) == _native.SDV_ERR_SHAPE


def test_gather_checks(lib):
    assert _gather(lib, vs=128) == _native.SDV_ERR_SHAPE
    assert _gather(lib, k=ODD) == _native.SDV_ERR_ALIGN


def test_attention_checks(lib):
    assert _attend(lib, H=13) == _native.SDV_ERR_SHAPE
    assert _attend(lib, S=0) == _native.SDV_ERR_SHAPE
    assert _attend(lib, T=0) == _native.SDV_ERR_SHAPE
    assert _attend(lib, qs=1528) == _native.SDV_ERR_SHAPE
    assert _attend(lib, os=1540) == _native.SDV_ERR_ALIGN
    assert _attend(lib, q=ODD) == _native.SDV_ERR_ALIGN
    assert _attend(lib, tree=P, S=65) == _native.SDV_ERR_UNSUPPORTED
    assert _attend(lib, tree=ctypes.c_void_p(0x1004)) == _native.SDV_ERR_ALIGN
    assert _attend(lib, ws=N) == _native.SDV_ERR_WORKSPACE
    assert _attend(lib, ws=ctypes.c_void_p(0x1010)) == _native.SDV_ERR_WORKSPACE
    assert _attend(lib, wsb=64) == _native.SDV_ERR_WORKSPACE
    assert _attend(lib, T=2 ** 31 - 1) == _native.SDV_ERR_SHAPE      # more than the 32-bit sums hold
    assert _attend(lib, n=1 << 25, T=1 << 25) == _native.SDV_ERR_SHAPE
    need = lib.sdv_kv8_attention_workspace_size(1, 4, 12, 2, 128, 4, 64)
    assert need > 0 and _attend(lib, wsb=need - 1) == _native.SDV_ERR_WORKSPACE
    assert lib.sdv_kv8_attention_workspace_size(1, 4, 12, 2, 96, 4, 64) == 0
    assert lib.sdv_kv8_attention_workspace_size(1, 4, 12, 5, 128, 4, 64) == 0


def test_a_workspace_for_the_largest_call_serves_the_smaller(lib):
    rng = random.Random(4)
    for _ in range(3000):
        G, kv, d = rng.choice([1, 6, 7]), rng.choice([1, 2, 8]), rng.choice([64, 128])
        big = [rng.randint(1, 64), rng.randint(1, 4096), rng.randint(1, 600), 1 << rng.randint(4, 17)]
        small = [rng.randint(1, x) for x in big]
        a, b = [lib.sdv_kv8_attention_workspace_size(c[0], c[1], G * kv, kv, d, c[2], c[3]) for c in (small, big)]
        assert 0 < a <= b, (G, kv, d, small, big)


def test_tensors_on_the_cpu_are_refused():
    kp = torch.zeros((2, 2, 4, 8, 4, 16), dtype=torch.int8)
    vp, sc = torch.zeros((2, 2, 128, 16), dtype=torch.int8), torch.ones((2, 2, 2, 16))
    bt, cu, ln = torch.zeros((1, 2), dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    x = torch.zeros((1, 2, 128), dtype=torch.bfloat16)
    with pytest.raises(SdvError, match="HIP device"):
        ops.kv8_append(x, x, kp, vp, sc, bt, cu, ln)
    with pytest.raises(SdvError, match="HIP device"):
        ops.kv8_gather(kp, vp, sc, bt, cu, ln, 1)
    with pytest.raises(SdvError, match="HIP device"):
        ops.kv8_attention(x, kp, vp, sc, bt, cu, ln, 1, 16)


def test_extension_module_leaves_cpu_tensors_to_the_general_path():
    b = _native.binding()
    kp, vp, sc = torch.zeros((2, 2, 4, 8, 4, 16), dtype=torch.int8), torch.zeros((2, 2, 128, 16), dtype=torch.int8), torch.ones((2, 2, 2, 16))
    bt, cu, ln = torch.zeros((1, 2), dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    x = torch.zeros((1, 2, 128), dtype=torch.bfloat16)
    assert b.append(x, x, kp, vp, sc, bt, cu, ln, 0) is None
    assert b.gather(kp, vp, sc, bt, cu, ln, 1) is None
    assert b.attention(x, kp, vp, sc, bt, cu, ln, 1, 16, None, None) is None
    for bad in ((), (None,) * 11, (1, "x", None, 2.0, [], {}, (), 0, 0, 0, 0)):
        assert b.attention(*bad) is None and b.append(*bad) is None and b.gather(*bad) is None
    with pytest.raises(TypeError):
        b.bind(1)
    with pytest.raises(ValueError):
        b.bind(0, 0, 0, 0)
    with pytest.raises(TypeError):
        b.bind("a", "b", "c", "d")


def test_fake_tensors_propagate_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        kp = torch.empty((9, 2, 4, 8, 4, 16), dtype=torch.float8_e4m3fn, device="cuda")
        vp, sc = torch.empty((9, 2, 128, 16), dtype=torch.float8_e4m3fn, device="cuda"), torch.empty((9, 2, 2, 16), device="cuda")
        bt, cu, ln = (torch.empty(n, dtype=torch.int32, device="cuda") for n in ((3, 4), (4,), (3,)))
        q, x = (torch.empty((7, h, 128), dtype=torch.bfloat16, device="cuda") for h in (12, 2))
        out = torch.ops.sdv.kv8_attention(q, kp, vp, sc, bt, cu, ln, 3, 60)
        assert out.shape == q.shape and out.dtype is torch.bfloat16
        k, v = torch.ops.sdv.kv8_gather(kp, vp, sc, bt, cu, ln, 11)
        assert k.shape == v.shape == (11, 2, 128) and k.dtype is torch.bfloat16
        assert torch.ops.sdv.kv8_append(x, x, kp, vp, sc, bt, cu, None, 60) is None
    schema = str(torch.ops.sdv.kv8_append.default._schema)
    assert all(re.search(r"Tensor\(a\d+!\) " + name, schema) for name in ("k_pages", "v_pages", "scales"))
    assert "!" not in str(torch.ops.sdv.kv8_attention.default._schema)


def test_int8_quotient_gives_the_ieee_codes(tmp_path):
    cc = shutil.which("gcc")
    if cc is None:
        pytest.skip("gcc not found")
    exe = tmp_path / "quotient_check_int8"
    src = str(ROOT / "tests" / "native" / "quotient_check_int8.c")
    base = ["-O2", "-ffp-contract=off", "-fopenmp", "-o", str(exe), src, "-lm"]
    if subprocess.run([cc, "-march=native", *base], capture_output=True).returncode != 0:
        subprocess.run([cc, *base], check=True)
    env = dict(os.environ, OMP_NUM_THREADS=str(min(8, os.cpu_count() or 1)))
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=600, env=env)
    m = re.match(r"(\d+) pairs, (\d+) differences", res.stdout)
    assert m and res.returncode == 0, res.stdout + res.stderr
    assert int(m[1]) == 495_922_945 and int(m[2]) == 0
