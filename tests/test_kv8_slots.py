"""The slots of sdv_kv8_attention_slot: refusals on the host, before any HIP call."""
from __future__ import annotations

import ctypes

import pytest

from conftest import ROOT
from specdec_amd import _native
from test_kv8_abi import N, P


@pytest.mark.parametrize("slot,status", [(-1, _native.SDV_OK), (0, _native.SDV_OK), (2047, _native.SDV_OK), (2048, _native.SDV_ERR_WORKSPACE),
                                         (-2, _native.SDV_ERR_WORKSPACE), (2 ** 31 - 1, _native.SDV_ERR_WORKSPACE)])
@pytest.mark.parametrize("rows_each", [1, 300])
def test_slots(slot, status, rows_each):
    lib = _native.load()
    assert "#define SDV_KV8_SLOTS 2048" in (ROOT / "include" / "sdv.h").read_text()
    args = dict(q=P, qs=1536, kp=P, vp=P, sc=P, nb=8, fmt=0, bt=P, mb=4, cu=P, ln=P, tree=N, B=1, n=0, H=12, KV=2, D=128, S=rows_each, T=4096,
                scale=0.1, ws=P, wsb=1 << 30, slot=slot, out=P, os=1536)
    assert lib.sdv_kv8_attention_slot(*args.values(), N) == status  # no rows: nothing to do
    args.update(ws=ctypes.c_void_p(0), slot=0)
    assert lib.sdv_kv8_attention_slot(*args.values(), N) == _native.SDV_ERR_WORKSPACE
