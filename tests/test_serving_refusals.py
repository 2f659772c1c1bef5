"""What the serving-step entry points refuse, before any launch (CPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from paged_tierkv_amd import _lib, kernels
from paged_tierkv_amd.tierkv_hip import tierkv_extend_attention

P = 4096        # a non-null, aligned address that no refused call touches


def slot_map(**kw):
    a = dict(new=P, batch=2, rows=8, table=P, states=P, lengths=P, stride=8, nblocks=P, open=P, free=P, slots=16, ctl=P,
             bs=16, out=P, pos=P, cu=P, ctx=P, ws=P, nbytes=1 << 20)
    a.update(kw)
    return _lib.lib().tierkv_build_slot_map(
        a["new"], a["batch"], a["rows"], a["table"], a["states"], a["lengths"], a["stride"], a["nblocks"], a["open"],
        a["free"], a["slots"], a["ctl"], a["bs"], a["out"], a["pos"], a["cu"], a["ctx"], a["ws"], a["nbytes"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(new=None), 1), (dict(ctl=None), 1), (dict(out=None), 1), (dict(batch=0), 1), (dict(rows=-1), 1),
    (dict(stride=0), 1), (dict(slots=0), 1), (dict(out=P + 4), 1), (dict(ws=P + 8), 1), (dict(batch=4097), 2),
    (dict(bs=0), 2), (dict(bs=65), 2), (dict(slots=1 << 28), 2), (dict(stride=1 << 28), 2), (dict(rows=(1 << 30) + 1), 2),
    (dict(nbytes=100), 4),
])
def test_slot_map_refusals(kw, code):
    assert slot_map(**kw) == code and _lib.last_error()


def write(**kw):
    a = dict(k=P, kt=128, kh=64, v=P, vt=128, vh=64, dtype=0, slots=P, rows=4, hk=P, hv=P, pool=8, kv=2, bs=16, d=64)
    a.update(kw)
    return _lib.lib().tierkv_write_slots(a["k"], a["kt"], a["kh"], a["v"], a["vt"], a["vh"], a["dtype"], a["slots"],
                                         a["rows"], a["hk"], a["hv"], a["pool"], a["kv"], a["bs"], a["d"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(k=None), 1), (dict(slots=None), 1), (dict(hv=None), 1), (dict(dtype=2), 1), (dict(rows=-1), 1),
    (dict(kt=-1), 1), (dict(kv=0), 2), (dict(bs=65), 2), (dict(d=257), 2), (dict(pool=0), 2), (dict(pool=1 << 27), 2),
    (dict(rows=0), 0), (dict(rows=0, k=None), 0),
])
def test_write_slots_refusals(kw, code):
    assert write(**kw) == code


def extend(**kw):
    a = dict(q=P, qt=512, qh=64, dtype=0, out=P, cu=P, rows=8, most=8, table=P, states=P, lengths=P, stride=8, snb=None,
             blocks=8, hk=P, hv=P, hot=4, wk=P, wv=P, warm=4, ks=P, kz=P, vs=P, vz=P, fmt=0, cold=0, batch=2, heads=8,
             kv=2, bs=16, d=64, scaling=0.125, ws=P, nbytes=1 << 40)
    a.update(kw)
    return _lib.lib().tierkv_extend_attention(
        a["q"], a["qt"], a["qh"], a["dtype"], a["out"], a["cu"], a["rows"], a["most"], a["table"], a["states"],
        a["lengths"], a["stride"], a["snb"], a["blocks"], a["hk"], a["hv"], a["hot"], a["wk"], a["wv"], a["warm"], a["ks"],
        a["kz"], a["vs"], a["vz"], a["fmt"], a["cold"], a["batch"], a["heads"], a["kv"], a["bs"], a["d"],
        ctypes.c_float(a["scaling"]), a["ws"], a["nbytes"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), 1), (dict(cu=None), 1), (dict(ws=None), 1), (dict(rows=-1), 1), (dict(most=-1), 1), (dict(batch=0), 1),
    (dict(heads=7), 1), (dict(blocks=0), 1), (dict(blocks=9), 1), (dict(dtype=2), 1), (dict(fmt=2), 1), (dict(cold=2), 1),
    (dict(hk=None), 1), (dict(warm=0), 1), (dict(kz=None), 1), (dict(scaling=float("inf")), 1),
    (dict(scaling=float("nan")), 1), (dict(qt=510), 1), (dict(qh=-64), 1), (dict(q=P + 2), 1), (dict(out=P + 8), 1),
    (dict(bs=0), 2), (dict(bs=65), 2), (dict(d=60), 2), (dict(d=136), 2), (dict(rows=1 << 28), 2), (dict(nbytes=4096), 4),
    (dict(rows=0), 0), (dict(most=0), 0),
])
def test_extend_attention_refusals(kw, code):
    assert extend(**kw) == code


def sample(**kw):
    a = dict(x=P, dtype=2, stride=100, batch=2, vocab=100, u=P, tokens=P, probs=None, ws=P, nbytes=1 << 30)
    a.update(kw)
    f = ctypes.c_float
    return _lib.lib().tierkv_sample_tokens(a["x"], a["dtype"], a["stride"], a["batch"], a["vocab"], a["u"], None, f(1.0),
                                           None, 0, None, f(1.0), None, f(0.0), a["tokens"], a["probs"], a["ws"],
                                           a["nbytes"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(x=None), 1), (dict(u=None), 1), (dict(tokens=None), 1), (dict(ws=None), 1), (dict(batch=0), 1),
    (dict(vocab=0), 1), (dict(dtype=3), 1), (dict(stride=99), 1), (dict(vocab=(1 << 20) + 1, stride=1 << 21), 2),
    (dict(nbytes=16), 4),
])
def test_sampling_refusals(kw, code):
    assert sample(**kw) == code


def test_workspace_sizes_refuse_bad_geometry():
    lib = _lib.lib()
    assert lib.tierkv_slot_map_workspace_bytes(0) < 0 < lib.tierkv_slot_map_workspace_bytes(1)
    assert lib.tierkv_sample_workspace_bytes(0, 5) < 0 and lib.tierkv_sample_workspace_bytes(1, 0) < 0
    assert lib.tierkv_extend_workspace_bytes(1, 4, 4, 7, 2, 8, 16, 64) < 0
    assert lib.tierkv_extend_workspace_bytes(1, 4, 4, 8, 2, 0, 16, 64) < 0
    small = lib.tierkv_extend_workspace_bytes(2, 4, 4, 8, 2, 8, 16, 64)
    assert 0 < small <= lib.tierkv_extend_workspace_bytes(2, 400, 400, 8, 2, 8, 16, 64)


def test_wrappers_refuse_cpu_tensors():
    i32 = torch.zeros((2, 4), dtype=torch.int32)
    v = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        kernels.build_slot_map(v, i32, i32, i32, v, v, v, torch.zeros(4, dtype=torch.int32), 16, 8)
    pool = torch.zeros((2, 2, 16, 64), dtype=torch.float16)
    rows = torch.zeros((3, 2, 64), dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU"):
        kernels.write_slots(rows, rows, torch.zeros(3, dtype=torch.int32), pool, pool)
    with pytest.raises(ValueError, match="GPU"):
        kernels.sample_tokens(torch.zeros((2, 9)), torch.zeros(2))
    with pytest.raises(ValueError, match="packed rows"):
        tierkv_extend_attention(pool, v, i32, i32, i32, pool, pool, pool, pool, pool, None, pool, None, 4, 1, 1.0)
    with pytest.raises(ValueError, match="GPU"):
        tierkv_extend_attention(rows, v, i32, i32, i32, pool, pool, pool, pool, pool, None, pool, None, 4, 1, 1.0)
