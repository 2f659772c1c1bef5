"""What the entry points of rotated, quantized and read-back rows refuse,
before any launch (CPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from paged_tierkv_amd import _lib, kernels

P = 4096        # a non-null, aligned address that no refused call touches


def rotate(**kw):
    a = dict(q=P, qt=512, qh=64, qo=P, k=P, kt=128, kh=64, ko=None, v=P, vt=128, vh=64, dtype=0, pos=P, rows=4, freq=P,
             rot=64, pairs=0, amp=1.0, qw=None, kw=None, wt=0, eps=1e-6, slots=P, hk=P, hv=P, pool=8, heads=8, kv=2, bs=16,
             d=64)
    a.update(kw)
    f = ctypes.c_float
    return _lib.lib().tierkv_rotate_rows(
        a["q"], a["qt"], a["qh"], a["qo"], a["k"], a["kt"], a["kh"], a["ko"], a["v"], a["vt"], a["vh"], a["dtype"], a["pos"],
        a["rows"], a["freq"], a["rot"], a["pairs"], f(a["amp"]), a["qw"], a["kw"], a["wt"], f(a["eps"]), a["slots"], a["hk"],
        a["hv"], a["pool"], a["heads"], a["kv"], a["bs"], a["d"], None)


NO_POOLS = dict(v=None, slots=None, hk=None, hv=None)


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), 1), (dict(qo=None), 1), (dict(k=None), 1), (dict(pos=None), 1), (dict(freq=None), 1), (dict(rows=-1), 1),
    (dict(dtype=2), 1), (dict(wt=1), 1), (dict(rot=65), 1), (dict(rot=66), 1), (dict(rot=-2), 1), (dict(qt=-1), 1),
    (dict(vh=-8), 1), (dict(amp=float("nan")), 1), (dict(eps=-1.0), 1), (dict(eps=float("nan")), 1),
    (dict(eps=float("inf")), 1), (dict(slots=None), 1), (dict(hv=None), 1), (dict(v=None), 1), (NO_POOLS, 1),
    (dict(heads=0), 2), (dict(kv=0), 2), (dict(heads=65536), 2), (dict(d=0), 2), (dict(d=257), 2), (dict(bs=0), 2),
    (dict(bs=65), 2), (dict(pool=0), 2), (dict(pool=1 << 27), 2), (dict(pool=1 << 60), 2), (dict(rows=1 << 26, heads=64), 2),
    (dict(rows=0), 0), (dict(rows=0, q=None, **NO_POOLS), 0),
])
def test_rotate_rows_refusals(kw, code):
    assert rotate(**kw) == code
    assert code == 0 or _lib.last_error()


def quantize(**kw):
    a = dict(k=P, kt=128, kh=64, v=P, vt=128, vh=64, dtype=0, slots=P, rows=4, wk=P, wv=P, pool=8, ks=P, kz=P, vs=P, vz=P,
             fmt=0, kv=2, bs=16, d=64)
    a.update(kw)
    return _lib.lib().tierkv_quantize_rows(
        a["k"], a["kt"], a["kh"], a["v"], a["vt"], a["vh"], a["dtype"], a["slots"], a["rows"], a["wk"], a["wv"], a["pool"],
        a["ks"], a["kz"], a["vs"], a["vz"], a["fmt"], a["kv"], a["bs"], a["d"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(k=None), 1), (dict(slots=None), 1), (dict(wv=None), 1), (dict(ks=None), 1), (dict(kz=None), 1), (dict(dtype=2), 1),
    (dict(fmt=2), 1), (dict(rows=-1), 1), (dict(kt=-1), 1), (dict(kv=0), 2), (dict(kv=65536), 2), (dict(bs=0), 2),
    (dict(bs=65), 2), (dict(d=257), 2), (dict(pool=0), 2), (dict(pool=1 << 27), 2), (dict(pool=1 << 60), 2), (dict(rows=1 << 26), 2),
    (dict(rows=0), 0), (dict(rows=0, k=None, fmt=1, kz=None), 0),
])
def test_quantize_rows_refusals(kw, code):
    assert quantize(**kw) == code


def read(**kw):
    a = dict(start=P, cu=P, rows=8, table=P, states=P, lengths=P, stride=8, snb=None, blocks=8, hk=P, hv=P, hot=4, wk=P, wv=P,
             warm=4, ks=P, kz=P, vs=P, vz=P, fmt=0, ok=P, ov=P, dtype=0, batch=2, kv=2, bs=16, d=64)
    a.update(kw)
    return _lib.lib().tierkv_read_rows(
        a["start"], a["cu"], a["rows"], a["table"], a["states"], a["lengths"], a["stride"], a["snb"], a["blocks"], a["hk"],
        a["hv"], a["hot"], a["wk"], a["wv"], a["warm"], a["ks"], a["kz"], a["vs"], a["vz"], a["fmt"], a["ok"], a["ov"],
        a["dtype"], a["batch"], a["kv"], a["bs"], a["d"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(start=None), 1), (dict(cu=None), 1), (dict(table=None), 1), (dict(ok=None), 1), (dict(rows=-1), 1),
    (dict(batch=0), 1), (dict(blocks=0), 1), (dict(blocks=9), 1), (dict(fmt=2), 1), (dict(dtype=3), 1), (dict(hk=None), 1),
    (dict(hot=0), 1), (dict(wk=None), 1), (dict(warm=0), 1), (dict(vz=None), 1), (dict(kv=0), 2), (dict(bs=0), 2),
    (dict(bs=65), 2), (dict(d=257), 2), (dict(batch=65536), 2), (dict(blocks=1 << 27, stride=1 << 27), 2),
    (dict(blocks=1 << 25, stride=1 << 25), 2), (dict(rows=0), 0), (dict(rows=0, ok=None, ov=None), 0),
])
def test_read_rows_refusals(kw, code):
    assert read(**kw) == code


def test_wrappers_refuse_cpu_tensors():
    rows = torch.zeros((3, 2, 64), dtype=torch.float16)
    v = torch.zeros(3, dtype=torch.int32)
    pool = torch.zeros((2, 2, 16, 64), dtype=torch.float16)
    codes = torch.zeros((2, 2, 16, 64), dtype=torch.int8)
    scale = torch.zeros((2, 2))
    with pytest.raises(ValueError, match="GPU"):
        kernels.rotate_rows(rows, rows, v, torch.zeros(32))
    with pytest.raises(ValueError, match="GPU"):
        kernels.quantize_rows(rows, rows, v, codes, codes, scale, None, scale, None, "absmax_i8")
    with pytest.raises(ValueError, match="warm_format"):
        kernels.quantize_rows(rows, rows, v, codes, codes, scale, None, scale, None, "fp8")
    with pytest.raises(ValueError, match="GPU"):
        kernels.read_rows(v, v, 3, v.view(3, 1), v.view(3, 1), v.view(3, 1), v, pool, pool, codes, codes, scale, None, scale, None)


def prefix(**kw):
    a = dict(q=P, qt=512, qh=64, dtype=0, out=P, cu=P, rows=8, most=8, table=P, states=P, lengths=P, stride=8, snb=None,
             blocks=8, of=P, pt=P, ps=P, pl=P, pstride=16, pnb=None, pblocks=16, prefixes=2, hk=P, hv=P, hot=4, wk=P, wv=P,
             warm=4, ks=P, kz=P, vs=P, vz=P, fmt=0, cold=0, batch=2, heads=8, kv=2, bs=16, d=64, scaling=0.125, ws=P,
             nbytes=1 << 40)
    a.update(kw)
    return _lib.lib().tierkv_prefix_attention(
        a["q"], a["qt"], a["qh"], a["dtype"], a["out"], a["cu"], a["rows"], a["most"], a["table"], a["states"],
        a["lengths"], a["stride"], a["snb"], a["blocks"], a["of"], a["pt"], a["ps"], a["pl"], a["pstride"], a["pnb"],
        a["pblocks"], a["prefixes"], a["hk"], a["hv"], a["hot"], a["wk"], a["wv"], a["warm"], a["ks"], a["kz"], a["vs"],
        a["vz"], a["fmt"], a["cold"], a["batch"], a["heads"], a["kv"], a["bs"], a["d"], ctypes.c_float(a["scaling"]), a["ws"],
        a["nbytes"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), 1), (dict(ws=None), 1), (dict(rows=-1), 1), (dict(batch=0), 1), (dict(heads=7), 1), (dict(blocks=9), 1),
    (dict(scaling=float("inf")), 1), (dict(qt=510), 1), (dict(out=P + 8), 1), (dict(of=None), 1), (dict(pt=None), 1),
    (dict(pl=None), 1), (dict(prefixes=0), 1), (dict(pblocks=0), 1), (dict(pblocks=17), 1), (dict(prefixes=4095), 2),
    (dict(pblocks=1 << 27, pstride=1 << 27), 2), (dict(bs=65), 2), (dict(d=136), 2), (dict(rows=1 << 28), 2),
    (dict(rows=1 << 27, heads=2, nbytes=1 << 62), 2), (dict(nbytes=4096), 4), (dict(rows=0), 0), (dict(most=0), 0),
])
def test_prefix_attention_refusals(kw, code):
    assert prefix(**kw) == code


def test_prefix_workspace_sizes():
    size = lambda *a: _lib.lib().tierkv_prefix_workspace_bytes(*a)   # noqa: E731
    assert size(2, 0, 8, 8, 8, 2, 8, 8, 16, 64) < 0 and size(2, 1, 8, 8, 7, 2, 8, 8, 16, 64) < 0
    assert size(2, 1, 8, 8, 8, 2, 8, 0, 16, 64) < 0
    # geometries that no call takes: blocks longer than a workgroup's list of one request's range among them
    assert size(2, 1, 8, 8, 8, 2, 8, 8, 2000, 64) < 0 and size(2, 1, 8, 8, 8, 2, 8, 8, 65, 64) < 0
    assert size(2, 1, 8, 8, 8, 2, 8, 8, 16, 136) < 0 and size(2, 1, 8, 8, 8, 2, 8, 8, 64, 128) > 0
    small = size(2, 1, 8, 8, 8, 2, 8, 8, 16, 64)
    assert 0 < small <= size(2, 1, 800, 800, 8, 2, 8, 8, 16, 64) and small < size(2, 3, 8, 8, 8, 2, 8, 800, 16, 64)
    assert prefix(nbytes=small - 1, pblocks=8, prefixes=1) == 4
