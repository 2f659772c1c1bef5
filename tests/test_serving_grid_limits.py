"""Calls whose launch would have 2^32 threads or more in a dimension, which the
device does not take, are refused before the first launch (CPU; the addresses
are never touched)."""

from __future__ import annotations

import ctypes

import pytest

from paged_tierkv_amd import _lib

P = 4096


@pytest.mark.parametrize("rows,kv,d,wide", [
    (1 << 25, 8, 128, True),          # 2^32 threads of eight elements
    (1 << 22, 8, 128, False),         # 2^32 threads of one element (an odd stride)
    ((1 << 31) - 1, 1, 256, True),
])
def test_write_slots(rows, kv, d, wide):
    rc = _lib.lib().tierkv_write_slots(P, kv * d + (0 if wide else 1), d, P, kv * d, d, 0, P, rows, P, P, 64, kv, 16, d, None)
    assert rc == _lib.TIERKV_ERR_UNSUPPORTED and "too large" in _lib.last_error()


@pytest.mark.parametrize("rows,batch,heads,kv", [(1 << 26, 1, 32, 32), (1 << 22, 4096, 512, 512), ((1 << 27) - 5, 7, 32, 8)])
def test_extend_attention(rows, batch, heads, kv):
    lib = _lib.lib()
    need = lib.tierkv_extend_workspace_bytes(batch, rows, rows, heads, kv, 8, 16, 8)
    assert need > 0
    rc = lib.tierkv_extend_attention(P, 0, 0, 0, P, P, rows, rows, P, P, P, 8, None, 8, P, P, 4, P, P, 4, P, P, P, P, 0, 0,
                                     batch, heads, kv, 16, 8, ctypes.c_float(0.125), P, need, None)
    assert rc == _lib.TIERKV_ERR_UNSUPPORTED and "grid" in _lib.last_error()
