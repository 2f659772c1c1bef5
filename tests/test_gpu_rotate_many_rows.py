"""Rotation of more rows than a wave per (row, head) can have in one launch:
each row gives the bits that it gives among fewer."""

from __future__ import annotations

import pytest
import torch

from paged_tierkv_amd import kernels

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,rot,norm", [(6, 4, True), (16, 16, False)])      # any layout; 16-byte chunks
def test_rows_times_heads_past_2_26(device, d, rot, norm):
    rows, part = (1 << 26) // 3 + 1001, 1 << 22                               # a row has three heads
    print(f"[rotate] {rows} rows of 3 heads of {d}", flush=True)
    g = torch.Generator(device=device).manual_seed(d)
    x = torch.randn((rows, 3, d), generator=g, device=device).half()
    pos = torch.randint(-1, 100000, (rows,), generator=g, device=device, dtype=torch.int32)
    f = 10000.0 ** (-torch.arange(0, rot, 2, device=device) / rot)
    w = torch.ones(d, device=device) * 0.75 if norm else None
    slots = torch.full((rows,), -1, dtype=torch.int32, device=device)
    slots[-96:] = torch.randperm(96, device=device).int()
    pools = torch.zeros((2, 2, 6, 1, 16, d), dtype=torch.float16, device=device)
    call = lambda a, b, p, out: kernels.rotate_rows(                          # noqa: E731
        x[a:b, :1], x[a:b, 1:2], pos[a:b], f, q_weight=w, k_weight=w, value=x[a:b, 2:], slots=slots[a:b], hot_k=p[0],
        hot_v=p[1], q_out=out)
    got, want = torch.full((rows, 1, d), 7.0, dtype=torch.float16, device=device), None
    call(0, rows, pools[0], got)
    for a in range(0, rows, part):
        b = min(a + part, rows)
        want = torch.full((b - a, 1, d), 7.0, dtype=torch.float16, device=device)
        call(a, b, pools[1], want)
        assert torch.equal(got[a:b], want), a
    assert torch.equal(pools[0], pools[1]) and pools[0].any()
