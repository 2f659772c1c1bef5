"""Rows rotated, quantized and read back where pools and rows pass 2^31
elements, and a prefix whose blocks lie there."""

from __future__ import annotations

import pytest
import torch

from paged_tierkv_amd import kernels
from paged_tierkv_amd.tierkv_hip import tierkv_prefix_attention

pytestmark = pytest.mark.gpu
KV, BS, D = 8, 16, 128
SLOTS = (1 << 31) // (KV * BS * D) + 9        # 2^31 elements and more
HOT, WARM = 0, 1


def test_rows_at_the_end_of_large_pools(device):
    g = torch.Generator(device=device).manual_seed(1)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)   # noqa: E731
    k, v = torch.randn((2, 40, KV, D), generator=g, device=device).half()
    q = torch.randn((40, 16, D), generator=g, device=device).half()
    f = torch.ones(64, device=device) / 7
    at = torch.arange(40, device=device)
    far = (SLOTS - 3) * BS + at
    # HOT: rotated into the last slots of a large pool, and into a small one.
    big = torch.zeros((2, SLOTS, KV, BS, D), dtype=torch.float16, device=device)
    small = torch.zeros((2, 3, KV, BS, D), dtype=torch.float16, device=device)
    for pool, slots in ((big, far), (small, at)):
        kernels.rotate_rows(q, k, at.int(), f, value=v, slots=slots.int(), hot_k=pool[0], hot_v=pool[1])
    assert torch.equal(big[:, SLOTS - 3:], small) and not big[:, :2].any()
    # WARM, of both formats, and tokens read back from both tiers.
    for fmt, kind in (("absmax_i8", torch.int8), ("ref_u8", torch.uint8)):
        i8 = fmt == "absmax_i8"
        meta = lambda n: torch.zeros((n, KV), device=device) if i8 else torch.zeros((n, KV, BS, 1), dtype=torch.float16, device=device)   # noqa: E731,B023
        large = [torch.zeros((SLOTS, KV, BS, D), dtype=kind, device=device) for _ in range(2)]
        codes = [torch.zeros((3, KV, BS, D), dtype=kind, device=device) for _ in range(2)]
        ml, ms = [meta(SLOTS) for _ in range(4)], [meta(3) for _ in range(4)]
        for c, m, slots in ((large, ml, far), (codes, ms, at)):
            kernels.quantize_rows(k, v, slots.int(), *c, *m, warm_format=fmt)
        assert all(torch.equal(a[SLOTS - 3:], b) for a, b in zip(large, codes))
        states, lens = i32(WARM, HOT, WARM)[None], i32(16, 16, 8)[None]
        both = []
        for c, m, h, table in ((large, ml, big, i32(SLOTS - 3, SLOTS - 2, SLOTS - 1)[None]), (codes, ms, small, i32(0, 1, 2)[None])):
            both.append(kernels.read_rows(i32(3), i32(0, 37), 37, table, states, lens, None, h[0], h[1], *c, *m))
            own = torch.zeros((1, 1), dtype=torch.int32, device=device)
            both[-1] += (tierkv_prefix_attention(q[:1], i32(0, 1), own, own, own, h[0], h[1], *c, *m, 1, 2, 0.1, i32(0), table,
                                                 states, lens, cold_mode="masked"),)
        assert all(torch.equal(a, b) for a, b in zip(*both))
        del large, ml


def test_rows_past_2_31_elements(device):
    """A step of rows whose outputs have more than 2^31 elements."""
    rows, heads = (1 << 31) // (256 * 64) + 5, 256
    x = torch.zeros((1, heads, 64), dtype=torch.float16, device=device)
    x[..., 0], x[..., 32] = 1, 2
    k = x[:, :1]
    pos = torch.zeros(rows, dtype=torch.int32, device=device)
    pos[-1] = 1
    q, kk = kernels.rotate_rows(x.expand(rows, heads, 64), k.expand(rows, 1, 64), pos, torch.full((32,), torch.pi / 2, device=device))
    assert torch.equal(q[-2], x[0]) and torch.equal(kk[-2], k[0])
    turned = torch.zeros_like(x[0])
    turned[:, 0], turned[:, 32] = -2, 1                    # a quarter turn
    assert (q[-1].float() - turned.float()).abs().max() <= 2.0 ** -20      # (the frequency is pi / 2 in 32 bits)
    assert torch.equal(q[rows // 2], x[0]) and torch.equal(q[0], x[0])
