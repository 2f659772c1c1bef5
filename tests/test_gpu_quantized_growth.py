"""How far the values of an absmax block move while it is filled token by token
and its scale grows (quantize_rows).

A token's codes are rounded when it is written and once more whenever the scale
grows after it: each time by at most half a step of the scale then, s / 2, which
is at most half of the last one.  Written at position p of b tokens, its values
see b - p scales at most: they end within (b - p) / 2 steps of the last scale.
The products and quotients are 32-bit, two or three roundings each time of a
magnitude of at most 127 steps: 3 * 127 * 2^-24 steps more.
"""

from __future__ import annotations

import pytest
import torch

from paged_tierkv_amd import kernels

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bs", [16, 64])
@pytest.mark.parametrize("d", [128, 30])                       # 16-byte chunks; any layout
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("growth", [0.0, 0.013, 0.1, 0.5])     # of a token's magnitude over the one before
def test_values_of_a_block_filled_token_by_token(device, bs, d, dtype, growth):
    print(f"[growth] blocks of {bs}, {d} dims, {dtype}, tokens {1 + growth} times the one before", flush=True)
    kv, blocks = 3, 2
    g = torch.Generator(device=device).manual_seed(bs + d)
    size = torch.clamp((1 + growth) ** torch.arange(bs, device=device, dtype=torch.float32), max=4096.0)
    x = (torch.randn((2, blocks, bs, kv, d), generator=g, device=device) * size[:, None, None]).to(dtype)
    codes = [torch.zeros((blocks, kv, bs, d), dtype=torch.int8, device=device) for _ in range(2)]
    scales = [torch.zeros((blocks, kv), device=device) for _ in range(2)]
    for p in range(bs):
        slots = torch.arange(blocks, dtype=torch.int32, device=device) * bs + p
        kernels.quantize_rows(x[0, :, p], x[1, :, p], slots, *codes, scales[0], None, scales[1], None, "absmax_i8")
    steps = (bs - torch.arange(bs, device=device, dtype=torch.float64)) * (0.5 + 3 * 127 * 2.0 ** -24)
    for rows, q, s in zip(x, codes, scales):
        rows = rows.half().double().transpose(1, 2)            # [blocks, kv, tokens, d]
        s = s.double()[:, :, None, None]
        torch.testing.assert_close(s[:, :, 0, 0], rows.abs().amax((2, 3)) / 127, rtol=2.0 ** -23, atol=0)
        off = (q.double() * s - rows).abs() / s
        print(f"[growth] up to {off.max():.2f} steps, {(off / steps[:, None]).max():.2f} of the bound", flush=True)
        assert (off <= steps[:, None]).all()
