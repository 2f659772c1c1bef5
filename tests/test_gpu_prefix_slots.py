"""Steps whose tokens' heads lie in two tiles of a prefix: with 3, 6 or 7 heads
per kv head a tile of 256 rows ends inside a token, and the next prefix's tiles
follow (bounds as in test_gpu_prefix_attention.py)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from paged_tierkv_amd.tierkv_hip import DecodeWorkspace
from test_gpu_prefix_attention import check, launch, step, tensors

pytestmark = pytest.mark.gpu

CASES = [
    # requests, new tokens of each, heads, kv, d
    (100, [1], 6, 2, 64),            # 300 rows, the 86th token's in both tiles
    (90, [1], 12, 2, 128),           # 540: tokens in both at each border
    (80, [1], 7, 1, 64),             # 560
    (40, [3], 6, 2, 128),            # 360, borders inside a request
    (60, [5, 1, 3, 0], 7, 1, 40),    # drafts of several lengths
    (70, [9, 2], 6, 1, 64),          # two tiles of 32 rows of a request's own beside them
]


@pytest.mark.parametrize("requests,new,heads,kv,d", CASES)
@pytest.mark.parametrize("fmt,cold,dtype", [("absmax_i8", "masked", torch.float16), ("ref_u8", "zero_logit", torch.bfloat16)])
@pytest.mark.parametrize("order", ["one_prefix_after_the_other", "mixed"])
def test_tokens_in_two_tiles(device, requests, new, heads, kv, d, fmt, cold, dtype, order):
    """Two prefixes of as many requests each, and a third of few."""
    print(f"[prefix] 2 x {requests} x {new} tokens, {heads}/{kv} x {d}, {fmt} {cold}, {order}", flush=True)
    member = [0] * requests + [1] * requests + [2, 2, -1]
    if order == "mixed":
        member = list(np.random.default_rng(requests).permutation(member))
    count = [new[i % len(new)] for i in range(len(member))]
    held = [n + (i * 7) % 23 for i, n in enumerate(count)]
    s = step(requests + heads, [90, 41, 200], member, count, held, heads, kv, d, 16, fmt, dtype)
    t = tensors(s, device)
    ws = DecodeWorkspace(device)
    out = torch.full_like(t["q"], 7.0)
    launch(t, s, cold, workspace=ws, max_tokens=max(new), out=out)
    assert ws.error_word() == 0
    check(out, s, cold)
    assert (out[s["cu"][-1]:] == 7.0).all()
