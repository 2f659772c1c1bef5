"""Serving-step calls whose pools, rows or logits pass 2^31 elements: what lies
behind that is read and written where the same call over small tensors has it,
bit for bit."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from paged_tierkv_amd import kernels
from paged_tierkv_amd.tierkv_hip import tierkv_extend_attention

from test_gpu_serving_step import HOT, WARM, gpu, step

pytestmark = pytest.mark.gpu

PAST = 2 ** 31 + 2 ** 20     # elements


@pytest.mark.parametrize("fmt", ["absmax_i8", "ref_u8"])
def test_blocks_far_into_the_pools(device, fmt):
    """Attention over blocks, and row writes into slots, past 2^31 elements of each pool."""
    kv, bs, d = 8, 16, 128
    s = step(81, [40, 3], [300, 200], 16, kv, d, fmt=fmt)
    near = [gpu(a, device) for a in (*s["hot"], *s["warm"], *s["meta"]) if a is not None]
    shift = PAST // (kv * bs * d)

    def far(t):
        out = torch.empty((shift + t.shape[0], *t.shape[1:]), dtype=t.dtype, device=device)
        out[shift:] = t
        return out

    def attend(pools, table):
        hk, hv, wk, wv, *meta = pools
        ks, kz, vs, vz = meta if len(meta) == 4 else (meta[0], None, meta[1], None)
        return tierkv_extend_attention(
            s["q"].to(device), gpu(s["cu"], device), gpu(table, device), gpu(s["states"], device), gpu(s["lengths"], device),
            hk, hv, wk, wv, ks, kz, vs, vz, table.shape[1], s["groups"], s["scaling"], cold_mode="masked",
            seq_num_blocks=gpu(s["nblocks"], device))

    want = attend(near, s["table"])
    pools = [far(t) for t in near]
    assert pools[0].numel() > 2 ** 31 and pools[2].numel() > 2 ** 31
    moved = np.where((s["states"] == HOT) | (s["states"] == WARM), s["table"] + shift, s["table"]).astype(np.int32)
    assert torch.equal(attend(pools, moved), want)

    rows = torch.randn((2, 50, kv, d), dtype=torch.float16, device=device)
    at = torch.randperm(near[0].shape[0] * bs, generator=torch.Generator().manual_seed(0))[:50].int().to(device)
    kernels.write_slots(rows[0], rows[1], at, near[0], near[1])
    kernels.write_slots(rows[0], rows[1], at + shift * bs, pools[0], pools[1])
    for a, b in zip(near[:2], pools[:2]):
        assert torch.equal(b[shift:], a)


def test_packed_rows_past_31_bits(device):
    """Queries, outputs and written K/V rows behind 2^31 elements."""
    heads, kv, d, bs, batch, n = 32, 8, 128, 16, 4096, 130
    rows = batch * n
    assert rows * heads * d > 2 ** 31
    per = -(-n // bs)
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=device)   # noqa: E731
    new = torch.full((batch,), n, dtype=torch.int32, device=device)
    slots = batch * per
    table, states, lengths = i32(batch, per) - 1, i32(batch, per) + 2, i32(batch, per)
    ctl = i32(4)
    ctl[0] = slots
    m = kernels.build_slot_map(new, table, states, lengths, i32(batch), i32(batch),
                               torch.arange(slots, dtype=torch.int32, device=device), ctl, bs, rows)
    assert int(ctl[3]) == 1 and int(m.cu_tokens[-1]) == rows
    # K/V as columns of rows so wide that the last lie past 2^31 elements too.
    wide = torch.empty((rows, 4096 + kv * d), dtype=torch.float16, device=device)
    wide[:, 4096:].normal_()
    k = wide[:, 4096:].view(rows, kv, d)
    assert k.storage_offset() + (rows - 1) * k.stride(0) > 2 ** 31
    hot = torch.empty((2, slots, kv, bs, d), dtype=torch.float16, device=device)
    kernels.write_slots(k, k, m.slots, hot[0], hot[1])
    q = torch.empty((rows, heads, d), dtype=torch.float16, device=device).normal_()
    warm = torch.zeros((1, kv, bs, d), dtype=torch.int8, device=device)
    scale = torch.ones((1, kv), device=device)
    args = (hot[0], hot[1], warm, warm, scale, None, scale, None, per, heads // kv, d ** -0.5)
    out = tierkv_extend_attention(q, m.cu_tokens, table, states, lengths, *args, cold_mode="masked", max_tokens=n)
    for b in (0, batch // 2, batch - 2):
        two = slice(b, b + 2)
        part = slice(b * n, (b + 2) * n)
        cu = torch.tensor([0, n, 2 * n], dtype=torch.int32, device=device)
        alone = tierkv_extend_attention(q[part], cu, table[two].contiguous(), states[two].contiguous(),
                                        lengths[two].contiguous(), *args, cold_mode="masked", max_tokens=n)
        # (cut otherwise: the partials of a tile are added in another order)
        torch.testing.assert_close(out[part], alone, atol=2.0 ** -9, rtol=2.0 ** -9)
    last = m.slots[-1].item()
    assert torch.equal(hot[0][last // bs, :, last % bs], k[-1])


def test_logits_past_31_bits(device):
    batch, vocab = 65536, 33000
    x = torch.empty((batch, vocab), dtype=torch.float16, device=device).normal_(std=2.0)
    assert x.numel() > 2 ** 31
    u = torch.rand(batch, device=device)
    for limits in (dict(top_p=0.9), dict(top_k=30), dict()):
        tok, prob = kernels.sample_tokens(x, u, **limits)
        at = torch.tensor([0, 1, 31000, batch - 2, batch - 1], device=device)
        few, few_prob = kernels.sample_tokens(x[at], u[at], **limits)
        assert torch.equal(tok[at], few) and torch.equal(prob[at], few_prob)
        assert ((tok >= 0) & (tok < vocab)).all()
