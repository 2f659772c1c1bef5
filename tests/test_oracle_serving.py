"""The serving-step oracle against independent statements of the same things:
the single-token decode oracle, a dense causal softmax in torch, the
reference's append rule, and closed forms of the sampling filters."""

from __future__ import annotations

import numpy as np
import torch

from oracle import codec
from oracle import decode as odecode
from oracle import serving


def _pools(rng, slots, kv, bs, d):
    k, v = (rng.standard_normal((slots, kv, bs, d)).astype(np.float16) for _ in range(2))
    qk, sk = codec.quantize_absmax_i8(k)
    qv, sv = codec.quantize_absmax_i8(v)
    return k, v, qk, qv, sk, None, sv, None


def test_one_query_per_request_is_the_decode_oracle():
    rng = np.random.default_rng(0)
    B, kv, G, D, bs, nblk = 3, 2, 2, 16, 16, 5
    pools = _pools(rng, 20, kv, bs, D)
    table = rng.permutation(20)[:B * nblk].reshape(B, nblk).astype(np.int32)
    states = rng.integers(0, 3, (B, nblk)).astype(np.int32)
    lengths = rng.integers(0, bs + 1, (B, nblk)).astype(np.int32)
    q = rng.standard_normal((B, kv * G, D))
    for cold in ("masked", "zero_logit"):
        out, mass, _ = serving.extend_attention(q, np.arange(B + 1), table, states, lengths, nblk, *pools, G, 0.25,
                                                "absmax_i8", cold)
        want = odecode.decode_attention(q, table, states, lengths, nblk, *pools, G, 0.25, warm_format="absmax_i8",
                                        cold_mode=cold)
        np.testing.assert_allclose(out, want, rtol=1e-6, atol=1e-9)
        assert (np.abs(out) <= mass + 1e-12).all()


def test_hot_tokens_are_plain_causal_attention():
    rng = np.random.default_rng(1)
    kv, G, D, bs, held, n = 2, 3, 16, 16, 41, 7
    nblk = 3
    pools = _pools(rng, nblk, kv, bs, D)
    table, states = np.arange(nblk, dtype=np.int32)[None], np.zeros((1, nblk), np.int32)
    lengths = np.array([[16, 16, 9]], np.int32)
    q = rng.standard_normal((n, kv * G, D))
    out, _, _ = serving.extend_attention(q, np.array([0, n]), table, states, lengths, nblk, *pools, G, 0.25,
                                         "absmax_i8", "masked")
    k, v = (torch.from_numpy(p.transpose(1, 0, 2, 3).reshape(kv, -1, D)[:, :held].astype(np.float64))
            .repeat_interleave(G, 0) for p in pools[:2])
    x = torch.einsum("nhd,htd->hnt", torch.from_numpy(q.astype(np.float32).astype(np.float64)), k) * 0.25
    hide = torch.arange(held)[None] > (held - n + torch.arange(n))[:, None]
    p = torch.softmax(x.masked_fill(hide[None], float("-inf")), -1)
    np.testing.assert_allclose(out, torch.einsum("hnt,htd->nhd", p, v).numpy(), rtol=1e-6, atol=1e-9)


def test_slot_map_fills_the_open_block_then_pops_in_order():
    table = np.full((3, 4), -1, np.int32)
    states, lengths = np.full((3, 4), 2, np.int32), np.zeros((3, 4), np.int32)
    table[0, 0], states[0, 0], lengths[0, 0] = 7, 0, 3
    table[1, 0], states[1, 0], lengths[1, 0] = 5, 0, 2
    nblocks, opened = np.array([1, 1, 0], np.int32), np.array([1, 0, 0], np.int32)
    free, ctl = np.array([9, 8, 6, 4, 3], np.int32), np.array([5, 0, 0, 0], np.int32)
    slots, pos, cu, ctx = serving.build_slot_map(np.array([3, 1, 6], np.int32), table, states, lengths, nblocks, opened,
                                                 free, ctl, 4, 12)
    #            open block, then block 3 | block 4 (the open flag is off) | blocks 6 and 8
    assert slots.tolist() == [31, 12, 13, 16, 24, 25, 26, 27, 32, 33, -1, -1]
    assert pos.tolist() == [3, 4, 5, 2, 0, 1, 2, 3, 4, 5, -1, -1]
    assert cu.tolist() == [0, 3, 4, 10] and ctx.tolist() == [6, 3, 6]
    assert nblocks.tolist() == [2, 2, 2] and opened.tolist() == [1, 1, 1] and ctl.tolist() == [1, 0, 0, 1]
    assert lengths[0].tolist() == [4, 2, 0, 0] and lengths[2].tolist() == [4, 2, 0, 0]
    before = table.copy()
    slots, _, cu, _ = serving.build_slot_map(np.array([9, 0, 0], np.int32), table, states, lengths, nblocks, opened,
                                             free, ctl, 4, 12)
    assert (slots == -1).all() and cu.tolist() == [0] * 4 and (table == before).all()
    assert ctl[2] == serving.ERR_HOT_EMPTY and ctl[3] == 0


def test_sampling_filters_by_closed_forms():
    x = np.log(np.array([0.1, 0.4, 0.2, 0.2, 0.1]))
    draw = lambda u, **kw: serving.sample_row(x, u, **kw)[0]
    assert [draw(u) for u in (0.0, 0.05, 0.15, 0.45, 0.55, 0.65, 0.75, 0.95)] == [0, 0, 1, 1, 2, 2, 3, 4]
    assert [draw(u, top_k=2) for u in (0.0, 0.6, 0.7, 0.999)] == [1, 1, 2, 2]      # the first of the equal 0.2
    assert [draw(u, top_p=0.5) for u in (0.0, 0.6, 0.7, 0.999)] == [1, 1, 2, 2]    # 0.4 < 0.5 <= 0.6
    assert [draw(u, top_p=0.3) for u in (0.0, 0.999)] == [1, 1]
    assert [draw(u, min_p=0.4) for u in (0.0, 0.6, 0.999)] == [1, 2, 3]
    assert draw(0.7, temperature=0.0) == 1 and draw(0.3, top_p=0.0) == 1
    assert serving.sample_row(np.full(4, -np.inf), 0.5) == (-1, 0.0)
    assert serving.sample_row(np.array([np.nan, 1.0, np.inf, 2.0]), 0.9) == (2, 1.0)
    counts = np.bincount([draw(u) for u in (np.arange(1000) + 0.5) / 1000], minlength=5)
    assert np.abs(counts - [100, 400, 200, 200, 100]).max() <= 1
