"""The shared-prompt oracle against independent forms (CPU)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import codec, serving, shared_prompt


def test_rotation_is_transformers_and_a_complex_product():
    from transformers.models.llama.modeling_llama import apply_rotary_pos_emb

    rng = np.random.default_rng(1)
    x = rng.standard_normal((9, 3, 16)).astype(np.float32)
    f = 10000.0 ** (-np.arange(0, 16, 2) / 16)
    pos = np.arange(5, 14)
    y, _ = shared_prompt.rotate(x, pos, f)
    angle = torch.from_numpy(pos[:, None] * f)
    emb = torch.cat([angle, angle], -1)[None]
    t = torch.from_numpy(x).double().transpose(0, 1)[None]
    want, _ = apply_rotary_pos_emb(t, t, emb.cos(), emb.sin())
    np.testing.assert_allclose(y, want[0].transpose(0, 1).numpy(), atol=1e-12)
    y, _ = shared_prompt.rotate(x, pos, f, interleaved=True)
    z = (x[..., 0::2] + 1j * x[..., 1::2]) * np.exp(1j * pos[:, None, None] * f)
    np.testing.assert_allclose(y[..., 0::2] + 1j * y[..., 1::2], z, atol=1e-12)
    w = rng.standard_normal(16)
    y, _ = shared_prompt.rotate(x, 0 * pos, f, weight=w, eps=0.0)
    np.testing.assert_allclose((y / w) ** 2 @ np.ones(16), 16.0, rtol=1e-6)


@pytest.mark.parametrize("fmt", ["absmax_i8", "ref_u8"])
def test_whole_blocks_are_the_block_codec(fmt):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((32, 2, 8)).astype(np.float16)
    codes = np.zeros((3, 2, 16, 8), np.uint8 if fmt == "ref_u8" else np.int8)
    scale = np.full((3, 2, 16, 1), 3, np.float16) if fmt == "ref_u8" else np.full((3, 2), 9, np.float32)
    zero = np.zeros((3, 2, 16, 1), np.float16) if fmt == "ref_u8" else None
    slots = np.concatenate([2 * 16 + np.arange(16), np.arange(16)]).astype(np.int32)
    shared_prompt.quantize_rows(x, slots, codes, scale, zero)
    tiles = x.reshape(2, 16, 2, 8).transpose(0, 2, 1, 3)[::-1]
    want = codec.quantize_ref_u8(tiles) if fmt == "ref_u8" else codec.quantize_absmax_i8(tiles)
    np.testing.assert_array_equal(codes[[0, 2]], want[0])
    np.testing.assert_array_equal(scale[[0, 2]], want[1])
    assert (codes[1] == 0).all()


def test_a_grown_absmax_block_stays_within_a_step():
    """Token by token: no held value moves by more than half a step of each
    scale it went through."""
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((16, 1, 8)) * np.exp(rng.standard_normal((16, 1, 1)))).astype(np.float16)
    codes, scale = np.zeros((1, 1, 16, 8), np.int8), np.zeros((1, 1), np.float32)
    moved = 0.0
    for i in range(16):
        before = float(scale[0, 0])
        shared_prompt.quantize_rows(x[i:i + 1], np.array([i], np.int32), codes, scale, None)
        if scale[0, 0] != before:
            moved += float(scale[0, 0]) / 2
        moved = max(moved, float(scale[0, 0]) / 2)
        err = np.abs(codes[0, 0, :i + 1] * float(scale[0, 0]) - x[:i + 1, 0].astype(np.float64))
        assert err.max() <= moved * (1 + 1e-5)
    assert scale[0, 0] == np.float32(np.abs(x.astype(np.float32)).max() / np.float32(127))


@pytest.mark.parametrize("cold", ["masked", "zero_logit"])
def test_prefix_attention_is_extend_attention_with_the_prefix_in_every_row(cold):
    rng = np.random.default_rng(4)
    kv, bs, d, heads = 2, 4, 8, 4
    hot = rng.standard_normal((2, 12, kv, bs, d)).astype(np.float16)
    (wk, ks), (wv, vs) = (codec.quantize_absmax_i8(rng.standard_normal((5, kv, bs, d)).astype(np.float16)) for _ in range(2))
    pre = (np.array([[3, 1, 0], [7, 4, -1]]), np.array([[0, 1, 0], [0, 1, 2]]), np.array([[4, 4, 2], [4, 4, 3]]), [3, 3])
    mine = (np.array([[5, 6], [2, 8], [9, 10]]), np.array([[0, 0], [1, 0], [0, 0]]), np.array([[4, 1], [4, 3], [2, 0]]), [2, 2, 1])
    cu, member = np.array([0, 2, 5, 6]), [1, 0, -1]
    q = rng.standard_normal((6, heads, d)).astype(np.float16)
    got = shared_prompt.prefix_attention(q, cu, mine, member, pre, *hot, wk, wv, ks, None, vs, None, 2, 0.4, "absmax_i8", cold)
    joined = [[], [], []]
    for b, g in enumerate(member):
        for out, p, m in zip(joined, pre, mine):
            out.append(([] if g < 0 else list(p[g][:pre[3][g]])) + list(m[b][:mine[3][b]]))
    nb = [len(x) for x in joined[0]]
    table, states, lengths = (np.array([x + [0] * (5 - len(x)) for x in rows]) for rows in joined)
    want = serving.extend_attention(q, cu, table, states, lengths, nb, *hot, wk, wv, ks, None, vs, None, 2, 0.4, "absmax_i8", cold)
    for a, b in zip(got, want):
        np.testing.assert_allclose(a, b, rtol=1e-10, atol=1e-12)
