"""Operators of a step whose requests share prompts (oracle; test
infrastructure only): norms and rotation of packed rows, rows quantized as they
are written, rows read back, and attention over a shared prefix, each as a host
program would do it, one row at a time, in float64.

The reference rotates a model's q and k with transformers' apply_rotary_pos_emb
(modeling_llama.py:376-377), quantizes whole blocks (write_warm_block,
tierkv_policy.py:969-1002) and reads one sequence back (reconstruct_layer,
1818-1841); norms and shared prefixes have no counterpart there.  Pinned by:
transformers' rotation and a complex product, the block codecs of
``oracle.codec``, ``oracle.serving.extend_attention`` over tables in which every
request holds the prefix itself (tests/test_oracle_shared_prompt.py).
"""

from __future__ import annotations

import numpy as np

from . import COLD_STATE, HOT_STATE, WARM_STATE
from .codec import quantize_ref_u8
from .decode import gather_sequence_kv


def rotate(x, positions, inv_freq, weight=None, eps=1e-6, scaling=1.0, interleaved=False):
    """x [N, heads, D] -> (rotated rows, size): float64, size what error bounds
    are made of, |x'_a| + |x'_b| of each element's pair.  Rows of negative
    positions are NaN."""
    x = np.asarray(x).astype(np.float32).astype(np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + float(np.float32(eps))) * np.asarray(weight).astype(np.float64)
    f = np.asarray(inv_freq).astype(np.float64)
    half, y, size = len(f), x.copy(), np.abs(x)
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    for r, pos in enumerate(np.asarray(positions)):
        if pos < 0:
            y[r] = np.nan
            continue
        c, s = np.cos(float(pos) * f) * float(scaling), np.sin(float(pos) * f) * float(scaling)
        y[r][:, a] = x[r][:, a] * c - x[r][:, b] * s
        y[r][:, b] = x[r][:, b] * c + x[r][:, a] * s
        size[r][:, a] = size[r][:, b] = (np.abs(x[r][:, a]) + np.abs(x[r][:, b])) * abs(scaling)
    return y, size


def quantize_rows(rows, slots, codes, scale, zero):
    """Writes rows [N, kv, D] (fp16) into codes [slots, kv, bs, D] and their
    metadata in place; zero None: the absmax format."""
    bs, total = codes.shape[2], codes.shape[0] * codes.shape[2]
    x = np.asarray(rows).astype(np.float16)
    todo = [r for r in range(len(slots)) if 0 <= slots[r] < total]
    if zero is not None:
        for r in todo:
            q, s, z = quantize_ref_u8(x[r])
            at = (slots[r] // bs, slice(None), slots[r] % bs)
            codes[at], scale[at], zero[at] = q, s, z
        return
    f32 = np.float32
    for block in sorted({int(slots[r]) // bs for r in todo}):
        mine = [r for r in todo if slots[r] // bs == block]
        first = min(int(slots[r]) % bs for r in mine)
        for h in range(codes.shape[1]):
            old = f32(scale[block, h]) if first else f32(0)
            peak = f32(max(np.abs(x[r, h].astype(f32)).max() for r in mine))
            s = max(abs(old), f32(peak / f32(127)))
            with np.errstate(invalid="ignore", divide="ignore"):
                code = lambda v: np.clip(np.rint(v / s), -127, 127) if s != 0 else np.zeros_like(v)   # noqa: E731
                if first and s != old:
                    codes[block, h, :first] = code(codes[block, h, :first].astype(f32) * old)
                for r in mine:
                    codes[block, h, slots[r] % bs] = code(x[r, h].astype(f32))
            scale[block, h] = s


def read_rows(start, cu, rows, table, states, lengths, nblocks, hot_k, hot_v, warm_k, warm_v, k_scale, k_zero, v_scale,
              v_zero, warm_format):
    """K, V rows [rows, kv, D] float32 (rows of no request: NaN)."""
    kv, bs, d = hot_k.shape[1:]
    out = np.full((2, rows, kv, d), np.nan, np.float32)
    for b in range(len(start)):
        n = cu[b + 1] - cu[b]
        if n <= 0:
            continue
        out[:, cu[b]:cu[b + 1]] = 0
        states_b = np.array(states[b])
        for i in range(nblocks[b]):      # what is out of range reads as evicted
            pool = hot_k if states_b[i] == HOT_STATE else warm_k
            if states_b[i] not in (HOT_STATE, WARM_STATE) or not 0 <= table[b, i] < len(pool):
                states_b[i] = COLD_STATE
        if not nblocks[b]:
            continue
        k, v, _, _ = gather_sequence_kv(table[b], states_b, lengths[b], nblocks[b], hot_k, hot_v, warm_k, warm_v, k_scale,
                                        k_zero, v_scale, v_zero, warm_format, "zero_logit")
        valid = (np.arange(bs)[None] < np.asarray(lengths[b, :nblocks[b]])[:, None]).ravel()
        s = max(int(start[b]), 0)
        for o, x in zip(out, (k, v)):
            part = x[:, valid][:, s:s + n].transpose(1, 0, 2)
            o[cu[b]:cu[b] + len(part)] = part
    return out[0], out[1]


def prefix_attention(query, cu, tables, prefix_of, prefix_tables, hot_k, hot_v, warm_k, warm_v, k_scale, k_zero, v_scale,
                     v_zero, groups, scaling, warm_format, cold_mode):
    """tables and prefix_tables: (table, states, lengths, nblocks).  Returns
    (out, mass, logit) as ``oracle.serving.extend_attention``."""
    q = np.asarray(query).astype(np.float32).astype(np.float64)
    rows, heads, dim = q.shape
    bs = hot_k.shape[2]
    out, mass, logit = np.full((rows, heads, dim), np.nan), np.zeros((rows, heads, dim)), np.zeros((rows, heads))

    def tokens(t, b):
        table, states, lengths, nblocks = t
        if b < 0 or nblocks[b] == 0:
            z = np.zeros((hot_k.shape[1], 0, dim))
            return z, z, np.zeros(0, int), 0
        k, v, enters, _ = gather_sequence_kv(table[b], states[b], lengths[b], nblocks[b], hot_k, hot_v, warm_k, warm_v,
                                             k_scale, k_zero, v_scale, v_zero, warm_format, cold_mode)
        valid = (np.arange(bs)[None] < np.asarray(lengths[b, :nblocks[b]])[:, None]).ravel()
        keep = valid & enters
        return k[:, keep].astype(np.float64), v[:, keep].astype(np.float64), (np.cumsum(valid) - 1)[keep], int(valid.sum())

    for b in range(len(cu) - 1):
        n = int(cu[b + 1] - cu[b])
        if n <= 0:
            continue
        out[cu[b]:cu[b + 1]] = 0.0
        pk, pv, _, _ = tokens(prefix_tables, int(prefix_of[b]) if 0 <= prefix_of[b] < len(prefix_tables[3]) else -1)
        k, v, ordinal, held = tokens(tables, b)
        for i in range(n):
            see = ordinal <= held - n + i
            for h in range(heads):
                kk = np.concatenate([pk[h // groups], k[h // groups][see]])
                vv = np.concatenate([pv[h // groups], v[h // groups][see]])
                if not len(kk):
                    continue
                x = kk @ q[cu[b] + i, h] * float(np.float32(scaling))
                p = np.exp(x - x.max())
                p /= p.sum()
                out[cu[b] + i, h] = p @ vv
                mass[cu[b] + i, h] = p @ np.abs(vv)
                logit[cu[b] + i, h] = (np.abs(kk) @ np.abs(q[cu[b] + i, h])).max() * abs(scaling)
    return out, mass, logit
