"""A serving step over requests of different lengths (oracle; test
infrastructure only): slot maps, attention of several query tokens per
request, and the choice of the next tokens, each as a host program would do
it, one token at a time, in float64 and whole numbers.

The reference serves one sequence per table (append_to_layer,
tierkv_policy.py:1768-1816); ``build_slot_map`` is that append for a batch
whose requests bring different numbers of tokens.  ``extend_attention`` is
``oracle.decode.decode_attention`` with a causal limit per query row.
``sample`` has no counterpart there.  Pinned by: the single-token decode
oracle (one query per request), a torch softmax over dense causal inputs,
and closed forms (tests/test_oracle_serving.py).
"""

from __future__ import annotations

import math

import numpy as np

from . import HOT_STATE
from .decode import gather_sequence_kv

WEIGHT_ONE = float(1 << 42)
ERR_HOT_EMPTY, ERR_TABLE_FULL, ERR_OPEN_STATE, ERR_ROWS = 1, 4, 8, 16


def build_slot_map(new, table, states, lengths, nblocks, opened, free, ctl, block_size, rows):
    """Returns (slots, positions, cu, context) and updates the arrays in
    place, or leaves them alone when the step does not fit."""
    batch, width = table.shape
    held = np.array([int(np.clip(lengths[b, :max(0, min(nblocks[b], width))], 0, block_size).sum())
                     for b in range(batch)], np.int64)
    slots, positions = np.full(rows, -1, np.int32), np.full(rows, -1, np.int32)
    cu = np.zeros(batch + 1, np.int32)
    t, s, ln, nb, op = table.copy(), states.copy(), lengths.copy(), nblocks.copy(), opened.copy()
    top, row, err = int(ctl[0]), 0, 0
    if (new < 0).any() or int(np.maximum(new, 0).astype(np.int64).sum()) > rows:
        err = ERR_ROWS
    out_of_blocks = False
    for b in range(batch):
        n = max(int(new[b]), 0)
        if n == 0:
            cu[b + 1] = row
            continue
        last = nb[b] - 1
        filling = nb[b] > 0 and op[b] != 0 and s[b, last] == HOT_STATE and ln[b, last] < block_size
        if nb[b] > 0 and op[b] != 0 and s[b, last] != HOT_STATE and ln[b, last] < block_size:
            ctl[2] |= ERR_OPEN_STATE
        for i in range(n if not err else 0):
            if not filling or ln[b, nb[b] - 1] == block_size:
                if nb[b] >= width:
                    err |= ERR_TABLE_FULL
                    break
                top -= 1
                if top < 0:
                    out_of_blocks = True
                    t[b, nb[b]] = -1
                else:
                    t[b, nb[b]] = free[top]
                s[b, nb[b]], ln[b, nb[b]] = HOT_STATE, 0
                nb[b] += 1
                filling = True
            slots[row] = t[b, nb[b] - 1] * block_size + ln[b, nb[b] - 1]
            positions[row] = held[b] + i
            ln[b, nb[b] - 1] += 1
            row += 1
        op[b] = int(ln[b, nb[b] - 1] < block_size)
        cu[b + 1] = row
    if out_of_blocks and not err:
        err = ERR_HOT_EMPTY
    if err:
        ctl[2] |= err
        ctl[3] = 0
        return np.full(rows, -1, np.int32), np.full(rows, -1, np.int32), np.zeros(batch + 1, np.int32), held.astype(np.int32)
    table[:], states[:], lengths[:], nblocks[:], opened[:] = t, s, ln, nb, op
    ctl[0], ctl[3] = top, 1
    return slots, positions, cu, (held + new).astype(np.int32)


def extend_attention(query, cu, table, states, lengths, num_blocks, hot_k, hot_v, warm_k, warm_v, k_scale, k_zero,
                     v_scale, v_zero, groups, scaling, warm_format, cold_mode):
    """query [N, H, D]; num_blocks: an int or [B].  Returns (out, mass, logit):
    out [N, H, D] float64 (rows of no request: NaN), mass [N, H, D] the sums
    of p |v|, logit [N, H] the largest scaling * sum |q_d k_d| a row sees (what
    error bounds are made of)."""
    q = np.asarray(query).astype(np.float32).astype(np.float64)   # as the decode oracle takes them
    rows, heads, dim = q.shape
    batch, block_size = table.shape[0], hot_k.shape[2]
    nb = np.broadcast_to(np.asarray(num_blocks, np.int64), (batch,))
    out = np.full((rows, heads, dim), np.nan)
    mass = np.zeros((rows, heads, dim))
    logit = np.zeros((rows, heads))
    for b in range(batch):
        n = int(cu[b + 1] - cu[b])
        if n == 0:
            continue
        out[cu[b]:cu[b + 1]] = 0.0
        if nb[b] == 0:
            continue
        k, v, enters, _ = gather_sequence_kv(table[b], states[b], lengths[b], nb[b], hot_k, hot_v, warm_k, warm_v,
                                             k_scale, k_zero, v_scale, v_zero, warm_format, cold_mode)
        valid = (np.arange(block_size)[None] < np.asarray(lengths[b, :nb[b]])[:, None]).ravel()
        ordinal = np.cumsum(valid) - 1
        held = int(valid.sum())
        for i in range(n):
            seen = np.nonzero(enters & valid & (ordinal <= held - n + i))[0]
            if not len(seen):
                continue
            for h in range(heads):
                kk = k[h // groups][seen].astype(np.float64)
                vv = v[h // groups][seen].astype(np.float64)
                x = kk @ q[cu[b] + i, h] * float(np.float32(scaling))
                p = np.exp(x - x.max())
                p /= p.sum()
                out[cu[b] + i, h] = p @ vv
                mass[cu[b] + i, h] = p @ np.abs(vv)
                logit[cu[b] + i, h] = (np.abs(kk) @ np.abs(q[cu[b] + i, h])).max() * abs(scaling)
    return out, mass, logit


def sample_row(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row: (token, probability).  x: 1-D; the limits as fp32 values."""
    x = np.asarray(x, dtype=np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    f = lambda a: float(np.float32(a))
    if not (x > -np.inf).any():
        return -1, 0.0
    order = np.argsort(-x, kind="stable")
    t = f(temperature)
    if not t > 0:
        return int(order[0]), 1.0
    top = x[order[0]]
    with np.errstate(invalid="ignore", over="ignore"):
        d = np.where(x == top, 0.0, x - top)
        w = np.where(x == top, 1.0, np.where(np.isneginf(d), 0.0, np.exp(d / t)))
    w = np.rint(w * WEIGHT_ONE).astype(np.int64)
    kept = order[:top_k] if top_k > 0 else order
    p = f(top_p)
    if p < 1:
        sums = np.cumsum(w[kept])
        inside = (sums - w[kept]).astype(np.float64) < p * float(sums[-1])
        inside[0] = True
        kept = kept[inside]
    m = f(min_p)
    if m > 0:
        kept = kept[w[kept].astype(np.float64) >= min(m, 1.0) * WEIGHT_ONE]
    kept = np.sort(kept)
    sums = np.cumsum(w[kept])
    target = min(math.floor(float(u) * float(sums[-1])), int(sums[-1]) - 1) if u > 0 else 0
    i = int(np.searchsorted(sums, target, side="right"))
    return int(kept[i]), float(w[kept[i]]) / float(sums[-1])
