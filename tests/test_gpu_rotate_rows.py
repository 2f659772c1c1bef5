"""Norms and rotation of packed rows on the GPU against the row-by-row float64
oracle (oracle/shared_prompt.py).

Error bound of an element, from the oracle's S = A (|x'_a| + |x'_b|) of its pair:
* the angle's fraction of a turn, at most a half, becomes 32 bits (half a step,
  2^-26 turns, 9.4e-8 in the angle) and its sine and cosine are off by a few
  2^-24: together below 2^-22, so 2^-22 S;
* the mean square is a sum of D products in 32 bits, off by at most D 2^-24 of
  itself, its root by half of that, the root, the division and the products by
  a few 2^-24: (D / 2 + 12) 2^-24 S;
* the output's rounding, half a step of its type, 2^-25 (fp16 below its normal range).
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import shared_prompt
from paged_tierkv_amd import kernels

pytestmark = pytest.mark.gpu
EPS = 1e-6


def bound(y, size, d, dtype):
    return size * (2.0 ** -22 + (d / 2 + 12) * 2.0 ** -24) + np.abs(y) * torch.finfo(dtype).eps / 2 + 2.0 ** -25


def close(got, y, size, dtype, what):
    got = got.double().cpu().numpy()
    rows = ~np.isnan(y).reshape(len(y), -1).any(1)
    err, tol = np.abs(got - y)[rows], bound(y, size, y.shape[-1], dtype)[rows]
    print(f"[rotate] {what}: {(err / tol).max() if err.size else 0:.2f} of its bound", flush=True)
    assert (err <= tol).all()


def step(seed, rows, heads, kv, d, rot, dtype, norm, far=5000, pad=2):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((rows + pad, (heads + 2 * kv) * d), generator=g) * 1.5).to(dtype)
    rng = np.random.default_rng(seed)
    pos = np.full(rows + pad, -1, np.int32)
    pos[:rows] = rng.integers(0, far, rows)
    if rows > 3:
        pos[1], pos[2] = 0, -3               # the first token; a row of no request in between
    f = (10000.0 ** (-np.arange(0, rot, 2) / max(rot, 1))).astype(np.float32)
    w = [(1 + 0.4 * torch.randn(d, generator=g)).to(dtype) if norm else None for _ in range(2)]
    cut = lambda t, a, n: t[:, a * d:(a + n) * d].view(rows + pad, n, d)   # noqa: E731
    return dict(x=x, q=lambda t: cut(t, 0, heads), k=lambda t: cut(t, heads, kv), v=lambda t: cut(t, heads + kv, kv), pos=pos,
                f=f, w=w, rows=rows + pad, heads=heads, kv=kv, d=d, dtype=dtype)


def up(a, device):
    return None if a is None else (a if torch.is_tensor(a) else torch.from_numpy(a)).to(device)


def expect(s, pairs, scaling=1.0):
    w = [None if w is None else w.float().numpy() for w in s["w"]]
    return [shared_prompt.rotate(s[n](s["x"]).float().numpy(), s["pos"], s["f"], wi, EPS, scaling, pairs)
            for n, wi in zip("qk", w)]


GEOMETRIES = [
    # rows, heads, kv, d, rot
    (1, 1, 1, 64, 64), (5, 8, 2, 128, 128), (37, 14, 2, 64, 32), (130, 32, 8, 128, 128), (9, 6, 3, 96, 96),
    (9, 4, 2, 256, 128), (9, 4, 4, 8, 8), (7, 4, 1, 40, 16), (7, 4, 1, 40, 24), (11, 3, 1, 30, 10), (300, 4, 2, 80, 80),
    (6, 5, 5, 72, 0), (1030, 3, 1, 128, 64),
]


@pytest.mark.parametrize("rows,heads,kv,d,rot", GEOMETRIES)
@pytest.mark.parametrize("dtype,norm,pairs", [(torch.float16, False, False), (torch.bfloat16, True, False),
                                              (torch.float16, True, True), (torch.bfloat16, False, True)])
def test_rows_match_the_oracle(device, rows, heads, kv, d, rot, dtype, norm, pairs):
    print(f"[rotate] {rows} rows {heads}/{kv} x {d}, {rot} rotated", flush=True)
    s = step(rows + d, rows, heads, kv, d, rot, dtype, norm)
    x = s["x"].to(device)
    wq, wk = (up(w, device) for w in s["w"])
    q_out = torch.full((s["rows"], heads, d), 7.0, dtype=dtype, device=device)
    k_out = torch.full((s["rows"], kv, d), 7.0, dtype=dtype, device=device)
    got = kernels.rotate_rows(s["q"](x), s["k"](x), up(s["pos"], device), up(s["f"], device), q_weight=wq, k_weight=wk,
                              eps=EPS, attention_scaling=1.25, interleaved=pairs, q_out=q_out, k_out=k_out)
    assert got[0] is q_out and got[1] is k_out
    out = torch.from_numpy(s["pos"] < 0).to(device)
    assert (q_out[out] == 7).all() and (k_out[out] == 7).all()            # rows of no request
    for o, (y, size), what in zip(got, expect(s, pairs, 1.25), "qk"):
        close(o, y, size, dtype, what)
    # Into the pools: the same keys in fp16, the values as write_slots puts them.
    bs = 16 if rows % 2 else 20
    blocks = -(-s["rows"] // bs) + 2
    order = np.random.default_rng(rows).permutation(blocks * bs)[:s["rows"]].astype(np.int32)
    order[0] = -1 if rows > 1 else order[0]                              # rotated, not stored
    order[-1] = blocks * bs                                              # outside the pool
    slots = up(order, device)
    pools = [torch.full((blocks, kv, bs, d), 3.0, dtype=torch.float16, device=device) for _ in range(4)]
    q2, none = kernels.rotate_rows(s["q"](x), s["k"](x), up(s["pos"], device), up(s["f"], device), q_weight=wq,
                                   k_weight=wk, eps=EPS, attention_scaling=1.25, interleaved=pairs, value=s["v"](x),
                                   slots=slots, hot_k=pools[0], hot_v=pools[1], q_out=torch.full_like(q_out, 7.0))
    assert none is None and torch.equal(q2, q_out)
    kept = torch.where(out, -1, slots)
    kernels.write_slots(s["k"](x), s["v"](x), kept, pools[2], pools[3])
    assert torch.equal(pools[1], pools[3])
    touched = (pools[2] != 3).any(-1)
    assert ((pools[0] != 3).any(-1) <= touched).all()
    y, size = expect(s, pairs, 1.25)[1]
    rows_of = pools[0].transpose(1, 2).reshape(-1, kv, d)
    at = kept.cpu().numpy()
    live = np.nonzero((at >= 0) & (at < blocks * bs))[0]
    close(rows_of[torch.from_numpy(at[live]).long().to(device)], y[live], size[live], torch.float16, "pool")


def test_far_positions_keep_their_angle(device):
    """Positions up to 2^31 - 1: the angle is formed in 64 bits."""
    s = step(5, 6, 2, 1, 64, 64, torch.float16, False)
    s["pos"][:6] = [0, 1, 131072, 16777217, 2 ** 30 + 1, 2 ** 31 - 1]
    x = s["x"].to(device)
    got = kernels.rotate_rows(s["q"](x), s["k"](x), up(s["pos"], device), up(s["f"], device))
    for o, (y, size) in zip(got, expect(s, False)):
        close(o, y, size, torch.float16, "far")


def test_layouts_and_weights(device):
    """Strided rows, rows that start off a 16-byte boundary, a last dim that is
    not contiguous, one row for all tokens, fp32 weights, one weight alone."""
    s = step(6, 20, 4, 2, 64, 64, torch.bfloat16, True)
    x, pos, f = s["x"].to(device), up(s["pos"], device), up(s["f"], device)
    q, k = s["q"](x).contiguous(), s["k"](x).contiguous()
    wq, wk = (w.to(device) for w in s["w"])
    fresh = lambda: dict(q_out=torch.zeros_like(q), k_out=torch.zeros_like(k))   # noqa: E731
    base = kernels.rotate_rows(q, k, pos, f, q_weight=wq, k_weight=wk, **fresh())
    same = lambda got: all(torch.equal(a, b) for a, b in zip(got, base))   # noqa: E731
    close_to = lambda got: [close(o, y, z, torch.bfloat16, "layout") for o, (y, z) in zip(got, expect(s, False))]   # noqa: E731
    assert same(kernels.rotate_rows(s["q"](x), s["k"](x), pos, f, q_weight=wq, k_weight=wk, **fresh()))
    by_head = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)   # noqa: E731
    assert same(kernels.rotate_rows(by_head(q), by_head(k), pos, f, q_weight=wq, k_weight=wk, **fresh()))
    close_to(kernels.rotate_rows(q, k, pos, f, q_weight=wq.float(), k_weight=wk.float(), **fresh()))
    odd = lambda t: torch.nn.functional.pad(t, (1, 2))[:, :, 1:-2]   # noqa: E731
    close_to(kernels.rotate_rows(odd(q), odd(k), pos, f, q_weight=wq, k_weight=wk, **fresh()))
    turned = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)   # noqa: E731
    close_to(kernels.rotate_rows(turned(q), turned(k), pos, f, q_weight=wq, k_weight=wk, **fresh()))
    one = kernels.rotate_rows(q[:1].expand_as(q), k[:1].expand_as(k), torch.full_like(pos, int(pos[0])), f, q_weight=wq,
                              k_weight=wk, **fresh())
    assert all(torch.equal(o, b[:1].expand_as(o)) for o, b in zip(one, base))
    alone = kernels.rotate_rows(q, k, pos, f, q_weight=wq, **fresh())
    assert torch.equal(alone[0], base[0]) and not torch.equal(alone[1], base[1])
    assert torch.equal(alone[1], kernels.rotate_rows(q, k, pos, f, **fresh())[1])


def test_special_values(device):
    """A row of zeros stays zero under its norm; an infinity or NaN stays in
    its own head; bf16 keys past fp16's range become infinities in the pool."""
    q = torch.randn((4, 2, 64), device=device).to(torch.bfloat16)
    k = torch.randn((4, 2, 64), device=device).to(torch.bfloat16)
    pos, f = torch.arange(4, dtype=torch.int32, device=device), up((10000.0 ** (-np.arange(0, 64, 2) / 64)).astype(np.float32), device)
    w = torch.ones(64, dtype=torch.bfloat16, device=device)
    clean, _ = kernels.rotate_rows(q, k, pos, f, q_weight=w, k_weight=w)
    q[0, 0], q[1, 1, 3], q[2, 0, 5] = 0, float("nan"), float("inf")
    got, _ = kernels.rotate_rows(q, k, pos, f, q_weight=w, k_weight=w)
    assert (got[0, 0] == 0).all()
    same = torch.ones((4, 2), dtype=torch.bool, device=device)
    same[0, 0] = same[1, 1] = same[2, 0] = False
    assert torch.equal(got[same], clean[same])
    assert got[1, 1].isnan().all()
    k[0, 0, :] = 1e5
    pool = torch.zeros((2, 1, 2, 2, 64), dtype=torch.float16, device=device)
    pool = pool.view(2, 1, 2, 2, 64)
    kernels.rotate_rows(q, k, 0 * pos, f, value=k, slots=torch.tensor([0, 1, -1, -1], dtype=torch.int32, device=device),
                        hot_k=pool[0], hot_v=pool[1])
    assert pool[:, 0, 0, 0].isinf().all() and pool[:, 0, 1].isfinite().all()


def test_empty_steps_and_refusals(device):
    z = lambda *shape: torch.zeros(shape, dtype=torch.float16, device=device)   # noqa: E731
    f = torch.ones(32, device=device)
    i = lambda n: torch.zeros(n, dtype=torch.int32, device=device)   # noqa: E731
    q, k = kernels.rotate_rows(z(0, 4, 64), z(0, 2, 64), i(0), f)
    assert q.shape == (0, 4, 64) and k.shape == (0, 2, 64)
    pool = z(2, 2, 16, 64)
    q, k = kernels.rotate_rows(z(0, 4, 64), z(0, 2, 64), i(0), f, value=z(0, 2, 64), slots=i(0), hot_k=pool, hot_v=pool)
    assert q.shape == (0, 4, 64) and k is None
    ok = dict(query=z(3, 4, 64), key=z(3, 2, 64), positions=i(3), inv_freq=f)
    pools = dict(value=z(3, 2, 64), slots=i(3), hot_k=z(2, 2, 16, 64), hot_v=z(2, 2, 16, 64))
    kernels.rotate_rows(**ok, **{**pools, "slots": torch.arange(3, dtype=torch.int32, device=device)})
    for bad in (dict(query=z(3, 4, 64).float()), dict(key=z(2, 2, 64)), dict(key=z(3, 2, 64).bfloat16()), dict(positions=i(4)),
                dict(positions=i(3).long()), dict(inv_freq=torch.ones(33, device=device)), dict(inv_freq=f.double()),
                dict(q_weight=z(63)), dict(q_weight=z(64).bfloat16()), dict(q_weight=z(64), k_weight=z(64).float()),
                dict(q_out=z(3, 4, 63)), dict(k_out=z(3, 4, 64)), dict(eps=-1.0), dict(attention_scaling=float("inf")),
                dict(slots=i(3)), {**pools, "value": None}, {**pools, "hot_v": z(3, 2, 16, 64)}, {**pools, "slots": i(2)},
                {**pools, "hot_k": z(2, 4, 16, 64), "hot_v": z(2, 4, 16, 64)}, dict(positions=i(3).cpu())):
        with pytest.raises(ValueError):
            kernels.rotate_rows(**{**ok, **bad})


def test_replays_match_eager_calls(device):
    """Captured, replayed with other positions and rows between eager calls."""
    s = step(8, 50, 8, 2, 128, 128, torch.float16, True, pad=0)
    x, pos, f = s["x"].to(device), up(s["pos"], device), up(s["f"], device)
    wq, wk = (w.to(device) for w in s["w"])
    pool = torch.zeros((2, 5, 2, 16, 128), dtype=torch.float16, device=device)
    q_out = torch.zeros((50, 8, 128), dtype=torch.float16, device=device)
    slots = torch.randperm(80, device=device)[:50].int()

    def call(out, p):
        return kernels.rotate_rows(s["q"](x), s["k"](x), pos, f, q_weight=wq, k_weight=wk, value=s["v"](x), slots=slots,
                                   hot_k=p[0], hot_v=p[1], q_out=out)

    call(q_out, pool)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(q_out, pool)
    for i in range(3):
        x.copy_(torch.randn_like(x))
        pos.copy_(torch.randint(-1, 90000, (50,), device=device).int())
        q_out.zero_()
        pool.zero_()
        g.replay()
        torch.cuda.synchronize()
        want, fresh = torch.zeros_like(q_out), torch.zeros_like(pool)
        call(want, fresh)
        assert torch.equal(q_out, want) and torch.equal(pool, fresh)
