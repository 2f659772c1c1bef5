"""Packed rows quantized into WARM slots as they are written, and tokens of a
tiered cache read back, on the GPU: codes and metadata bit for bit against the
oracle (oracle/shared_prompt.py), values read back to half a step of their type."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import shared_prompt
from paged_tierkv_amd import kernels

pytestmark = pytest.mark.gpu
HOT, WARM, COLD = 0, 1, 2


def pools(rng, slots, kv, bs, d, fmt):
    if fmt == "ref_u8":
        return dict(codes=rng.integers(0, 256, (slots, kv, bs, d)).astype(np.uint8),
                    scale=np.abs(rng.standard_normal((slots, kv, bs, 1)) * 0.02 + 0.01).astype(np.float16),
                    zero=rng.integers(0, 256, (slots, kv, bs, 1)).astype(np.float16))
    return dict(codes=rng.integers(-127, 128, (slots, kv, bs, d)).astype(np.int8),
                scale=(np.abs(rng.standard_normal((slots, kv))) * 0.01 + 0.004).astype(np.float32), zero=None)


def up(a, device):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(device)


def write(device, k, v, slots, pk, pv, fmt):
    dk, dv = ({n: up(p[n], device) for n in ("codes", "scale", "zero")} for p in (pk, pv))
    kernels.quantize_rows(k, v, up(np.asarray(slots, np.int32), device), dk["codes"], dv["codes"], dk["scale"], dk["zero"],
                          dv["scale"], dv["zero"], fmt)
    return dk, dv


def same(dev, host):
    for n in ("codes", "scale", "zero"):
        if host[n] is not None:
            np.testing.assert_array_equal(dev[n].cpu().numpy(), host[n], err_msg=n)


# (first position, rows) of runs, each in a block of its own
RUNS = {
    "token": [(0, 1)], "tokens": [(5, 1), (0, 1), (15, 1), (8, 1)], "prompt": [(0, 16)] * 5 + [(0, 3)],
    "pieces": [(4, 12), (0, 16), (0, 16), (0, 9)], "mixed": [(15, 1), (3, 2), (0, 16), (7, 9), (0, 1), (1, 15)],
    "many": [(i % 16, 1) for i in range(75)], "long": [(9, 7)] + [(0, 16)] * 40 + [(0, 5)],
}


@pytest.mark.parametrize("runs", list(RUNS))
@pytest.mark.parametrize("kv,d,bs", [(8, 128, 16), (2, 64, 16), (1, 40, 16), (3, 30, 16), (2, 256, 16), (4, 8, 64), (2, 96, 20)])
@pytest.mark.parametrize("fmt", ["absmax_i8", "ref_u8"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_codes_match_the_oracle(device, runs, kv, d, bs, fmt, dtype):
    rng = np.random.default_rng(d * bs + len(RUNS[runs]))
    count = len(RUNS[runs])
    order = rng.permutation(count + 2)
    slots = np.concatenate([order[i] * bs + p + np.arange(n) for i, (p, n) in enumerate(RUNS[runs])])
    x = rng.standard_normal((2, len(slots), kv, d)) * np.exp(0.7 * rng.standard_normal((2, len(slots), 1, 1)))
    k, v = (torch.from_numpy(a.astype(np.float32)).to(dtype) for a in x)
    pk, pv = pools(rng, count + 2, kv, bs, d, fmt), pools(rng, count + 2, kv, bs, d, fmt)
    dk, dv = write(device, k.to(device), v.to(device), slots, pk, pv, fmt)
    for rows, p in ((k, pk), (v, pv)):
        shared_prompt.quantize_rows(rows.to(torch.float16).numpy(), slots, p["codes"], p["scale"], p["zero"])
    same(dk, pk)
    same(dv, pv)


@pytest.mark.parametrize("copies", [1, 6])           # few rows and many
@pytest.mark.parametrize("d", [8, 128])
def test_long_runs_beside_short_ones(device, copies, d):
    """Blocks of 64 tokens: runs of every length that start close together,
    some of them past the next 64 rows."""
    kinds = [(0, 1), (5, 1), (63, 1), (3, 61), (0, 64), (0, 1), (9, 1), (0, 2), (1, 63), (0, 17), (60, 4), (0, 50), (8, 1),
             (0, 1), (2, 1), (0, 64), (0, 64), (7, 3)] * copies
    rng = np.random.default_rng(copies)
    order = rng.permutation(len(kinds))
    slots = np.concatenate([order[i] * 64 + p + np.arange(n) for i, (p, n) in enumerate(kinds)])
    k, v = (torch.from_numpy((rng.standard_normal((len(slots), 3, d)) * np.exp(rng.standard_normal((len(slots), 1, 1)))
                              ).astype(np.float16)) for _ in range(2))
    pk, pv = pools(rng, len(kinds), 3, 64, d, "absmax_i8"), pools(rng, len(kinds), 3, 64, d, "absmax_i8")
    dk, dv = write(device, k.to(device), v.to(device), slots, pk, pv, "absmax_i8")
    for rows, p in ((k, pk), (v, pv)):
        shared_prompt.quantize_rows(rows.numpy(), slots, p["codes"], p["scale"], None)
    same(dk, pk)
    same(dv, pv)


@pytest.mark.parametrize("fmt", ["absmax_i8", "ref_u8"])
def test_a_cache_grown_token_by_token_is_the_oracle_s(device, fmt):
    """One call per token, scales that grow and stay, a row of zeros among them."""
    rng = np.random.default_rng(3)
    pk, pv = (pools(rng, 3, 2, 16, 64, fmt) for _ in range(2))
    dk, dv = ({n: up(p[n], device) for n in ("codes", "scale", "zero")} for p in (pk, pv))
    for i in range(21):
        x = (rng.standard_normal((2, 1, 2, 64)) * np.exp(rng.standard_normal())).astype(np.float16)
        if i in (0, 4):
            x[:] = 0
        slots = np.array([(2 if i < 16 else 0) * 16 + i % 16], np.int32)
        kernels.quantize_rows(up(x[0], device), up(x[1], device), up(slots, device), dk["codes"], dv["codes"], dk["scale"],
                              dk["zero"], dv["scale"], dv["zero"], fmt)
        for rows, p in zip(x, (pk, pv)):
            shared_prompt.quantize_rows(rows, slots, p["codes"], p["scale"], p["zero"])
        same(dk, pk)
        same(dv, pv)


@pytest.mark.parametrize("fmt", ["absmax_i8", "ref_u8"])
def test_special_values(device, fmt):
    """Zeros, equal values, the largest and smallest fp16, bf16 past its range:
    the codec's results; skipped rows leave the pools alone."""
    rng = np.random.default_rng(4)
    x = rng.standard_normal((6, 2, 64)).astype(np.float32)
    x[0], x[1], x[2, :, 3], x[3], x[4] = 0, 1.5, 65504, 2.0 ** -24, -65504
    for dtype in (torch.float16, torch.bfloat16):
        rows = torch.from_numpy(x).to(dtype)
        slots = np.array([0, 16, 32, 48, 64, 80], np.int32)
        pk, pv = (pools(rng, 7, 2, 16, 64, fmt) for _ in range(2))
        dk, dv = write(device, rows.to(device), rows.to(device), slots, pk, pv, fmt)
        for p in (pk, pv):
            with np.errstate(over="ignore", invalid="ignore"):
                shared_prompt.quantize_rows(rows.to(torch.float16).numpy(), slots, p["codes"], p["scale"], p["zero"])
        if dtype == torch.float16:                       # (infinite rows: no codes to compare)
            same(dk, pk)
            same(dv, pv)
    pk, pv = (pools(rng, 3, 2, 16, 64, fmt) for _ in range(2))
    rows = torch.randn((4, 2, 64), device=device).half()
    dk, dv = write(device, rows, rows, [-1, 48, -7, 2 ** 31 - 1], pk, pv, fmt)
    same(dk, pk)
    same(dv, pv)
    dk, dv = write(device, rows[:0], rows[:0], [], pk, pv, fmt)
    same(dk, pk)


def test_strided_and_unaligned_rows(device):
    rng = np.random.default_rng(5)
    slots = np.concatenate([np.arange(16, 32), [3, 4, 5]])
    for fmt in ("absmax_i8", "ref_u8"):
        pk, pv = pools(rng, 3, 4, 16, 64, fmt), pools(rng, 3, 4, 16, 64, fmt)
        fused = torch.randn((19, 8 * 64 + 3), device=device).to(torch.bfloat16)
        k, v = fused[:, 1:1 + 4 * 64].view(19, 4, 64), fused[:, 3 + 4 * 64:].view(19, 4, 64)
        dk, dv = write(device, k, v, slots, pk, pv, fmt)
        ck, cv = write(device, k.contiguous(), v.transpose(1, 2).contiguous().transpose(1, 2), slots, pk, pv, fmt)
        for a, b in ((dk, ck), (dv, cv)):
            assert all(torch.equal(a[n], b[n]) for n in ("codes", "scale") + (("zero",) if fmt == "ref_u8" else ()))


def test_written_rows_agree_with_demotion(device):
    """Whole blocks written as rows are the blocks that demote_to_warm makes."""
    tiles = torch.randn((2, 5, 4, 16, 128), device=device).half()
    idx = torch.arange(5, dtype=torch.int32, device=device)
    for fmt in ("absmax_i8", "ref_u8"):
        rng = np.random.default_rng(6)
        p = [{n: up(x, device) for n, x in pools(rng, 5, 4, 16, 128, fmt).items()} for _ in range(4)]
        kernels.demote_to_warm(tiles[0], tiles[1], idx, idx, torch.full_like(idx, 16), p[0]["codes"], p[1]["codes"],
                               p[0]["scale"], p[0]["zero"], p[1]["scale"], p[1]["zero"], fmt)
        k, v = (t.transpose(1, 2).reshape(80, 4, 128) for t in tiles)
        kernels.quantize_rows(k, v, torch.arange(80, dtype=torch.int32, device=device), p[2]["codes"], p[3]["codes"],
                              p[2]["scale"], p[2]["zero"], p[3]["scale"], p[3]["zero"], fmt)
        for a, b in ((p[0], p[2]), (p[1], p[3])):
            assert torch.equal(a["codes"], b["codes"]) and torch.equal(a["scale"], b["scale"])


def cache(seed, lens, kv, d, bs, fmt, spare=2):
    """Tables and pools of requests whose blocks hold these many tokens."""
    rng = np.random.default_rng(seed)
    width = max(max(len(x) for x in lens), 1) + spare
    states = rng.choice([HOT, WARM, COLD], (len(lens), width)).astype(np.int32)
    lengths = rng.integers(0, bs + 1, (len(lens), width)).astype(np.int32)        # past the count: never read
    for b, x in enumerate(lens):
        lengths[b, :len(x)] = x
    hot = [rng.standard_normal((9, kv, bs, d)).astype(np.float16) for _ in range(2)]
    warm = [pools(rng, 7, kv, bs, d, fmt) for _ in range(2)]
    table = np.where(states == HOT, rng.integers(0, 9, states.shape), np.where(states == WARM, rng.integers(0, 7, states.shape), -1))
    return dict(table=table.astype(np.int32), states=states, lengths=lengths, nb=np.array([len(x) for x in lens], np.int32),
                hot=hot, warm=warm, fmt=fmt)


def read(device, c, start, counts, dtype, rows=None, out=None, nb=True):
    cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    (k, v), w = c["hot"], c["warm"]
    args = [up(x, device) for x in (c["table"], c["states"], c["lengths"], c["nb"] if nb else None, k, v, w[0]["codes"],
                                    w[1]["codes"], w[0]["scale"], w[0]["zero"], w[1]["scale"], w[1]["zero"])]
    rows = int(cu[-1]) if rows is None else rows
    got = kernels.read_rows(up(np.array(start, np.int32), device), up(cu, device), rows, *args, dtype=dtype, out=out)
    nblocks = c["nb"] if nb else np.full(len(start), c["table"].shape[1])
    want = shared_prompt.read_rows(start, cu, rows, c["table"], c["states"], c["lengths"], nblocks, k, v, w[0]["codes"],
                                   w[1]["codes"], w[0]["scale"], w[0]["zero"], w[1]["scale"], w[1]["zero"], c["fmt"])
    for g, x in zip(got, want):
        live = ~np.isnan(x)
        g = g.double().cpu().numpy()
        # One rounding of a product that both form in 32 bits: half a step of
        # the type, 2^-24 of the 32-bit product, 2^-25 below fp16's normal range.
        tol = np.abs(x) * (torch.finfo(dtype).eps / 2 + 2.0 ** -24) + (2.0 ** -25 if dtype == torch.float16 else 0)
        assert (np.abs(g - x)[live] <= tol[live]).all()
    return got


@pytest.mark.parametrize("kv,d,bs", [(8, 128, 16), (2, 64, 16), (1, 40, 16), (3, 30, 16), (2, 256, 8), (4, 8, 64)])
@pytest.mark.parametrize("fmt,dtype", [("absmax_i8", torch.float16), ("ref_u8", torch.bfloat16), ("absmax_i8", torch.float32),
                                       ("ref_u8", torch.float32), ("ref_u8", torch.float16), ("absmax_i8", torch.bfloat16)])
def test_rows_read_back_match_the_oracle(device, kv, d, bs, fmt, dtype):
    rng = np.random.default_rng(d + bs)
    lens = [[bs] * 5 + [3 % bs + 1], [1], [], [bs, bs // 2, 0, bs, 1], list(rng.integers(0, bs + 1, 40)), [bs] * 13, [0, 0]]
    held = [int(sum(x)) for x in lens]
    c = cache(d, lens, kv, d, bs, fmt)
    whole = read(device, c, [0] * 7, held, dtype)
    assert whole[0].shape == (sum(held), kv, d)
    read(device, c, [max(0, h - 9) for h in held], [min(h, 9) for h in held], dtype)     # the last tokens
    start = [int(rng.integers(0, h + 1)) for h in held]
    read(device, c, start, [int(rng.integers(0, h - s + 1)) for h, s in zip(held, start)], dtype)
    read(device, c, [0, 0, 5, 3, -2, 13 * bs, 1], [held[0] + 20, 0, 4, 1, 6, 7, 2], dtype)     # past the end, nothing held


def test_rows_of_no_request_stay(device):
    c = cache(1, [[16, 16], [16, 4]], 2, 64, 16, "absmax_i8")
    out = tuple(torch.full((60, 2, 64), 5.0, dtype=torch.float16, device=device) for _ in range(2))
    got = read(device, c, [0, 2], [32, 18], torch.float16, rows=60, out=out)
    assert got[0] is out[0] and (out[0][50:] == 5).all() and (out[1][50:] == 5).all()
    got = read(device, c, [0, 2], [32, 18], torch.float16)
    # Fewer rows than the requests bring: those that there are.
    short = kernels.read_rows
    few = tuple(torch.full((40, 2, 64), 5.0, dtype=torch.float16, device=device) for _ in range(2))
    w = c["warm"]
    short(up(np.array([0, 2], np.int32), device), up(np.array([0, 32, 50], np.int32), device), 40,
          *[up(c[n], device) for n in ("table", "states", "lengths", "nb")], *[up(a, device) for a in c["hot"]],
          up(w[0]["codes"], device), up(w[1]["codes"], device), up(w[0]["scale"], device), None, up(w[1]["scale"], device), None,
          out=few)
    assert torch.equal(few[0], got[0][:40]) and torch.equal(few[1], got[1][:40])


def test_bad_slots_read_as_evicted_and_counts_default_to_the_table(device):
    c = cache(2, [[16, 16, 16, 16]], 2, 64, 16, "ref_u8", spare=0)
    c["states"][0] = [HOT, WARM, HOT, 7]
    c["table"][0] = [9, 7, 3, 0]
    got = read(device, c, [0], [64], torch.float16, nb=False)
    assert (got[0][:32] == 0).all() and (got[0][48:] == 0).all() and (got[0][32:48] != 0).any()


@pytest.mark.parametrize("d", [20, 24])
def test_a_short_window_of_a_very_long_context(device, d):
    """Ten tokens at the front and in the middle of 2^20 (evicted ones but for
    two blocks): what lies far behind a window writes nothing."""
    kv, bs, n = 64, 64, 1 << 14
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)   # noqa: E731
    states = torch.full((1, n), 2, dtype=torch.int32, device=device)
    states[0, [0, 9000]] = 0
    table = torch.zeros_like(states)
    table[0, 9000] = 1
    lengths = torch.full_like(states, bs)
    hot = torch.arange(2 * 2 * kv * bs * d, device=device).remainder(501).half().view(2, 2, kv, bs, d)
    codes, scale = torch.zeros((1, kv, bs, d), dtype=torch.int8, device=device), torch.zeros((1, kv), device=device)
    for start, slot in ((3, 0), (9000 * bs + 3, 1), (5 * bs, None)):
        out = torch.full((2, 30, kv, d), 7.0, dtype=torch.float16, device=device)
        kernels.read_rows(i32(start), i32(10, 20), 30, table, states, lengths, None, hot[0], hot[1], codes, codes, scale, None, scale,
                  None, out=(out[0], out[1]))
        want = torch.full_like(out, 7.0)
        want[:, 10:20] = 0 if slot is None else hot[:, slot, :, 3:13].transpose(1, 2)
        assert torch.equal(out, want)


def test_values_outside_the_tokens_do_not_matter(device):
    c = cache(3, [[5, 16]], 2, 64, 16, "absmax_i8", spare=0)
    c["states"][0], c["table"][0] = [HOT, HOT], [0, 1]
    clean = read(device, c, [0], [21], torch.float16)
    for p in c["hot"]:
        p[0, :, 5:] = np.nan
        p[2:] = np.inf
    again = read(device, c, [0], [21], torch.float16)
    assert torch.equal(clean[0], again[0]) and torch.equal(clean[1], again[1])


def test_what_was_written_comes_back(device):
    """Rows quantized, then read: within half a step of each scale."""
    rng = np.random.default_rng(7)
    for fmt in ("absmax_i8", "ref_u8"):
        p = [{n: up(x, device) for n, x in pools(rng, 6, 4, 16, 128, fmt).items()} for _ in range(2)]
        k, v = torch.randn((2, 70, 4, 128), device=device).half()
        slots = torch.arange(70, dtype=torch.int32, device=device)
        kernels.quantize_rows(k, v, slots, p[0]["codes"], p[1]["codes"], p[0]["scale"], p[0]["zero"], p[1]["scale"],
                              p[1]["zero"], fmt)
        i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)   # noqa: E731
        z = torch.zeros((1, 4, 16, 128), dtype=torch.float16, device=device)
        got = kernels.read_rows(i32(0), i32(0, 70), 70, i32(0, 1, 2, 3, 4)[None], i32(*[WARM] * 5)[None],
                                i32(16, 16, 16, 16, 6)[None], None, z, z, p[0]["codes"], p[1]["codes"], p[0]["scale"],
                                p[0]["zero"], p[1]["scale"], p[1]["zero"])
        for g, x in zip(got, (k, v)):
            # absmax: max|x| / 127 is at most 6 / 127 here; ref_u8: the range
            # over 255 and the zero point's own rounding, one step in all.
            step = x.abs().max() / 127 / 2 if fmt == "absmax_i8" else (x.max() - x.min()) / 255
            assert (g.float() - x.float()).abs().max() <= step * 1.01 + 2.0 ** -9


def test_refusals(device):
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)   # noqa: E731
    rows = torch.zeros((2, 2, 64), dtype=torch.float16, device=device)
    codes = torch.zeros((2, 2, 16, 64), dtype=torch.int8, device=device)
    scale = torch.zeros((2, 2), device=device)
    ok = dict(key=rows, value=rows, slots=i(0, 1), warm_k=codes, warm_v=codes.clone(), k_scale=scale, k_zero=None,
              v_scale=scale.clone(), v_zero=None, warm_format="absmax_i8")
    kernels.quantize_rows(**ok)
    for bad in (dict(key=rows.float()), dict(value=rows[:1]), dict(slots=i(0)), dict(slots=i(0, 1).long()),
                dict(warm_k=codes.byte()), dict(warm_v=codes[:1]), dict(k_scale=scale.half()), dict(v_scale=None),
                dict(warm_format="ref_u8"), dict(k_scale=scale[:1]), dict(slots=i(0, 1).cpu()), dict(warm_k=codes[..., :32])):
        with pytest.raises(ValueError):
            kernels.quantize_rows(**{**ok, **bad})
    pool = torch.zeros((2, 2, 16, 64), dtype=torch.float16, device=device)
    t = i(0, 1)[None]
    ok = dict(start=i(0), cu_tokens=i(0, 3), num_tokens=3, block_table=t, block_states=t, block_lengths=t,
              seq_num_blocks=i(2), hot_k=pool, hot_v=pool, warm_k=codes, warm_v=codes, k_scale=scale, k_zero=None,
              v_scale=scale, v_zero=None)
    kernels.read_rows(**ok)
    for bad in (dict(start=i(0, 0)), dict(cu_tokens=i(0)), dict(num_tokens=-1), dict(block_states=i(0)[None]),
                dict(block_table=i(0)), dict(hot_k=pool.float()), dict(hot_v=pool[:1]), dict(warm_k=codes[..., :32]),
                dict(k_scale=None), dict(dtype=torch.int8), dict(out=(rows, rows)), dict(seq_num_blocks=i(1, 1)),
                dict(warm_k=codes.byte()), dict(start=i(0).long()), dict(cu_tokens=i(0, 3).cpu())):
        with pytest.raises(ValueError):
            kernels.read_rows(**{**ok, **bad})


def test_replays_match_eager_calls(device):
    """A captured write and read over changing rows, eager calls between the replays."""
    rng = np.random.default_rng(8)
    start = [{n: up(x, device) for n, x in pools(rng, 4, 2, 16, 64, "absmax_i8").items()} for _ in range(2)]
    k, v = torch.randn((2, 21, 2, 64), device=device).half()
    slots = torch.arange(10, 31, dtype=torch.int32, device=device)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)   # noqa: E731
    z = torch.zeros((1, 2, 16, 64), dtype=torch.float16, device=device)
    one, cu, table, state, lens, nb = i32(3), i32(0, 28), i32(0, 1)[None], i32(WARM, WARM)[None], i32(16, 15)[None], i32(2)
    copy = lambda: [{n: None if x is None else x.clone() for n, x in p.items()} for p in start]   # noqa: E731
    held = copy()

    def call(p, out=None):
        kernels.quantize_rows(k, v, slots, p[0]["codes"], p[1]["codes"], p[0]["scale"], None, p[1]["scale"], None, "absmax_i8")
        return kernels.read_rows(one, cu, 28, table, state, lens, nb, z, z, p[0]["codes"], p[1]["codes"], p[0]["scale"], None,
                                 p[1]["scale"], None, out=out)

    out = tuple(torch.zeros((28, 2, 64), dtype=torch.float16, device=device) for _ in range(2))
    call(copy(), out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(held, out)
    for i in range(3):
        k.copy_(torch.randn_like(k) * (i + 1))
        for p, s in zip(held, start):
            p["codes"].copy_(s["codes"])
            p["scale"].copy_(s["scale"])
        g.replay()
        torch.cuda.synchronize()
        fresh = copy()
        want = call(fresh)
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        assert all(torch.equal(a["codes"], b["codes"]) and torch.equal(a["scale"], b["scale"]) for a, b in zip(held, fresh))
