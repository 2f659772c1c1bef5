"""Attention of requests that share prefixes on the GPU, against the oracle
that attends row by row (oracle/shared_prompt.py).

Error bounds, elementwise, from the oracle's A = sum p |v| and X = the largest
scaling * sum |q_d k_d| of the row, are those of extend attention
(test_gpu_serving_step.py): probabilities and WARM values are rounded to fp16
once each, 2 * 2^-11 A; logits are off by (D + 8) 2^-24 X, twice in p; the
output's rounding, half a step of its type, and 2^-24 of each value added.  The
parts of a row are joined in 32 bits with factors that are off by a few 2^-24:
2^-20 A more.
"""

from __future__ import annotations

import threading

import numpy as np
import pytest
import torch

from oracle import codec, shared_prompt
from paged_tierkv_amd.tierkv_hip import (DecodeWorkspace, extend_workspace, tierkv_extend_attention,
                                         tierkv_prefix_attention)

pytestmark = pytest.mark.gpu
HOT, WARM, COLD = 0, 1, 2


def blocks(rng, tokens, bs, holes):
    row, left = [], tokens
    while left > 0:
        x = min(left, int(rng.integers(0, bs + 1)) if holes else bs)
        row.append(x)
        left -= x
    return row


def step(seed, prefixes, member, new, held, heads, kv, d, bs=16, fmt="absmax_i8", dtype=torch.float16, cold=0.3, warm=0.5,
         pad=2, holes=False, spare=2):
    """Requests that hold ``held`` tokens of their own, the last ``new`` new, and
    prefixes of the given lengths, in blocks of random tiers."""
    rng = np.random.default_rng(seed)
    rows = [[blocks(rng, t, bs, holes) for t in prefixes], [blocks(rng, t, bs, holes) for t in held]]
    tables, used = [], {HOT: 0, WARM: 0}
    for k, group in enumerate(rows):
        width = max(max((len(x) for x in group), default=0), 1) + spare
        states = rng.choice([HOT, WARM, COLD], (len(group), width)).astype(np.int32)
        lengths = rng.integers(0, bs + 1, (len(group), width)).astype(np.int32)      # past the count: never read
        for b, row in enumerate(group):
            r = rng.random(len(row))
            lengths[b, :len(row)] = row
            states[b, :len(row)] = np.where(r < cold, COLD, np.where(r < cold + warm, WARM, HOT))
            if k:                                                                    # the new tokens' blocks are HOT
                for i in range(len(row)):
                    if sum(row[i:]) - row[i] < new[b]:
                        states[b, i] = HOT
        tables.append([np.full((len(group), width), -1, np.int32), states, lengths, np.array([len(x) for x in group], np.int32)])
    for table, states, lengths, nb in tables:
        for b in range(len(nb)):
            for i in range(nb[b]):
                t = states[b, i]
                if t != COLD:
                    table[b, i] = used[t]
                    used[t] += 1
    pools = []
    for t in (HOT, WARM):
        count = used[t] + 3
        mix = rng.permutation(count).astype(np.int32)
        for table, states, _, _ in tables:
            at = (states == t) & (table >= 0)
            table[at] = mix[table[at]]
        pools.append([rng.standard_normal((count, kv, bs, d)).astype(np.float16) for _ in range(2)])
    (hk, hv), (wk, wv) = pools
    hk[:, :, : min(3, bs)] *= np.float16(2)
    quant = codec.quantize_absmax_i8 if fmt == "absmax_i8" else codec.quantize_ref_u8
    k, v = quant(wk), quant(wv)
    qk, ks, kz = k if len(k) == 3 else (*k, None)
    qv, vs, vz = v if len(v) == 3 else (*v, None)
    q = torch.from_numpy(rng.standard_normal((sum(new) + pad, heads, d)).astype(np.float32)).to(dtype)
    return dict(q=q, cu=np.concatenate([[0], np.cumsum(new)]).astype(np.int32), pre=tables[0], own=tables[1],
                member=np.array(member, np.int32), hot=(hk, hv), warm=(qk, qv), meta=(ks, kz, vs, vz), groups=heads // kv,
                scaling=d ** -0.5, fmt=fmt, dtype=dtype)


def gpu(a, device):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(device)


def tensors(s, device):
    return dict(q=s["q"].to(device), cu=gpu(s["cu"], device), own=[gpu(a, device) for a in s["own"]],
                pre=[gpu(a, device) for a in s["pre"]], member=gpu(s["member"], device),
                pools=[gpu(a, device) for a in (*s["hot"], *s["warm"], *s["meta"])])


def launch(t, s, cold, **kw):
    table, states, lengths, nb = t["own"]
    return tierkv_prefix_attention(
        kw.pop("q", t["q"]), t["cu"], table, states, lengths, *t["pools"], table.shape[1], s["groups"], s["scaling"],
        t["member"], *t["pre"][:3], prefix_num_blocks=t["pre"][3], cold_mode=cold, seq_num_blocks=nb, **kw)


def call(s, device, cold, **kw):
    return launch(tensors(s, device), s, cold, **kw)


def check(out, s, cold, rows=None):
    exp, mass, logit = shared_prompt.prefix_attention(
        s["q"].float().numpy(), s["cu"], s["own"], s["member"], s["pre"], *s["hot"], *s["warm"], *s["meta"], s["groups"],
        s["scaling"], s["fmt"], cold)
    rows = np.arange(s["cu"][-1]) if rows is None else rows
    d = s["q"].shape[2]
    tol = mass * (2 * 2.0 ** -11 + 2.0 ** -20 + 2 * (d + 8) * 2.0 ** -24 * logit[:, :, None])
    tol += np.abs(exp) * torch.finfo(s["dtype"]).eps / 2 + 2.0 ** -23
    err = np.abs(out.double().cpu().numpy() - exp)[rows]
    print(f"[prefix] largest error {err.max():.2e}, {(err / tol[rows]).max():.2f} of its bound", flush=True)
    assert (err <= tol[rows]).all(), (err / tol[rows]).max()


CASES = [
    # prefixes, member, new, held, heads, kv, d, bs
    ([40], [0], [1], [1], 4, 4, 64, 16),
    ([1], [0, 0], [1, 1], [1, 9], 8, 2, 128, 16),
    ([100, 37], [1, 0, 1, -1, 0], [1, 1, 1, 1, 1], [17, 1, 40, 33, 5], 32, 8, 128, 16),
    ([333], [0] * 9, [5, 1, 3, 8, 2, 1, 1, 7, 4], [30, 1, 3, 90, 2, 41, 16, 7, 20], 8, 2, 128, 16),     # narrow and wide
    ([64, 0, 90], [2, 1, 0, 7, -5], [4, 3, 9, 2, 40], [4, 50, 9, 20, 41], 8, 2, 64, 16),   # empty, unused, unknown prefixes
    ([700], [0, 0], [70, 33], [70, 300], 6, 2, 64, 16),                    # prompts on a prefix, group 3
    ([50], [0] * 40, [1] * 40, [3] * 40, 16, 2, 64, 16),                   # 320 rows of one prefix: two tiles
    ([333, 20], [1, 0, 1], [40, 0, 3], [333, 20, 90], 4, 1, 128, 32),      # a request without new tokens
    ([21, 210], [0, 1], [21, 50], [210, 64], 8, 8, 96, 16),
    ([200], [0, 0, 0], [9, 2, 30], [30, 64, 30], 4, 2, 40, 8),
    ([133], [0, -1], [17, 5], [100, 30], 4, 2, 128, 20),                   # a block that ends inside a sub-tile
    ([90], [0, 0], [6, 2], [5, 0], 4, 2, 64, 16),                          # more rows than tokens; nothing of its own
    ([2500], [0, 0, 0], [1, 1, 3], [12, 600, 3], 4, 1, 64, 16),            # cut
    ([40, 60], [0, 1], [12, 3], [50, 33], 4, 2, 8, 1),
    ([700], [0, 0, -1], [130, 33, 140], [130, 300, 200], 8, 2, 64, 16),    # requests that walk their prefix themselves,
    ([90, 0, 40], [2, 0, 1, 0], [300, 1, 129, 2], [333, 20, 129, 9], 8, 1, 128, 16),   # beside others
    ([1800], [0, 0], [171, 1], [171, 20], 12, 4, 96, 16),
]


@pytest.mark.parametrize("prefixes,member,new,held,heads,kv,d,bs", CASES)
@pytest.mark.parametrize("fmt,cold,dtype", [("absmax_i8", "masked", torch.float16), ("absmax_i8", "zero_logit", torch.bfloat16),
                                            ("ref_u8", "zero_logit", torch.float16), ("ref_u8", "masked", torch.bfloat16)])
def test_prefix_attention_matches_oracle(device, prefixes, member, new, held, heads, kv, d, bs, fmt, cold, dtype):
    print(f"[prefix] {prefixes} {member} {new} {held} {heads}/{kv} x {d}, blocks of {bs}, {fmt} {cold}", flush=True)
    s = step(sum(held) + heads, prefixes, member, new, held, heads, kv, d, bs, fmt, dtype)
    out = torch.full(s["q"].shape, 7.0, dtype=dtype, device=device)
    got = call(s, device, cold, out=out, max_tokens=max(new))
    assert got.data_ptr() == out.data_ptr()
    check(out, s, cold)
    assert (out[s["cu"][-1]:] == 7.0).all()                  # rows behind the last request
    again = call(s, device, cold)                            # no bound given
    check(again, s, cold)


@pytest.mark.parametrize("cold", ["masked", "zero_logit"])
def test_blocks_of_any_length_and_everything_evicted(device, cold):
    s = step(5, [150, 70], [0, 1, 0], [20, 7, 40], [90, 300, 45], 8, 2, 64, holes=True, cold=0.5)
    check(call(s, device, cold), s, cold)
    s["pre"][1][:] = COLD
    check(call(s, device, cold), s, cold)
    s["own"][1][:] = COLD
    out = call(s, device, cold)
    assert (out[:67] == 0).all()
    check(out, s, cold)


def test_equals_extend_attention_over_joined_tables(device):
    """The same tokens in every request's own row."""
    s = step(6, [300, 77], [1, 0, 0, -1, 1], [3, 1, 50, 2, 1], [40, 1, 60, 30, 200], 8, 2, 128)
    t = tensors(s, device)
    got = launch(t, s, "masked")
    joined = [[], [], []]
    for b, g in enumerate(s["member"]):
        for out, p, m in zip(joined, s["pre"], s["own"]):
            out.append(list(p[g][:s["pre"][3][g]] if g >= 0 else []) + list(m[b][:s["own"][3][b]]))
    nb = torch.tensor([len(x) for x in joined[0]], dtype=torch.int32, device=device)
    width = int(nb.max())
    table, states, lengths = (torch.tensor([x + [0] * (width - len(x)) for x in rows], dtype=torch.int32, device=device)
                              for rows in joined)
    ref = tierkv_extend_attention(t["q"], t["cu"], table, states, lengths, *t["pools"], width, s["groups"], s["scaling"],
                                  cold_mode="masked", seq_num_blocks=nb)
    torch.testing.assert_close(got[:57], ref[:57], rtol=2e-3, atol=1e-3)


def test_values_that_no_row_sees_do_not_matter(device):
    """NaN and infinities past a block's length, in slots of no block and
    behind the counts change nothing, nor do those of a prefix for the requests
    of another; a later token's do not reach the rows before it."""
    s = step(7, [45, 90], [0, 1, 1], [9, 40, 1], [50, 77, 5], 8, 2, 128, pad=0)
    clean = call(s, device, "masked")
    hk, hv = s["hot"]
    used = np.zeros((len(hk), 16), bool)
    for table, states, lengths, nb in (s["pre"], s["own"]):
        for b in range(len(nb)):
            for i in range(nb[b]):
                if states[b, i] == HOT:
                    used[table[b, i], :lengths[b, i]] = True
        for b in range(len(nb)):
            table[b, nb[b]:], states[b, nb[b]:], lengths[b, nb[b]:] = 0, HOT, 16
    bad = np.array([np.nan, np.inf, -np.inf], np.float16)
    for p in (hk, hv):
        p[:] = np.where(used[:, None, :, None], p, np.random.default_rng(1).choice(bad, p.shape))
    assert torch.equal(call(s, device, "masked"), clean)
    # A key and a value of prefix 0: its request's rows are lost, the others' are not.
    table, states, lengths, nb = s["pre"]
    i = int(np.nonzero(states[0, :nb[0]] == HOT)[0][0]) if (states[0, :nb[0]] == HOT).any() else None
    if i is None:
        states[0, 0], table[0, 0], i = HOT, int(np.nonzero(~used.any(1))[0][0]), 0
        hk[table[0, 0]], hv[table[0, 0]] = 0, 0
        clean = call(s, device, "masked")
    hk[table[0, i], :, 0, 3] = np.nan
    out = call(s, device, "masked")
    assert torch.equal(out[9:50], clean[9:50]) and out[:9].isnan().all()


def test_visible_infinities_arrive_where_they_belong(device):
    s = step(8, [40], [0, -1], [40, 3], [45, 3], 4, 2, 64, cold=0, warm=0)
    clean = call(s, device, "masked")
    s["hot"][1][s["pre"][0][0, 1], 0, 5, 9] = -np.inf
    out = call(s, device, "masked")
    assert (out[:40, :2, 9] == -float("inf")).all()
    hit = torch.zeros_like(clean, dtype=torch.bool)
    hit[:40, :2, 9] = True
    hit[43:] = True                                     # rows of no request
    assert torch.equal(out[~hit], clean[~hit])


@pytest.mark.parametrize("bs,spare,many", [(16, 900, 1), (16, 5000, 1), (64, 700, 1), (16, 3000, 12)])
@pytest.mark.parametrize("cold", ["masked", "zero_logit"])
def test_tables_far_wider_than_their_rows(device, bs, spare, many, cold):
    """Rows of few blocks and of many in tables of thousands, which a step cuts
    by their width: its parts that a row does not have are left out."""
    s = step(18, [30, 4000, 0], [0, 1, 1, 2, -1] * many, [1, 3, 1, 0, 2] * many, [20, 5000, 64, 9, 300] + [20, 50, 64, 9, 300] * (many - 1),
             8, 2, 64, bs=bs, spare=spare)
    t = tensors(s, device)
    ws = DecodeWorkspace(device)
    out = launch(t, s, cold, workspace=ws, max_tokens=3)
    assert ws.error_word() == 0
    check(out, s, cold)
    t["own"][3].zero_()                                  # no blocks of their own: the prefix alone
    s["own"][3][:] = 0
    check(launch(t, s, cold, workspace=ws, max_tokens=3), s, cold)


def test_order_of_requests_and_repeated_calls_keep_the_bits(device):
    """The same inputs twice give the same bits; a request's result does not
    depend on where its rows stand, up to the joins' rounding."""
    s = step(9, [900, 300], [0, 1, 0, 0, 1, -1], [1, 5, 1, 33, 2, 4], [30, 5, 44, 33, 90, 10], 16, 4, 64)
    t = tensors(s, device)
    first = launch(t, s, "masked", out=torch.zeros_like(t["q"]))
    for _ in range(3):
        assert torch.equal(launch(t, s, "masked", out=torch.zeros_like(t["q"])), first)
    order = [4, 0, 5, 2, 1, 3]
    rows = np.concatenate([np.arange(s["cu"][b], s["cu"][b + 1]) for b in order])
    n = np.diff(s["cu"])[order]
    r = dict(s, cu=np.concatenate([[0], np.cumsum(n)]).astype(np.int32), member=s["member"][order],
             own=[a[order] for a in s["own"]], q=torch.cat([s["q"][rows], s["q"][len(rows):]]))
    out = call(r, device, "masked")
    torch.testing.assert_close(out[:len(rows)], first[torch.from_numpy(rows).to(device)], rtol=2e-3, atol=1e-3)


def test_strided_queries_and_defaults(device):
    s = step(10, [64, 32], [0, 1], [9, 33], [80, 70], 8, 2, 64, pad=0, spare=0)
    for _, states, lengths, nb in (s["pre"], s["own"]):                 # whole rows: no counts given
        for b in range(len(nb)):
            lengths[b, nb[b]:] = 0
    t = tensors(s, device)
    base = launch(t, s, "zero_logit")
    wide = torch.zeros((42, 12, 72), dtype=torch.float16, device=device)
    wide[:, 2:10, :64] = t["q"]
    assert torch.equal(launch(t, s, "zero_logit", q=wide[:, 2:10, :64]), base)
    odd = torch.zeros((42, 8, 67), dtype=torch.float16, device=device)
    odd[:, :, 1:65] = t["q"]
    assert torch.equal(launch(t, s, "zero_logit", q=odd[:, :, 1:65]), base)
    table, states, lengths, _ = t["own"]
    plain = tierkv_prefix_attention(t["q"], t["cu"], table, states, lengths, *t["pools"], table.shape[1], 4, s["scaling"],
                                    t["member"], *t["pre"][:3])
    torch.testing.assert_close(plain, base, rtol=2e-3, atol=1e-3)


def test_bad_slots_are_reported_and_max_tokens_leaves_rows_out(device):
    s = step(11, [60, 40], [0, 1, 0], [3, 6, 1], [20, 30, 9], 4, 2, 64, cold=0)
    s["pre"][0][0, 1], s["pre"][1][0, 1] = 10 ** 6, HOT
    s["pre"][1][1, 0] = 9
    s["own"][0][1, 0], s["own"][1][1, 0] = -4, WARM
    ws = DecodeWorkspace(device)
    out = call(s, device, "masked", workspace=ws)
    assert ws.error_word() == 3 and ws.error_word() == 0
    t = dict(s, pre=[a.copy() for a in s["pre"]], own=[a.copy() for a in s["own"]])
    t["pre"][1][0, 1] = t["pre"][1][1, 0] = t["own"][1][1, 0] = COLD
    check(out, t, "masked")
    out = torch.full(s["q"].shape, 7.0, dtype=torch.float16, device=device)
    call(t, device, "masked", workspace=ws, max_tokens=4, out=out)
    assert ws.error_word() == 4
    check(out, t, "masked", rows=np.array([0, 1, 2, 3, 4, 5, 6, 9]))
    assert (out[7:9] == 7).all() and (out[10:] == 7).all()


@pytest.mark.parametrize("most", [1, 24])       # a step's way and a plan's
def test_row_ranges_that_overlap_do_no_harm(device, most):
    """Ranges out of order, so that requests' rows overlap: rows of no request
    stay as they are, the error word says so if any row was left out, and the
    next call finds nothing of it."""
    s = step(17, [60, 40], [0, 1, 0, 0], [3 * most, most, 4 * most, most], [200, 30, 210, 60], 4, 2, 64, spare=0)
    t = tensors(s, device)
    ws = DecodeWorkspace(device)
    want = launch(t, s, "masked", workspace=ws).clone()
    n = int(s["cu"][-1])
    good = t["cu"].clone()
    for cu in ([0, n - 1, 0, n, n], [5 * n, -3, 7, 2, n], [n, n - 1, 1, 0, n]):
        t["cu"].copy_(torch.tensor(cu, dtype=torch.int32))
        out = torch.full_like(t["q"], 7.0)
        launch(t, s, "masked", workspace=ws, out=out)
        assert (out[n:] == 7).all() and ws.error_word() in (0, 4)
    t["cu"].copy_(good)
    assert torch.equal(launch(t, s, "masked", workspace=ws)[:n], want[:n]) and ws.error_word() == 0


def test_no_rows_and_no_tokens(device):
    s = step(12, [30], [0, 0], [0, 0], [5, 20], 4, 2, 64, pad=3)
    out = torch.full(s["q"].shape, 7.0, dtype=torch.float16, device=device)
    call(s, device, "masked", out=out)
    assert (out == 7).all()
    s["q"] = s["q"][:0]
    assert call(s, device, "masked").shape == (0, 4, 64)


def test_one_workspace_for_calls_of_any_shape(device):
    """Prefix, extend and smaller prefix calls through one buffer, in turn."""
    big = step(13, [500, 60], [0, 1] * 20, [1] * 40, [20] * 40, 8, 2, 64)
    small = step(14, [20], [0, -1], [2, 3], [9, 9], 4, 2, 128, fmt="ref_u8", dtype=torch.bfloat16)
    ws = DecodeWorkspace(device)
    tb, ts = tensors(big, device), tensors(small, device)
    want_b, want_s = launch(tb, big, "masked"), launch(ts, small, "zero_logit")
    table, states, lengths, nb = ts["own"]
    ext = lambda w: tierkv_extend_attention(ts["q"], ts["cu"], table, states, lengths, *ts["pools"], table.shape[1], 2,   # noqa: E731
                                            small["scaling"], seq_num_blocks=nb, workspace=w)
    want_e = ext(None)
    for _ in range(2):
        assert torch.equal(launch(ts, small, "zero_logit", workspace=ws)[:5], want_s[:5])
        assert torch.equal(launch(tb, big, "masked", workspace=ws)[:40], want_b[:40])
        assert torch.equal(ext(ws)[:5], want_e[:5])
    assert ws.error_word() == 0


def test_replays_match_eager_calls(device):
    """Captured with a workspace of its own, replayed over other queries and
    other prefixes, eager calls of the same shape between the replays."""
    s = step(15, [300, 90], [0, 1, 0, 1], [1, 3, 1, 2], [30, 3, 20, 40], 8, 2, 64, pad=0)
    t = tensors(s, device)
    ws = extend_workspace(device, 4, 7, 8, 2, t["own"][0].shape[1], 64, max_tokens=3, prefixes=2,
                          prefix_blocks=t["pre"][0].shape[1])
    out = torch.zeros_like(t["q"])
    launch(t, s, "masked", workspace=ws, out=out, max_tokens=3)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        launch(t, s, "masked", workspace=ws, out=out, max_tokens=3)
    for i in range(4):
        t["q"].copy_(torch.randn_like(t["q"]))
        t["member"].copy_(torch.tensor([[0, 1, 0, 1], [1, 1, 1, 1], [-1, 0, 0, -1], [1, 0, 1, 0]][i], dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(launch(t, s, "masked", max_tokens=3), out)
        r = dict(s, q=t["q"].cpu(), member=t["member"].cpu().numpy())
        check(out, r, "masked")
    assert ws.error_word() == 0
    with pytest.raises(RuntimeError):
        launch(t, s, "masked", workspace=DecodeWorkspace(device, 4096, growable=False))


def test_threads_and_streams_get_their_own_results(device):
    steps = [step(20 + i, [200 + 90 * i], [0, 0, 0], [1, 2, 1], [20, 9, 33], 8, 2, 64) for i in range(4)]
    ts = [tensors(s, device) for s in steps]
    want = [launch(t, s, "masked") for t, s in zip(ts, steps)]
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        stream = torch.cuda.Stream(device) if i % 2 else torch.cuda.default_stream(device)
        with torch.cuda.stream(stream):
            for _ in range(20):
                got[i] = launch(ts[i], steps[i], "masked")

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for x in threads:
        x.start()
    for x in threads:
        x.join()
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert torch.equal(g[:4], w[:4])


def test_refusals(device):
    s = step(30, [40], [0, 0], [1, 2], [9, 5], 4, 2, 64)
    t = tensors(s, device)
    table, states, lengths, nb = t["own"]
    ok = dict(query_states=t["q"], cu_tokens=t["cu"], block_table=table, block_states=states, block_lengths=lengths,
              **dict(zip(("hot_k_pool", "hot_v_pool", "warm_k_pool", "warm_v_pool", "k_scale", "k_zero", "v_scale", "v_zero"),
                         t["pools"])), num_blocks=table.shape[1], num_key_value_groups=2, scaling=0.125, prefix_of=t["member"],
              prefix_table=t["pre"][0], prefix_states=t["pre"][1], prefix_lengths=t["pre"][2], prefix_num_blocks=t["pre"][3],
              seq_num_blocks=nb)
    tierkv_prefix_attention(**ok)
    p = t["pre"][0]
    for bad in (dict(prefix_of=t["member"].long()), dict(prefix_of=t["member"][:1]), dict(prefix_of=t["member"].cpu()),
                dict(prefix_table=p[0]), dict(prefix_states=p[:, :1]), dict(prefix_lengths=p.long()), dict(prefix_table=p.cpu()),
                dict(prefix_num_blocks=t["cu"]), dict(prefix_table=p[:0], prefix_states=p[:0], prefix_lengths=p[:0], prefix_num_blocks=None),
                dict(scaling=float("nan")), dict(query_states=t["q"].float()), dict(max_tokens=-1), dict(cold_mode="other")):
        with pytest.raises(ValueError):
            tierkv_prefix_attention(**{**ok, **bad})


@pytest.mark.parametrize("fmt,dtype", [("absmax_i8", torch.float16), ("ref_u8", torch.bfloat16)])
def test_tiles_for_more_than_a_round_equal_extend_attention(device, fmt, dtype):
    """Requests of many wide tiles each, the last of which are cut, beside
    single tokens: the same tokens in every request's own row."""
    s = step(31, [300], [0, 0, -1, 0], [1500, 1, 1100, 700], [1500, 40, 1100, 701], 32, 32, 64, fmt=fmt, dtype=dtype, pad=0)
    t = tensors(s, device)
    got = launch(t, s, "masked")
    rows = [[], [], []]
    for b, g in enumerate(s["member"]):
        for out, p, m in zip(rows, s["pre"], s["own"]):
            out.append(list(p[g][:s["pre"][3][g]] if g >= 0 else []) + list(m[b][:s["own"][3][b]]))
    nb = torch.tensor([len(x) for x in rows[0]], dtype=torch.int32, device=device)
    width = int(nb.max())
    joined = [torch.tensor([x + [0] * (width - len(x)) for x in r], dtype=torch.int32, device=device) for r in rows]
    ref = tierkv_extend_attention(t["q"], t["cu"], *joined, *t["pools"], width, s["groups"], s["scaling"], cold_mode="masked",
                                  seq_num_blocks=nb)
    # Both round probabilities and WARM values once: each is off the exact
    # output by 2 * 2^-11 of sum p |v|, at most the largest |v| (normal values,
    # below 8 here), and by its own rounding.
    tol = 2 * (2 * 2.0 ** -11 * 8) + ref.abs().float() * torch.finfo(dtype).eps
    assert ((got.float() - ref.float()).abs() <= tol).all()
    again = launch(t, s, "masked")
    assert torch.equal(again, got)
