"""A serving step over requests of different lengths on the GPU: slot maps and
K/V row writes (bit for bit), attention of several query tokens per request
and token choice, against the one-token-at-a-time oracle (oracle/serving.py).

Error bounds of the attention, elementwise, from the oracle's A = sum p |v|
and X = the largest scaling * sum |q_d k_d| of the row:
* probabilities and WARM values are rounded to fp16 once each: at most half a
  step, 2^-11 of the value, so 2 * 2^-11 A;
* logits: a sum of D products in 32 bits is off by at most D * 2^-24 X, the
  scale's product and the exponential's argument by a few 2^-24 X more; a logit off by e
  changes p by a factor exp(e), in the sum as well: 2 (D + 8) 2^-24 X A;
* reference-format K becomes fp16(code - zero), exact for |code - zero| <= 2048, as these inputs are;
* the output's rounding, half a step of its type, and 2^-24 (fp16 values below its normal range) of each value added.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import codec, serving
from paged_tierkv_amd import kernels
from paged_tierkv_amd.tierkv_hip import DecodeWorkspace, extend_workspace, tierkv_decode_attention, tierkv_extend_attention

pytestmark = pytest.mark.gpu
HOT, WARM, COLD = 0, 1, 2


def step(seed, new, held, heads, kv, d, bs=16, fmt="absmax_i8", dtype=torch.float16, cold=0.3, warm=0.5, pad=0,
         spare=2, holes=False):
    """Requests that hold ``held`` tokens, the last ``new`` of them new, in
    blocks of random tiers; ``holes``: blocks of any length, 0 included."""
    rng = np.random.default_rng(seed)
    batch = len(new)
    lens = []
    for n, h in zip(new, held):
        row, left = [], h
        while left > 0:
            x = min(left, int(rng.integers(0, bs + 1)) if holes else bs)
            row.append(x)
            left -= x
        lens.append(row)
    width = max(max((len(x) for x in lens), default=0), 1) + spare
    states = np.full((batch, width), COLD, np.int32)
    lengths = np.zeros((batch, width), np.int32)
    for b, row in enumerate(lens):
        r = rng.random(len(row))
        lengths[b, :len(row)] = row
        states[b, :len(row)] = np.where(r < cold, COLD, np.where(r < cold + warm, WARM, HOT))
        for i in range(len(row)):          # the new tokens' blocks are HOT
            if sum(row[i:]) - row[i] < new[b] or i == 0:
                states[b, i] = HOT
    table = np.full((batch, width), -1, np.int32)
    pools = []
    for tier in (HOT, WARM):
        at = np.nonzero((states == tier) & (np.arange(width)[None] < np.array([len(x) for x in lens])[:, None]))
        count = len(at[0]) + 3
        table[at] = rng.permutation(count)[:len(at[0])]
        pools.append([rng.standard_normal((count, kv, bs, d)).astype(np.float16) for _ in range(2)])
    (hk, hv), (wk, wv) = pools
    hk[:, :, : min(4, bs)] *= np.float16(2)
    quant = codec.quantize_absmax_i8 if fmt == "absmax_i8" else codec.quantize_ref_u8
    k, v = quant(wk), quant(wv)
    qk, ks, kz = k if len(k) == 3 else (*k, None)
    qv, vs, vz = v if len(v) == 3 else (*v, None)
    q = torch.from_numpy(rng.standard_normal((sum(new) + pad, heads, d)).astype(np.float32)).to(dtype)
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    nblocks = np.array([len(x) for x in lens], np.int32)
    return dict(q=q, cu=cu, table=table, states=states, lengths=lengths, nblocks=nblocks, hot=(hk, hv), warm=(qk, qv),
                meta=(ks, kz, vs, vz), groups=heads // kv, scaling=d ** -0.5, fmt=fmt, dtype=dtype)


def gpu(a, device):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(device)


def call(s, device, cold, **kw):
    ks, kz, vs, vz = (gpu(a, device) for a in s["meta"])
    q = kw.pop("q", None)
    return tierkv_extend_attention(
        s["q"].to(device) if q is None else q, gpu(s["cu"], device), gpu(s["table"], device), gpu(s["states"], device),
        gpu(s["lengths"], device), gpu(s["hot"][0], device), gpu(s["hot"][1], device), gpu(s["warm"][0], device),
        gpu(s["warm"][1], device), ks, kz, vs, vz, s["table"].shape[1], s["groups"], s["scaling"], cold_mode=cold,
        seq_num_blocks=gpu(s["nblocks"], device), **kw)


def want(s, cold):
    return serving.extend_attention(s["q"].float().numpy(), s["cu"], s["table"], s["states"], s["lengths"],
                                    s["nblocks"], *s["hot"], *s["warm"], *s["meta"], s["groups"], s["scaling"],
                                    s["fmt"], cold)


def check(out, s, cold, rows=None):
    exp, mass, logit = want(s, cold)
    got = out.float().cpu().numpy().astype(np.float64)
    rows = np.arange(s["cu"][-1]) if rows is None else rows
    d = s["q"].shape[2]
    tol = mass * (2 * 2.0 ** -11 + 2 * (d + 8) * 2.0 ** -24 * logit[:, :, None])
    tol += np.abs(exp) * torch.finfo(s["dtype"]).eps / 2 + 2.0 ** -23
    err = np.abs(got - exp)[rows]
    print(f"[extend] largest error {err.max():.2e}, {(err / tol[rows]).max():.2f} of its bound", flush=True)
    assert (err <= tol[rows]).all(), (err / tol[rows]).max()


CASES = [
    # new, held (the new ones included), heads, kv, d, bs
    ([1], [1], 4, 4, 64, 16),
    ([1, 1, 1], [17, 1, 40], 8, 2, 128, 16),
    ([5, 5], [100, 37], 32, 8, 128, 16),                     # narrow tiles of 20 rows
    ([8, 9, 0, 31], [60, 9, 50, 300], 8, 2, 128, 16),        # 32 rows and 36; a request without new tokens
    ([70], [70], 6, 2, 64, 16),                              # from nothing, group 3
    ([33, 1, 130], [500, 600, 131], 16, 1, 64, 16),          # group 16, wide beside narrow
    ([40, 3], [333, 900], 4, 1, 128, 32),
    ([21, 50], [210, 64], 8, 8, 96, 16),                     # head_dim between the tiles'
    ([21, 50], [210, 64], 4, 2, 40, 8),
    ([17], [100], 4, 2, 128, 20),                            # a block that ends inside a sub-tile
    ([17, 2], [180, 64], 4, 2, 8, 64),
    ([12, 3], [50, 33], 4, 2, 64, 1),
    ([6], [5], 4, 2, 64, 16),                                # more rows than tokens: the first sees nothing
    ([2, 3], [0, 20], 4, 2, 64, 16),                         # a request that holds nothing
    ([3], [2100], 4, 1, 64, 16),                             # cut: many items per tile
]


@pytest.mark.parametrize("new,held,heads,kv,d,bs", CASES)
@pytest.mark.parametrize("fmt,cold,dtype", [("absmax_i8", "masked", torch.float16), ("absmax_i8", "zero_logit", torch.bfloat16),
                                            ("ref_u8", "zero_logit", torch.float16), ("ref_u8", "masked", torch.bfloat16)])
def test_extend_attention_matches_oracle(device, new, held, heads, kv, d, bs, fmt, cold, dtype):
    s = step(sum(held) + heads, new, held, heads, kv, d, bs, fmt, dtype, pad=2)
    out = torch.full(s["q"].shape, 7.0, dtype=dtype, device=device)
    got = call(s, device, cold, out=out, max_tokens=max(new))
    assert got.data_ptr() == out.data_ptr()
    check(out, s, cold)
    assert (out[s["cu"][-1]:] == 7.0).all()                  # rows behind the last request
    again = call(s, device, cold)                            # no bound given: the same rows, cut as they may be
    check(again, s, cold)


@pytest.mark.parametrize("cold", ["masked", "zero_logit"])
def test_extend_attention_with_blocks_of_any_length(device, cold):
    """Partial and empty blocks anywhere, COLD ones among the new tokens."""
    s = step(5, [20, 7, 40], [90, 300, 45], 8, 2, 64, holes=True, cold=0.4)
    rng = np.random.default_rng(9)
    inside = np.arange(s["table"].shape[1])[None] < s["nblocks"][:, None]
    s["states"][inside & (rng.random(inside.shape) < 0.3)] = COLD
    check(call(s, device, cold), s, cold)


def test_all_cold_and_all_masked_rows(device):
    s = step(6, [3, 4], [50, 60], 4, 2, 64)
    s["states"][0] = COLD
    out = call(s, device, "masked")
    assert (out[:3] == 0).all()
    check(out, s, "masked")
    out = call(s, device, "zero_logit")
    assert (out[:3] == 0).all()
    check(out, s, "zero_logit")


def test_values_that_no_row_sees_do_not_matter(device):
    """NaN and infinities past a block's length, in slots of no block and
    behind the block count change nothing; nor do those of a later token for
    the rows before it."""
    s = step(7, [9, 40], [50, 77], 8, 2, 128, spare=3)
    clean = call(s, device, "masked")
    hk, hv = s["hot"]
    used = np.zeros(hk.shape[:3:2], bool)
    for b in range(2):
        for i in range(s["nblocks"][b]):
            if s["states"][b, i] == HOT:
                used[s["table"][b, i], :s["lengths"][b, i]] = True
    bad = np.array([np.nan, np.inf, -np.inf], np.float16)
    for p in (hk, hv):
        fill = np.random.default_rng(1).choice(bad, p.shape)
        p[:] = np.where(used[:, None, :, None], p, fill)
    s["states"][:, -3:] = HOT
    s["table"][:, -3:] = 0
    s["lengths"][:, -3:] = 16
    assert torch.equal(call(s, device, "masked"), clean)
    # The last token of request 1: its own row is lost, the rows before it are not.
    last = s["nblocks"][1] - 1
    slot, pos = s["table"][1, last], s["lengths"][1, last] - 1
    for value in (np.nan, np.inf):
        hk[slot, :, pos, 3], hv[slot, :, pos, 5] = value, value
        out = call(s, device, "masked")
        assert torch.equal(out[:48], clean[:48])
        assert not torch.isfinite(out[48].float()).all()


def test_visible_infinities_arrive_where_they_belong(device):
    """An infinite V entry of a visible token gives that entry's dimension, in
    the rows that see it, and nothing else."""
    s = step(8, [40], [45], 4, 2, 64, cold=0, warm=0)
    clean = call(s, device, "masked")
    order = [(s["table"][0, i], t) for i in range(s["nblocks"][0]) for t in range(s["lengths"][0, i])]
    slot, pos = order[20]
    s["hot"][1][slot, 0, pos, 9] = -np.inf
    slot, pos = order[30]
    s["hot"][1][slot, 0, pos, 11] = np.inf
    out = call(s, device, "masked")
    first = 20 - 5                                # row of ordinal 20
    assert (out[first:, :2, 9] == -float("inf")).all() and (out[first + 10:, :2, 11] == float("inf")).all()
    hit = torch.zeros_like(clean, dtype=torch.bool)
    hit[first:, :2, 9] = True
    hit[first + 10:, :2, 11] = True
    assert torch.equal(out[~hit], clean[~hit])


def test_one_token_per_request_agrees_with_the_decode_kernel(device):
    s = step(11, [1] * 6, [30, 400, 16, 77, 5, 260], 32, 8, 128)
    out = call(s, device, "masked")
    ks, kz, vs, vz = (gpu(a, device) for a in s["meta"])
    ref, _ = tierkv_decode_attention(
        s["q"].to(device)[:, :, None], gpu(s["table"], device), gpu(s["states"], device), gpu(s["lengths"], device),
        gpu(s["hot"][0], device), gpu(s["hot"][1], device), gpu(s["warm"][0], device), gpu(s["warm"][1], device), ks, kz,
        vs, vz, s["table"].shape[1], 4, s["scaling"], cold_mode="masked", seq_num_blocks=gpu(s["nblocks"], device))
    torch.testing.assert_close(out, ref[:, 0], rtol=2e-3, atol=1e-3)
    check(out, s, "masked")


def test_strided_queries_and_any_memory_order(device):
    s = step(12, [9, 33], [80, 70], 8, 2, 64)
    q = s["q"].to(device)
    base = call(s, device, "masked")
    wide = torch.zeros((42, 8 + 4, 64 + 8), dtype=torch.float16, device=device)
    wide[:, 2:10, :64] = q
    assert torch.equal(call(s, device, "masked", q=wide[:, 2:10, :64]), base)
    by_head = q.transpose(0, 1).contiguous().transpose(0, 1)         # [heads, tokens, dim] storage
    assert torch.equal(call(s, device, "masked", q=by_head), base)
    odd = torch.zeros((42, 8, 67), dtype=torch.float16, device=device)
    odd[:, :, 1:65] = q
    assert torch.equal(call(s, device, "masked", q=odd[:, :, 1:65]), base)


@pytest.mark.parametrize("dtype,scale", [(torch.bfloat16, 2.0 ** 40), (torch.bfloat16, 2.0 ** -40), (torch.bfloat16, 0.0),
                                         (torch.float16, 0.0)])
def test_queries_far_from_one(device, dtype, scale):
    """bf16 rows of any magnitude: the scaling takes it back, so the logits are
    ordinary; a row of zeros is a mean."""
    s = step(13, [5, 40], [80, 70], 4, 2, 64, dtype=dtype)
    s["q"] = (s["q"].float() * scale).to(dtype)
    if scale:
        s["scaling"] = s["scaling"] / scale
    check(call(s, device, "masked"), s, "masked")


def test_bad_slots_and_states_are_skipped_and_reported(device):
    s = step(14, [3, 40], [200, 90], 4, 2, 64, cold=0)
    s["table"][0, 1], s["states"][0, 1] = 10 ** 6, HOT
    s["table"][0, 2], s["states"][0, 2] = -5, WARM
    s["states"][1, 1] = 9
    ws = DecodeWorkspace(device)
    out = call(s, device, "masked", workspace=ws)
    assert ws.error_word() == 3 and ws.error_word() == 0
    t = {**s, "states": s["states"].copy()}
    t["states"][0, 1] = t["states"][0, 2] = t["states"][1, 1] = COLD
    check(out, t, "masked")


def test_extend_attention_is_reproducible_and_shares_a_workspace(device):
    """The same bits in any workspace, after launches of other shapes and
    single-token launches that used it in between."""
    s = step(15, [3, 200], [2500, 700], 8, 2, 128)
    small = step(16, [1, 1], [700, 90], 8, 2, 128)
    ws = DecodeWorkspace(device)
    first = call(s, device, "masked", workspace=ws)
    ks, kz, vs, vz = (gpu(a, device) for a in small["meta"])
    for _ in range(2):
        for splits in (None, 3):
            out, _ = tierkv_decode_attention(
                small["q"].to(device)[:, :, None], gpu(small["table"], device), gpu(small["states"], device),
                gpu(small["lengths"], device), gpu(small["hot"][0], device), gpu(small["hot"][1], device),
                gpu(small["warm"][0], device), gpu(small["warm"][1], device), ks, kz, vs, vz, small["table"].shape[1], 4,
                small["scaling"], cold_mode="masked", seq_num_blocks=gpu(small["nblocks"], device), workspace=ws,
                splits=splits)
            torch.testing.assert_close(out[:, 0], call(small, device, "masked", workspace=ws), rtol=2e-3, atol=1e-3)
        assert torch.equal(call(s, device, "masked", workspace=ws), first)
    assert torch.equal(call(s, device, "masked"), first)


def tables(rng, batch, width, bs, slots, full=False):
    nblocks = rng.integers(0, max(1, width // 2), batch).astype(np.int32)
    table = np.full((batch, width), -1, np.int32)
    states, lengths = np.full((batch, width), COLD, np.int32), np.zeros((batch, width), np.int32)
    ids = rng.permutation(slots).astype(np.int32)
    used = 0
    for b in range(batch):
        n = nblocks[b]
        table[b, :n] = ids[used:used + n]
        used += n
        states[b, :n] = rng.choice([HOT, WARM, COLD], n)
        lengths[b, :n] = bs
        if n:
            lengths[b, n - 1] = rng.integers(1, bs + 1)
            states[b, n - 1] = HOT if rng.random() < 0.9 else WARM
    opened = (rng.random(batch) < 0.7).astype(np.int32)
    free = np.ascontiguousarray(ids[used:])
    return table, states, lengths, nblocks, opened, free, np.array([len(free), 0, 0, 0], np.int32)


@pytest.mark.parametrize("batch,top,width,bs,slack", [
    (1, 1, 8, 16, 0), (1, 40, 16, 16, 3), (64, 1, 40, 16, 0), (64, 5, 40, 16, 7), (7, 300, 64, 8, 1),
    (300, 90, 40, 16, 5), (1025, 3, 12, 16, 2), (4096, 2, 8, 16, 0), (2, 5000, 700, 16, 0), (33, 70, 12, 64, 9),
    (5, 9, 80, 1, 0),
])
def test_slot_map_matches_oracle(device, batch, top, width, bs, slack):
    rng = np.random.default_rng(batch * 31 + top)
    new = rng.integers(0, top + 1, batch).astype(np.int32)
    if batch == 1:
        new[:] = top
    state = tables(rng, batch, width, bs, batch * (width + top // bs + 2))
    rows = int(new.sum()) + slack
    host = [a.copy() for a in state]
    dev = [gpu(a, device) for a in state]
    for _ in range(2):          # two steps in a row
        exp = serving.build_slot_map(new, *host, bs, rows)
        m = kernels.build_slot_map(gpu(new, device), *dev, bs, rows)
        for name, g, e in zip(("slots", "positions", "cu", "context"), m, exp):
            np.testing.assert_array_equal(g.cpu().numpy(), e, err_msg=name)
        for name, g, e in zip(("table", "states", "lengths", "nblocks", "open", "free", "ctl"), dev, host):
            np.testing.assert_array_equal(g.cpu().numpy(), e, err_msg=name)


@pytest.mark.parametrize("batch", [3, 1500])
@pytest.mark.parametrize("why,bit", [("blocks", 1), ("table", 4), ("rows", 16), ("negative", 16)])
def test_a_step_that_does_not_fit_changes_nothing(device, batch, why, bit):
    rng = np.random.default_rng(batch)
    state = list(tables(rng, batch, 12, 16, batch * 16))
    new = np.full(batch, 20, np.int32)
    rows = int(new.sum())
    if why == "blocks":
        state[6][0] = batch          # each needs one block at least, some two
    if why == "table":
        new[batch - 1] = 16 * 12 + 1
        rows += 16 * 12
    if why == "rows":
        rows -= 1
    if why == "negative":
        new[1] = -1
    host, dev = [a.copy() for a in state], [gpu(a, device) for a in state]
    exp = serving.build_slot_map(new, *host, 16, rows)
    m = kernels.build_slot_map(gpu(new, device), *dev, 16, rows)
    assert (m.slots == -1).all() and (m.positions == -1).all() and (m.cu_tokens == 0).all()
    np.testing.assert_array_equal(m.context.cpu().numpy(), exp[3])
    for g, e in zip(dev[:6], state[:6]):
        np.testing.assert_array_equal(g.cpu().numpy(), e)
    assert dev[6][2].item() & bit and dev[6][3].item() == 0 and dev[6][0].item() == state[6][0]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,kv,d,bs,layout", [
    (1, 1, 64, 16, "plain"), (37, 8, 128, 16, "plain"), (300, 4, 96, 16, "fused"), (50, 2, 20, 8, "plain"),
    (50, 2, 33, 16, "fused"), (64, 3, 64, 64, "heads"), (40, 2, 64, 16, "odd"), (1, 2, 64, 16, "dims"),
])
def test_write_slots_matches_indexing(device, dtype, n, kv, d, bs, layout):
    g = torch.Generator().manual_seed(n + d)
    x = torch.randn((2, n, kv, d), generator=g).to(dtype).to(device)
    k, v = x[0], x[1]
    if layout == "fused":
        f = torch.cat([k.reshape(n, -1), v.reshape(n, -1)], 1)
        k, v = f[:, :kv * d].view(n, kv, d), f[:, kv * d:].view(n, kv, d)
    if layout == "heads":
        k, v = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (k, v))
    if layout == "odd":
        k, v = (torch.cat([t, t[..., :3]], 2)[..., :d] for t in (k, v))
    if layout == "dims":
        k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    blocks = (n + bs - 1) // bs + 2
    hot = torch.randn((2, blocks, kv, bs, d), generator=g).half().to(device)
    slots = torch.randperm(blocks * bs, generator=g)[:n].int()
    slots[::7] = -1
    if n > 3:
        slots[3] = blocks * bs          # past the pool: skipped
    exp = hot.clone()
    keep = (slots >= 0) & (slots < blocks * bs)
    s, at = slots[keep].long().to(device), keep.nonzero()[:, 0].to(device)
    for p, t in zip(exp, (k, v)):
        p[s // bs, :, s % bs] = t[at].half()
    kernels.write_slots(k, v, slots.to(device), hot[0], hot[1])
    assert torch.equal(hot, exp)


def logits(rng, batch, vocab, dtype, kind):
    x = rng.standard_normal((batch, vocab)) * 2.5
    if kind == "peaked":
        x[np.arange(batch), rng.integers(0, vocab, batch)] += 14
    if kind == "flat":
        x[:] = 0.75
    if kind == "ties":
        x = np.round(x)
    if kind == "masked":
        x[rng.random(x.shape) < 0.6] = -np.inf
        x[:, vocab // 2] = np.nan
        low = rng.random(x.shape) < 0.2
        x[low] = -6e4
    return torch.from_numpy(x.astype(np.float32)).to(dtype)


LIMITS = [dict(), dict(temperature=0.0), dict(top_k=1), dict(top_k=40), dict(top_k=10 ** 6), dict(top_p=0.9), dict(top_p=0.0),
          dict(min_p=0.05), dict(temperature=0.6, top_k=50, top_p=0.8, min_p=0.01), dict(temperature=3.0, top_p=0.97),
          dict(temperature=1e-4), dict(temperature=float("inf"), top_k=7), dict(min_p=1.0)]


@pytest.mark.parametrize("kind", ["plain", "peaked", "flat", "ties", "masked"])
@pytest.mark.parametrize("batch,vocab,dtype", [(1, 1, torch.float32), (3, 2, torch.float16), (5, 63, torch.bfloat16),
                                               (4, 1000, torch.float32), (3, 32000, torch.float16),
                                               (2, 50257, torch.bfloat16), (2, 128256, torch.float32)])
def test_sampling_matches_oracle(device, kind, batch, vocab, dtype):
    rng = np.random.default_rng(vocab + batch)
    x = logits(rng, batch, vocab, dtype, kind)
    for i, kw in enumerate(LIMITS):
        u = rng.random(batch).astype(np.float32)
        u[0] = (0.0, 1 - 2.0 ** -24, u[0])[i % 3]
        tok, prob = kernels.sample_tokens(x.to(device), torch.from_numpy(u).to(device), **kw)
        exp = [serving.sample_row(x[b].float().numpy(), u[b], **kw) for b in range(batch)]
        assert tok.tolist() == [e[0] for e in exp], (kind, kw)
        np.testing.assert_allclose(prob.cpu().numpy(), [e[1] for e in exp], rtol=2.0 ** -23)


def test_sampling_with_limits_of_each_row(device):
    rng = np.random.default_rng(3)
    batch, vocab = 40, 5000
    x = logits(rng, batch, vocab, torch.float16, "plain")
    u = rng.random(batch).astype(np.float32)
    t = np.where(rng.random(batch) < 0.2, 0, rng.random(batch) * 2).astype(np.float32)
    k = rng.integers(0, 60, batch).astype(np.int32)
    p = rng.random(batch).astype(np.float32) * 1.2
    m = (rng.random(batch) * 0.2).astype(np.float32)
    dev = lambda a: torch.from_numpy(a).to(device)
    wide = torch.zeros((batch, vocab + 40), dtype=torch.float16)
    wide[:, :vocab] = x
    got, _ = kernels.sample_tokens(wide.to(device)[:, :vocab], dev(u), dev(t), dev(k), dev(p), dev(m))
    assert got.tolist() == [serving.sample_row(x[b].float().numpy(), u[b], t[b], int(k[b]), p[b], m[b])[0]
                            for b in range(batch)]


def test_rows_without_a_token(device):
    x = torch.full((3, 100), -float("inf"), device=device)
    x[1, 40] = float("inf")
    x[2] = float("nan")
    tok, prob = kernels.sample_tokens(x, torch.tensor([0.5, 0.5, 0.5], device=device), top_k=5, top_p=0.5)
    assert tok.tolist() == [-1, 40, -1] and prob.tolist() == [0.0, 1.0, 0.0]


def test_a_step_as_a_server_runs_it_captured_and_replayed(device):
    """Lengths -> slot map -> row writes -> attention -> tokens, eager and as a
    graph replayed with other lengths, against the oracle step by step."""
    rng = np.random.default_rng(21)
    B, heads, kv, d, bs, width, vocab, cap = 5, 8, 2, 64, 16, 24, 999, 48
    slots = B * width
    state = [np.full((B, width), -1, np.int32), np.full((B, width), COLD, np.int32), np.zeros((B, width), np.int32),
             np.zeros(B, np.int32), np.zeros(B, np.int32), rng.permutation(slots).astype(np.int32),
             np.array([slots, 0, 0, 0], np.int32)]
    host, dev = [a.copy() for a in state], [gpu(a, device) for a in state]
    hk, hv = (np.zeros((slots, kv, bs, d), np.float16) for _ in range(2))
    pools = [gpu(hk, device), gpu(hv, device)]
    warm = [torch.zeros((1, kv, bs, d), dtype=torch.int8, device=device)] * 2
    meta = torch.ones((1, kv), device=device)
    new = torch.zeros(B, dtype=torch.int32, device=device)
    q = torch.zeros((cap, heads, d), dtype=torch.float16, device=device)
    kx, vx = (torch.zeros((cap, kv, d), dtype=torch.float16, device=device) for _ in range(2))
    x, u = torch.zeros((B, vocab), device=device), torch.zeros(B, device=device)
    out = torch.zeros_like(q)
    ws = extend_workspace(device, B, cap, heads, kv, width, d)

    def run():
        m = kernels.build_slot_map(new, *dev, bs, cap)
        kernels.write_slots(kx, vx, m.slots, *pools)
        tierkv_extend_attention(q, m.cu_tokens, dev[0], dev[1], dev[2], *pools, *warm, meta, None, meta, None, width,
                                heads // kv, d ** -0.5, cold_mode="masked", seq_num_blocks=dev[3], workspace=ws, out=out)
        return m, kernels.sample_tokens(x, u, top_p=0.9)

    graph = None
    for it, lens in enumerate([[7, 0, 1, 20, 3], [1, 1, 1, 1, 1], [0, 9, 30, 1, 2], [1, 2, 3, 4, 5], [16, 0, 0, 16, 16],
                               [0, 0, 0, 0, 0], [3, 1, 1, 1, 1]]):
        n = np.array(lens, np.int32)
        total = int(n.sum())
        new.copy_(gpu(n, device))
        for t in (q, kx, vx, x, u):
            t.copy_(torch.from_numpy((rng.random(t.shape) if t is u else rng.standard_normal(t.shape)).astype(np.float32)))
        if it == 2:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                res = run()
        if graph is not None:
            graph.replay()
        else:
            res = run()
        torch.cuda.synchronize()
        m, (tok, _) = res
        exp = serving.build_slot_map(n, *host, bs, cap)
        for g, e in zip(m, exp):
            np.testing.assert_array_equal(g.cpu().numpy(), e)
        for r in range(total):
            for pool, rows in ((hk, kx), (hv, vx)):
                pool[exp[0][r] // bs, :, exp[0][r] % bs] = rows[r].cpu().numpy()
        assert torch.equal(pools[0].cpu(), torch.from_numpy(hk)) and torch.equal(pools[1].cpu(), torch.from_numpy(hv))
        s = dict(q=q.cpu(), cu=exp[2], table=host[0], states=host[1], lengths=host[2], nblocks=host[3], hot=(hk, hv),
                 warm=[w.cpu().numpy() for w in warm], meta=(meta.cpu().numpy(), None, meta.cpu().numpy(), None),
                 groups=heads // kv, scaling=d ** -0.5, fmt="absmax_i8", dtype=torch.float16)
        if total:
            check(out, s, "masked", np.arange(total))
        assert tok.tolist() == [serving.sample_row(x[b].cpu().numpy(), u[b].item(), top_p=0.9)[0] for b in range(B)]


def test_steps_on_two_streams_do_not_mix(device):
    a, b = step(31, [3, 90], [900, 200], 8, 2, 64), step(32, [60, 2], [70, 1500], 8, 2, 128)
    xa = torch.randn((8, 40000), device=device)
    ua = torch.rand(8, device=device)
    base = call(a, device, "masked"), call(b, device, "masked"), kernels.sample_tokens(xa, ua, top_p=0.9)[0]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    res = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                res[i].append((call((a, b)[i], device, "masked"), kernels.sample_tokens(xa, ua, top_p=0.9)[0]))
    torch.cuda.synchronize()
    for i in (0, 1):
        for out, tok in res[i]:
            assert torch.equal(out, base[i]) and torch.equal(tok, base[2])


def test_a_query_that_starts_off_a_16_byte_boundary(device):
    s = step(31, [3, 12], [40, 25], 8, 2, 64)
    q = s["q"].to(device)
    flat = torch.zeros(q.numel() + 3, dtype=q.dtype, device=device)
    flat[3:] = q.flatten()
    assert torch.equal(call(s, device, "masked", q=flat[3:].view(q.shape)), call(s, device, "masked"))


@pytest.mark.parametrize("new,held,heads,kv,d", [
    ([i % 4 for i in range(1500)], [5 + i % 37 for i in range(1500)], 4, 1, 32),      # more requests than plan threads
    ([100, 1, 70, 0, 2], [2000, 3000, 70, 50, 1], 16, 1, 64),                         # some tiles cut, others whole
    ([70] * 40, [70 + 10 * i for i in range(40)], 16, 8, 64),                         # more tiles than run at once
])
def test_cuts_of_many_tiles(device, new, held, heads, kv, d):
    s = step(32, new, held, heads, kv, d)
    out = call(s, device, "masked")
    rng = np.random.default_rng(32)
    check(out, s, "masked", np.sort(rng.choice(s["cu"][-1], min(400, int(s["cu"][-1])), replace=False)))
    assert torch.equal(out[:s["cu"][-1]], call(s, device, "masked")[:s["cu"][-1]])


def test_limits_of_each_row_past_32_bits(device):
    x = logits(np.random.default_rng(5), 3, 700, torch.float32, "plain").to(device)
    u = torch.tensor([0.9, 0.5, 0.99], device=device)
    k = torch.tensor([2 ** 32 + 1, -2 ** 40, 2 ** 31], dtype=torch.int64, device=device)   # all off
    got = kernels.sample_tokens(x, u, top_k=k)
    assert all(torch.equal(a, b) for a, b in zip(got, kernels.sample_tokens(x, u)))
    assert torch.equal(kernels.sample_tokens(x, u, top_k=2 ** 40)[0], got[0])


def test_one_graph_follows_the_requests_rows(device):
    """A captured call replayed with other numbers of new tokens, so other tiles and cuts, beside eager work."""
    s = step(33, [20, 20], [600, 90], 8, 2, 64)
    ks, kz, vs, vz = (gpu(a, device) for a in s["meta"])
    pools = [gpu(a, device) for a in (*s["hot"], *s["warm"])]
    tables = [gpu(s[n], device) for n in ("table", "states", "lengths", "nblocks")]
    q, cu = s["q"].to(device), gpu(s["cu"], device)
    out = torch.empty_like(q)
    ws = extend_workspace(device, 2, 40, 8, 2, s["table"].shape[1], 64)
    run = lambda: tierkv_extend_attention(q, cu, *tables[:3], *pools, ks, kz, vs, vz, s["table"].shape[1], 4, s["scaling"],
                                          cold_mode="masked", seq_num_blocks=tables[3], workspace=ws, out=out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            run()
    torch.cuda.synchronize()
    for rows in ([5, 30], [40, 0], [1, 1], [0, 0], [0, 33], [8, 9], [20, 20]):
        s["cu"] = np.array([0, rows[0], sum(rows)], np.int32)
        cu.copy_(torch.from_numpy(s["cu"]))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert (out[sum(rows):] == 7.0).all()
        if sum(rows):
            check(out, s, "masked")
            assert torch.equal(call(s, device, "masked")[:sum(rows)], out[:sum(rows)])   # (an eager call of its own)
