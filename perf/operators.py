"""The operators of a serving step over requests of different lengths, as
measurable cases: the slot map of the step's new tokens, the write of their
K/V rows, the attention of several query tokens per request over the tiered
cache, and the choice of the next tokens.

A case is a dict of plain values; ``prepare`` makes what a serving program
holds before the call from a seed, ``run`` makes one pass (the plain form in
elementary torch operations, or with ``own`` the package's entry points),
``work`` counts the bytes and operations a pass cannot do without, and
``exact`` gives the outputs in 64 bits from the definitions.

Kinds of cases:

* ``slots``   ``kernels.build_slot_map``: lengths of the requests' new tokens
              -> table entries of new blocks, the packed rows' slots and
              positions.  The tables are restored at the start of a pass.
* ``write``   ``kernels.write_slots``: packed K/V rows into the HOT pools.
* ``extend``  ``tierkv_extend_attention``: the last n[b] tokens of each
              request attend to the request's tokens up to themselves.
* ``sample``  ``kernels.sample_tokens``: temperature, top-k, top-p, min-p and
              the draw from given random numbers; the tokens and the
              probabilities that they had.
"""

import math

import numpy as np
import torch

own = False

HOT, WARM, COLD = 0, 1, 2
BS = 16                    # tokens per block, in every configuration of this package
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
WEIGHT_ONE = float(1 << 42)   # the likeliest token's weight when sampling


def _ceil(a, b):
    return -(-a // b)


# --- cases -------------------------------------------------------------------

def _slots(name, batch, new, blocks, pattern):
    return dict(name=name, op="slots", batch=batch, new=new, blocks=blocks, pattern=pattern)


def _write(name, tokens, kv_heads, head_dim, dtype, fused):
    return dict(name=name, op="write", tokens=tokens, kv_heads=kv_heads, head_dim=head_dim, dtype=dtype, fused=fused)


def _extend(name, batch, ctx, new, pattern, heads, kv_heads, head_dim, fmt="absmax_i8", cold="masked", dtype="fp16"):
    return dict(name=name, op="extend", batch=batch, ctx=ctx, new=new, pattern=pattern, heads=heads,
                kv_heads=kv_heads, head_dim=head_dim, fmt=fmt, cold=cold, dtype=dtype)


def _sample(name, batch, vocab, dtype, top_k, top_p, min_p, per_row):
    return dict(name=name, op="sample", batch=batch, vocab=vocab, dtype=dtype, top_k=top_k, top_p=top_p, min_p=min_p,
                per_row=per_row)


def listed():
    return [
        # A decode step of 64 requests: one new token each.
        _slots("slots_decode_64", 64, 1, 256, "same"),
        # A step that takes 256 requests' prompts of very different lengths at once.
        _slots("slots_prompts_256", 256, 700, 144, "ragged"),
        # The K/V rows of a decode step, 8 heads of 128.
        _write("write_decode_64", 64, 8, 128, "fp16", False),
        # The K/V rows of one prefill step, read out of a fused q/k/v projection.
        _write("write_prompts_16384", 16384, 8, 128, "bf16", True),
        # Drafted tokens to verify: 8 requests of 4096 tokens, 5 tokens each.
        _extend("verify_8x5_ctx4096", 8, 4096, 5, "same", 32, 8, 128),
        # Small-model requests (32 / 4 heads of 64) of very different lengths, one to a few new tokens,
        # the reference's WARM format and COLD rule.
        _extend("mixed_32_d64_ref", 32, 1500, 9, "ragged", 32, 4, 64, "ref_u8", "zero_logit", "bf16"),
        # A step of decoding requests together with one request's prompt piece.
        _extend("piece_512_beside_15", 16, 2048, 512, "one_long", 32, 8, 128, "absmax_i8", "masked", "bf16"),
        # Fresh prompts of odd lengths: no context, everything HOT, plain causal attention.
        _extend("prompts_4x1001", 4, 0, 1001, "ragged", 32, 8, 128),
        # A follow-up prompt of 2048 tokens on 32768 tokens of context.
        _extend("follow_up_2048_ctx32768", 1, 32768, 2048, "same", 32, 8, 128),
        # One request's next token, vocabulary of 32000.
        _sample("sample_1x32000", 1, 32000, "fp16", 50, 0.9, 0.0, False),
        # A decode step of 16 requests, vocabulary of 128256, nucleus sampling without a top-k.
        _sample("sample_16x128256", 16, 128256, "bf16", 0, 0.95, 0.0, False),
        # A large batch in 32 bits, every request with filters of its own.
        _sample("sample_256x128256", 256, 128256, "fp32", 64, 0.9, 0.02, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["slots", "write", "extend", "extend", "extend", "sample", "sample"])
    if op == "slots":
        batch = _log(rng, 1, 300)
        new = _log(rng, 1, max(1, 150000 // batch))
        case = _slots("", batch, min(new, 8000), _ceil(min(new, 8000), BS) + _log(rng, 8, 160),
                      rng.choice(["same", "ragged", "one_long"]))
    elif op == "write":
        kv_heads = rng.choice([1, 2, 4, 8])
        head_dim = rng.choice([64, 96, 128])
        case = _write("", _log(rng, 1, 16384 * 8 * 128 // (kv_heads * head_dim * 4)), kv_heads, head_dim,
                      rng.choice(["fp16", "bf16"]), rng.random() < 0.5)
    elif op == "extend":
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
        head_dim = rng.choice([64, 128])
        batch = _log(rng, 1, 48)
        pattern = rng.choice(["same", "ragged", "one_long"])
        rows = 1 if pattern == "one_long" else batch
        new = _log(rng, 1, max(1, min(2048, 8192 // rows)))
        ctx = 0 if rng.random() < 0.15 else _log(rng, 16, max(16, min(32768, 120000 // batch)))
        # No dearer than the dearest listed case: 2048 tokens of 32 heads of 128 on 32768.
        while rows * new * (ctx + new) * heads * head_dim > 1.2e11 and ctx > 16:
            ctx = max(16, ctx // 2)
        case = _extend("", batch, ctx, new, pattern, heads, kv_heads, head_dim, rng.choice(["absmax_i8", "ref_u8"]),
                       rng.choice(["masked", "zero_logit"]), rng.choice(["fp16", "bf16"]))
    else:
        vocab = _log(rng, 1000, 200000)
        case = _sample("", _log(rng, 1, max(1, min(256, 256 * 128256 // vocab))), vocab,
                       rng.choice(["fp16", "bf16", "fp32"]), rng.choice([0, 0, 1, 20, 50, 400]),
                       rng.choice([1.0, 0.5, 0.9, 0.98]), rng.choice([0.0, 0.0, 0.05]), rng.random() < 0.5)
    del case["name"]
    return case


# --- lengths -----------------------------------------------------------------

def _new_tokens(case):
    """New tokens per request."""
    n, batch = case["new"], case["batch"]
    if case["pattern"] == "same":
        return [n] * batch
    if case["pattern"] == "one_long":
        return [n] + [1] * (batch - 1)
    return [max(1, n - (b * 37) % max(1, n)) if b % 5 else n for b in range(batch)]


def _context(case):
    """Tokens each request holds before the step."""
    ctx, batch = case["ctx"], case["batch"]
    if case["pattern"] == "same" or ctx < 8:
        return [ctx] * batch
    return [ctx - (b * 131) % (ctx // 2 + 1) for b in range(batch)]


def _blocks_of(ctx, n):
    """Valid tokens of each block: the context's blocks (the last one partly
    filled), then the new tokens' own blocks, as this package appends them."""
    out = [BS] * (ctx // BS) + ([ctx % BS] if ctx % BS else [])
    return out + [BS] * (n // BS) + ([n % BS] if n % BS else [])


def _tiers(ctx, n, seed):
    """States of a request's blocks: the first, the last 4 of the context and
    every block of the new tokens HOT, of the others 10 % HOT, 60 % WARM and
    the rest COLD."""
    old = _ceil(ctx, BS)
    states = np.full(old + _ceil(n, BS), HOT, dtype=np.int32)
    if old > 5:
        r = np.random.default_rng(seed).random(old - 5)
        states[1:old - 4] = np.where(r < 0.1, HOT, np.where(r < 0.7, WARM, COLD))
    return states


# --- inputs ------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)
    return {"slots": _prepare_slots, "write": _prepare_write, "extend": _prepare_extend,
            "sample": _prepare_sample}[case["op"]](case, int(seed), gen)


def _prepare_slots(case, seed, gen):
    rng = np.random.default_rng(seed)
    batch, width = case["batch"], case["blocks"]
    new = np.array(_new_tokens(case), dtype=np.int32)
    room_for = width - _ceil(int(new.max()), BS)
    nb = rng.integers(1, max(2, room_for), batch).astype(np.int32)
    lengths = np.zeros((batch, width), np.int32)
    states = np.full((batch, width), COLD, np.int32)
    used = int(nb.sum())
    free = used + int(sum(_ceil(int(n), BS) for n in new)) + 64
    slots = rng.permutation(used + free).astype(np.int32)
    table = np.full((batch, width), -1, np.int32)
    at = 0
    for b in range(batch):
        lengths[b, :nb[b]] = BS
        lengths[b, nb[b] - 1] = rng.integers(1, BS + 1)
        states[b, :nb[b]] = rng.choice([HOT, WARM], nb[b])
        states[b, nb[b] - 1] = HOT
        table[b, :nb[b]] = slots[at:at + nb[b]]
        at += nb[b]
    last = lengths[np.arange(batch), nb - 1]
    opened = ((last < BS) & (rng.random(batch) < 0.8)).astype(np.int32)
    ctl = np.array([free, 0, 0, 0], np.int32)
    # One buffer for all of it, so that a pass restores the state with one copy.
    parts = [table, states, lengths, nb, opened, ctl]
    sizes = [_ceil(p.size, 64) * 64 for p in parts]
    flat = np.zeros(sum(sizes), np.int32)
    views, at = [], 0
    for p, s in zip(parts, sizes):
        flat[at:at + p.size] = p.ravel()
        views.append((at, p.size, p.shape))
        at += s
    start = torch.from_numpy(flat).cuda()
    work = start.clone()
    names = ("table", "states", "lengths", "nblocks", "open", "ctl")
    st = {name: work[a:a + n].view(shape) for name, (a, n, shape) in zip(names, views)}
    st.update(op="slots", start=start, work=work, new=torch.from_numpy(new).cuda(), rows=int(new.sum()) + 3,
              free=torch.from_numpy(np.ascontiguousarray(slots[used:])).cuda())
    return st


def _prepare_write(case, seed, gen):
    n, kv, d = case["tokens"], case["kv_heads"], case["head_dim"]
    dt = DTYPES[case["dtype"]]
    if case["fused"]:     # K and V are column ranges of one projection
        x = torch.randn((n, 4 * kv * d), generator=gen, device="cuda").to(dt)
        k = x[:, 2 * kv * d:3 * kv * d].view(n, kv, d)
        v = x[:, 3 * kv * d:].view(n, kv, d)
    else:
        k = torch.randn((n, kv, d), generator=gen, device="cuda").to(dt)
        v = torch.randn((n, kv, d), generator=gen, device="cuda").to(dt)
    blocks = _ceil(n, BS) + 16
    rng = np.random.default_rng(seed)
    order = rng.permutation(blocks)[:_ceil(n, BS)]
    rows = (order[:, None] * BS + np.arange(BS)[None]).ravel()[:n].astype(np.int32)
    rows[rng.random(n) < 0.01] = -1          # rows of a padded step
    pool = torch.randn((2, blocks, kv, BS, d), generator=gen, device="cuda").to(torch.float16)
    return dict(op="write", k=k, v=v, slots=torch.from_numpy(rows).cuda(), hot_k=pool[0], hot_v=pool[1])


def _quantize(x, fmt):
    """WARM codes and metadata of fp16 tiles [slots, kv, bs, d], in the shapes
    of the package's pools."""
    xf = x.float()
    if fmt == "absmax_i8":
        s = xf.abs().amax(dim=(2, 3)) / 127.0
        q = torch.round(xf / s[:, :, None, None]).clamp(-127, 127)
        return q.to(torch.int8), s, None
    lo, hi = xf.amin(-1, keepdim=True), xf.amax(-1, keepdim=True)
    s = ((hi - lo) / 255.0).to(torch.float16)
    z = (-torch.round(lo / s.float())).to(torch.float16)
    q = (torch.round(xf / s.float()) + z.float()).clamp(0, 255)
    return q.to(torch.uint8), s, z


def _prepare_extend(case, seed, gen):
    batch, kv, d = case["batch"], case["kv_heads"], case["head_dim"]
    new, ctx = _new_tokens(case), _context(case)
    lens = [_blocks_of(c, n) for c, n in zip(ctx, new)]
    width = max(len(x) for x in lens)
    rng = np.random.default_rng(seed)
    states = np.full((batch, width), COLD, np.int32)
    lengths = np.zeros((batch, width), np.int32)
    table = np.full((batch, width), -1, np.int32)
    for b in range(batch):
        k = len(lens[b])
        lengths[b, :k] = lens[b]
        states[b, :k] = _tiers(ctx[b], new[b], seed * 1000 + b)
    within = np.arange(width)[None] < np.array([len(x) for x in lens])[:, None]
    pools = {}
    for tier, name in ((HOT, "hot"), (WARM, "warm")):
        at = np.nonzero(within & (states == tier))
        count = max(1, len(at[0]))
        table[at] = rng.permutation(count)[:len(at[0])]
        x = torch.randn((2, count, kv, BS, d), generator=gen, device="cuda").to(torch.float16)
        if tier == HOT and ctx[0] > 0:
            first = torch.from_numpy(table[:, 0].astype(np.int64)).cuda()
            x[0, first, :, :4] *= 4          # the first tokens draw attention
        pools[name] = x
    (wk, ks, kz), (wv, vs, vz) = (_quantize(pools["warm"][i], case["fmt"]) for i in (0, 1))
    total = sum(new)
    q = torch.randn((total + 2, case["heads"], d), generator=gen, device="cuda").to(DTYPES[case["dtype"]])
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    cuda = lambda a: torch.from_numpy(a).cuda()
    return dict(op="extend", q=q, cu=cuda(cu), table=cuda(table), states=cuda(states), lengths=cuda(lengths),
                nblocks=cuda(np.array([len(x) for x in lens], np.int32)), hot_k=pools["hot"][0],
                hot_v=pools["hot"][1], warm_k=wk, warm_v=wv, k_scale=ks, k_zero=kz, v_scale=vs, v_zero=vz,
                width=width, groups=case["heads"] // kv, scaling=d ** -0.5, cold=case["cold"], new=new,
                held=[len(x) for x in lens], tokens=[sum(x) for x in lens], max_new=max(new),
                out=torch.zeros_like(q))    # the two rows behind the last request stay zero


def _prepare_sample(case, seed, gen):
    batch, vocab = case["batch"], case["vocab"]
    x = torch.randn((batch, vocab), generator=gen, device="cuda") * 2.2
    likely = torch.randint(0, vocab, (batch, 24), generator=gen, device="cuda")
    x.scatter_(1, likely, 6.0 + 3.0 * torch.randn((batch, 24), generator=gen, device="cuda"))
    x = x.to(DTYPES[case["dtype"]])
    u = torch.rand(batch, generator=gen, device="cuda")
    if case["per_row"]:
        r = torch.rand((4, batch), generator=gen, device="cuda")
        t = 0.4 + r[0]
        t[0] = 0.0                           # one request takes its likeliest token
        k = (r[1] * 2 * case["top_k"]).to(torch.int32)
        p = (case["top_p"] + (r[2] - 0.5) * 0.1).clamp(0.05, 1.0)
        m = r[3] * 2 * case["min_p"]
        return dict(op="sample", x=x, u=u, temperature=t, top_k=k, top_p=p, min_p=m)
    return dict(op="sample", x=x, u=u, temperature=0.8, top_k=case["top_k"], top_p=case["top_p"],
                min_p=case["min_p"])


# --- one pass ----------------------------------------------------------------

def run(state):
    return {"slots": _run_slots, "write": _run_write, "extend": _run_extend, "sample": _run_sample}[state["op"]](state)


def _run_slots(st):
    st["work"].copy_(st["start"])
    if own:
        from paged_tierkv_amd import kernels

        m = kernels.build_slot_map(st["new"], st["table"], st["states"], st["lengths"], st["nblocks"], st["open"],
                                   st["free"], st["ctl"], BS, st["rows"])
        slots, positions, cu, context = m.slots, m.positions, m.cu_tokens, m.context
    else:
        slots, positions, cu, context = _plain_slots(st)
    return dict(slots=slots, positions=positions, cu=cu, context=context, table=st["table"], states=st["states"],
                lengths=st["lengths"], nblocks=st["nblocks"], open=st["open"], ctl=st["ctl"])


def _plain_slots(st):
    n, nb = st["new"].long(), st["nblocks"].long()
    table, states, lengths, ctl = st["table"], st["states"], st["lengths"], st["ctl"]
    batch, width = table.shape
    rows = st["rows"]
    at = (nb - 1).clamp(min=0)[:, None]
    last = lengths.gather(1, at)[:, 0].long()
    open_ = (st["open"] != 0) & (nb > 0) & (states.gather(1, at)[:, 0] == HOT) & (last < BS)
    room = torch.where(open_, BS - last, 0)
    need = torch.div((n - room).clamp(min=0) + BS - 1, BS, rounding_mode="floor")
    first = need.cumsum(0) - need
    end = n.cumsum(0)
    cu = torch.cat([end.new_zeros(1), end])
    inside = torch.arange(width, device=n.device)[None] < nb[:, None]
    held = torch.where(inside, lengths, 0).sum(1)
    top = ctl[0].long()
    ok = (need.sum() <= top) & (nb + need <= width).all() & (end[-1] <= rows)
    r = torch.arange(rows, device=n.device)
    b = torch.searchsorted(end, r, right=True).clamp(max=batch - 1)
    valid = ok & (r < end[-1])
    i = r - cu[b]
    old = i < room[b]
    after = (i - room[b]).clamp(min=0)
    j, p = torch.div(after, BS, rounding_mode="floor"), after % BS
    pop = (top - 1 - (first[b] + j)).clamp(0, st["free"].numel() - 1)
    fresh = st["free"][pop].long()
    slot = torch.where(old, table.gather(1, at)[:, 0].long()[b], fresh)
    slots = torch.where(valid, slot * BS + torch.where(old, last[b] + i, p), -1).int()
    positions = torch.where(valid, held[b] + i, -1).int()
    cu = torch.where(ok, cu, 0).int()
    # Entries of new blocks, each by its first token's row.
    opens = valid & ~old & (p == 0)
    where = torch.where(opens, b * width + nb[b] + j, batch * width)

    def put(t, value):
        flat = torch.cat([t.reshape(-1), t.new_zeros(1)])
        t.copy_(flat.scatter(0, where, value.int())[:-1].view_as(t))

    taken = torch.minimum(room, n)
    grown = torch.where(ok & open_, last + taken, last).int()
    lengths.scatter_(1, at, torch.where(nb > 0, grown, lengths.gather(1, at)[:, 0])[:, None])
    put(table, fresh)
    put(states, torch.zeros_like(fresh))
    put(lengths, (n[b] - room[b] - j * BS).clamp(0, BS))
    tail = torch.where(need > 0, n - room - (need - 1) * BS, torch.where(open_, last + taken, 0))
    st["open"].copy_(torch.where(ok & (n > 0), ((tail > 0) & (tail < BS)).int(), st["open"]))
    st["nblocks"].copy_(torch.where(ok, nb + need, nb))
    ctl[0] = torch.where(ok, top - need.sum(), top).int()
    ctl[3] = ok.int()
    return slots, positions, cu, torch.where(ok, held + n, held).int()


def _run_write(st):
    if own:
        from paged_tierkv_amd import kernels

        kernels.write_slots(st["k"], st["v"], st["slots"], st["hot_k"], st["hot_v"])
    else:
        keep = st["slots"] >= 0
        slot, row = st["slots"][keep].long() // BS, st["slots"][keep].long() % BS
        st["hot_k"][slot, :, row] = st["k"][keep].float().half()
        st["hot_v"][slot, :, row] = st["v"][keep].float().half()
    return st["hot_k"], st["hot_v"]


def _run_extend(st):
    if own:
        from paged_tierkv_amd.tierkv_hip import tierkv_extend_attention

        return tierkv_extend_attention(
            st["q"], st["cu"], st["table"], st["states"], st["lengths"], st["hot_k"], st["hot_v"], st["warm_k"],
            st["warm_v"], st["k_scale"], st["k_zero"], st["v_scale"], st["v_zero"], st["width"], st["groups"],
            st["scaling"], cold_mode=st["cold"], seq_num_blocks=st["nblocks"], max_tokens=st["max_new"],
            out=st["out"])
    row = 0
    for b, n in enumerate(st["new"]):
        _plain_extend(st, b, row, n)
        row += n
    return st["out"]


def _values(st, slots, states, hot, warm, scale, zero):
    """A request's K or V rows [kv, tokens, d] in 32 bits."""
    h = hot[slots.clamp(0, hot.shape[0] - 1)].float()
    w = slots.clamp(0, warm.shape[0] - 1)
    if zero is None:
        x = warm[w].float() * scale[w][:, :, None, None]
    else:
        x = (warm[w].float() - zero[w].float()) * scale[w].float()
    tier = states[:, None, None, None]
    x = torch.where(tier == HOT, h, torch.where(tier == WARM, x, 0.0))
    return x.transpose(0, 1).reshape(hot.shape[1], -1, hot.shape[3])


def _plain_extend(st, b, row, n):
    blocks, groups = st["held"][b], st["groups"]
    slots, states, lens = st["table"][b, :blocks].long(), st["states"][b, :blocks], st["lengths"][b, :blocks]
    valid = (torch.arange(BS, device=lens.device)[None] < lens[:, None]).reshape(-1)
    ordinal = valid.long().cumsum(0) - 1
    if st["cold"] == "masked":
        valid = valid & (states != COLD).repeat_interleave(BS)
    k = _values(st, slots, states, st["hot_k"], st["warm_k"], st["k_scale"], st["k_zero"])
    v = _values(st, slots, states, st["hot_v"], st["warm_v"], st["v_scale"], st["v_zero"])
    v = torch.where(valid[None, :, None], v, 0.0)
    i = torch.arange(n, device=lens.device)
    seen = valid[None] & (ordinal[None] <= st["tokens"][b] - n + i[:, None])            # [n, tokens]
    seen = seen.repeat_interleave(groups, 0)
    q = st["q"][row:row + n].float()
    for h in range(k.shape[0]):
        qh = q[:, h * groups:(h + 1) * groups].reshape(n * groups, -1)
        x = (qh @ k[h].t()) * st["scaling"]
        x = torch.where(seen, x, float("-inf"))
        m = x.amax(1, keepdim=True)
        m = torch.where(torch.isinf(m), 0.0, m)
        e = torch.exp(x - m)
        total = e.sum(1, keepdim=True)
        o = (e @ v[h]) / torch.where(total > 0, total, 1.0)
        st["out"][row:row + n, h * groups:(h + 1) * groups] = o.view(n, groups, -1).to(st["out"].dtype)


def _run_sample(st):
    if own:
        from paged_tierkv_amd import kernels

        return kernels.sample_tokens(st["x"], st["u"], st["temperature"], st["top_k"], st["top_p"], st["min_p"])
    x, u = st["x"], st["u"].double()
    batch, vocab = x.shape
    as_row = lambda a, dt: (a if torch.is_tensor(a) else torch.full((batch,), a, device=x.device)).to(dt)[:, None]
    # Limits that a program passes as 32-bit numbers are those numbers in 64 bits.
    t, p, m = (as_row(st[key], torch.float32).double() for key in ("temperature", "top_p", "min_p"))
    k = as_row(st["top_k"], torch.int64)
    sorted_x, order = torch.sort(x.float(), dim=1, descending=True, stable=True)
    d = sorted_x.double() - sorted_x[:, :1].double()
    w = torch.round(torch.exp(d / torch.where(t > 0, t, 1.0)) * WEIGHT_ONE).long()     # whole numbers: sums are exact
    rank = torch.arange(vocab, device=x.device)[None]
    w = torch.where((k > 0) & (rank >= k), 0, w)
    before = w.cumsum(1) - w
    total = w.sum(1, keepdim=True)
    w = torch.where((p < 1) & (rank > 0) & (before.double() >= p * total.double()), 0, w)
    w = torch.where(w.double() >= m.clamp(max=1.0) * WEIGHT_ONE, w, 0)
    by_index = torch.zeros_like(w).scatter_(1, order, w)
    run_sum = by_index.cumsum(1)
    target = torch.floor(u * run_sum[:, -1].double()).long()
    token = torch.searchsorted(run_sum, target[:, None], right=True)[:, 0].clamp(max=vocab - 1)
    prob = by_index.gather(1, token[:, None])[:, 0].double() / run_sum[:, -1].double()
    drawn = t[:, 0] > 0
    return torch.where(drawn, token, order[:, 0]), torch.where(drawn, prob, 1.0).float()


# --- work --------------------------------------------------------------------

def _pairs(ctx, n, states, lens):
    """Visible (query, token) pairs of a request and its resident tokens."""
    resident = sum(l for s, l in zip(states, lens) if s != COLD)
    return resident * n - n * (n - 1) // 2, resident


def work(case):
    op = case["op"]
    if op == "slots":
        new = _new_tokens(case)
        rows = sum(new) + 3
        blocks = sum(_ceil(n, BS) for n in new)
        # Lengths of the blocks held, per-request words, table entries of new blocks, slots and positions.
        return {"bytes": case["batch"] * (case["blocks"] * 2 + 12 * 4) + blocks * 16 + rows * 8, "flops": rows * 4}
    if op == "write":
        elements = 2 * case["tokens"] * case["kv_heads"] * case["head_dim"]
        return {"bytes": elements * 4 + case["tokens"] * 4, "flops": 0}
    if op == "sample":
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": case["batch"] * (case["vocab"] * size + 28), "flops": case["batch"] * case["vocab"] * 4}
    kv, d = case["kv_heads"], case["head_dim"]
    warm = d if case["fmt"] == "absmax_i8" else d + 4
    total, pairs = 0, 0
    for ctx, n in zip(_context(case), _new_tokens(case)):
        lens = _blocks_of(ctx, n)
        states = _tiers(ctx, n, 0)
        more, _ = _pairs(ctx, n, states, lens)
        pairs += more
        for s, l in zip(states, lens):
            total += 12 + (0 if s == COLD else 2 * kv * l * (2 * d if s == HOT else warm))
        total += 2 * n * case["heads"] * d * 2
    return {"bytes": int(total), "flops": int(4 * pairs * case["heads"] * d)}


# --- the definitions in 64 bits ----------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    return {"slots": _exact_slots, "write": _exact_write, "extend": _exact_extend, "sample": _exact_sample}[
        case["op"]](st)


def _exact_slots(st):
    """Request by request and block by block, as a host program would do it."""
    start = st["start"].cpu().numpy().copy()
    base = st["work"].data_ptr()
    host = {name: start[(st[name].data_ptr() - base) // 4:][:st[name].numel()].reshape(tuple(st[name].shape))
            for name in ("table", "states", "lengths", "nblocks", "open", "ctl")}
    free, new = st["free"].cpu().numpy(), st["new"].cpu().numpy()
    slots = np.full(st["rows"], -1, np.int32)
    positions = np.full(st["rows"], -1, np.int32)
    cu, context = np.zeros(len(new) + 1, np.int32), np.zeros(len(new), np.int32)
    top, row = int(host["ctl"][0]), 0
    for b, n in enumerate(int(x) for x in new):
        nb = int(host["nblocks"][b])
        held = int(host["lengths"][b, :nb].sum())
        fresh = True
        if host["open"][b] and nb > 0 and host["states"][b, nb - 1] == HOT and host["lengths"][b, nb - 1] < BS:
            fresh = False
        for i in range(n):
            if fresh or host["lengths"][b, nb - 1] == BS:
                top -= 1
                host["table"][b, nb], host["states"][b, nb], host["lengths"][b, nb] = free[top], HOT, 0
                nb, fresh = nb + 1, False
            slots[row] = host["table"][b, nb - 1] * BS + host["lengths"][b, nb - 1]
            positions[row] = held + i
            host["lengths"][b, nb - 1] += 1
            row += 1
        host["nblocks"][b] = nb
        if n:
            host["open"][b] = int(host["lengths"][b, nb - 1] < BS)
        cu[b + 1], context[b] = row, held + n
    host["ctl"][0], host["ctl"][3] = top, 1
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a))
    return dict(slots=t(slots), positions=t(positions), cu=t(cu), context=t(context),
                **{name: t(host[name]) for name in ("table", "states", "lengths", "nblocks", "open", "ctl")})


def _exact_write(st):
    k, v = st["hot_k"].double().cpu(), st["hot_v"].double().cpu()
    slots = st["slots"].cpu().numpy()
    at = np.nonzero(slots >= 0)[0]
    dst = torch.from_numpy(slots[at].astype(np.int64))
    src = torch.from_numpy(at)
    for pool, rows in ((k, st["k"]), (v, st["v"])):
        pool.transpose(1, 2).index_put_((dst // BS, dst % BS), rows.cpu()[src].to(torch.float16).double())
    return k, v


def _exact_extend(st):
    """Each request's visible tokens gathered, one softmax per kv head in 64 bits."""
    out = torch.zeros(st["out"].shape, dtype=torch.float64, device="cuda")
    cu, groups = st["cu"].cpu().tolist(), st["groups"]
    table, states = st["table"].cpu().numpy(), st["states"].cpu().numpy()
    lengths, blocks = st["lengths"].cpu().numpy(), st["nblocks"].cpu().tolist()
    for b in range(len(blocks)):
        token = [(i, t) for i in range(blocks[b]) for t in range(int(lengths[b, i]))]
        order = np.arange(len(token))
        blk = np.array([x[0] for x in token])
        pos = torch.from_numpy(np.array([x[1] for x in token])).cuda()
        tier = states[b, blk]
        keep = np.ones(len(token), bool) if st["cold"] == "zero_logit" else tier != COLD
        order, blk, pos, tier = order[keep], blk[keep], pos[torch.from_numpy(keep).cuda()], tier[keep]
        slot = torch.from_numpy(table[b, blk].astype(np.int64)).cuda()
        kind = torch.from_numpy(tier).cuda()

        def rows(hot, warm, scale, zero, h):
            x = torch.zeros((len(order), hot.shape[3]), dtype=torch.float64, device="cuda")
            a = (kind == HOT).nonzero()[:, 0]
            x[a] = hot[slot[a], h, pos[a]].double()
            a = (kind == WARM).nonzero()[:, 0]
            code = warm[slot[a], h, pos[a]].double()
            if zero is None:
                x[a] = code * scale[slot[a], h].double()[:, None]
            else:
                x[a] = (code - zero[slot[a], h, pos[a]].double()) * scale[slot[a], h, pos[a]].double()
            return x

        n = cu[b + 1] - cu[b]
        limit = len(token) - n + torch.arange(n, device="cuda")
        hidden = torch.from_numpy(order).cuda()[None] > limit[:, None]
        for h in range(st["hot_k"].shape[1]):
            k = rows(st["hot_k"], st["warm_k"], st["k_scale"], st["k_zero"], h)
            v = rows(st["hot_v"], st["warm_v"], st["v_scale"], st["v_zero"], h)
            for g in range(h * groups, (h + 1) * groups):
                x = (st["q"][cu[b]:cu[b + 1], g].double() @ k.t()) * st["scaling"]
                x.masked_fill_(hidden, float("-inf"))
                out[cu[b]:cu[b + 1], g] = torch.nan_to_num(torch.softmax(x, 1)) @ v
    return out


def _exact_sample(st):
    """Row by row with numpy: a stable sort, whole-number weights, running sums."""
    x = st["x"].float().cpu().numpy()
    u = st["u"].cpu().numpy().astype(np.float64)
    get = lambda a, b: (a[b].item() if torch.is_tensor(a) else float(np.float32(a)))
    tokens, probs = [], []
    for b in range(x.shape[0]):
        order = np.argsort(-x[b], kind="stable")
        t = get(st["temperature"], b)
        if not t > 0:
            tokens.append(int(order[0]))
            probs.append(1.0)
            continue
        d = x[b].astype(np.float64) - float(x[b, order[0]])
        w = np.rint(np.exp(d / t) * WEIGHT_ONE).astype(np.int64)
        k = int(get(st["top_k"], b))
        kept = order[:k] if k > 0 else order
        p = get(st["top_p"], b)
        if p < 1:
            sums = np.cumsum(w[kept])
            before = (sums - w[kept]).astype(np.float64)
            kept = kept[:max(1, int(np.searchsorted(before, p * float(sums[-1]), side="left")))]
        kept = kept[w[kept].astype(np.float64) >= min(get(st["min_p"], b), 1.0) * WEIGHT_ONE]
        kept = np.sort(kept)
        sums = np.cumsum(w[kept])
        target = math.floor(u[b] * float(sums[-1]))
        at = int(kept[min(int(np.searchsorted(sums, target, side="right")), len(kept) - 1)])
        tokens.append(at)
        probs.append(float(w[at]) / float(sums[-1]))
    return torch.tensor(tokens, dtype=torch.int64), torch.tensor(probs, dtype=torch.float64)
