"""Operators of a serving step whose requests share prompts, as measurable
cases: the norms and position rotation of the step's rows on their way into
the cache, rows quantized as they are written and read back, and the attention
of requests that have a long prefix in common.

A case is a dict of plain values; ``prepare`` makes what a serving program
holds before the call from a seed, ``run`` makes one pass (the plain form in
elementary torch operations, or with ``own`` the package's entry points),
``work`` counts the bytes and operations a pass cannot do without, and
``exact`` gives the outputs in 64 bits from the definitions.

Kinds of cases:

* ``rotate``  ``kernels.rotate_rows``: per-head norms (where the model has
              them) and the rotation by position of packed query and key rows;
              keys and values go into their HOT slots, or the keys come back.
* ``store``   ``kernels.quantize_rows`` and ``kernels.read_rows``: packed K/V
              rows quantized into WARM slots, then the requests' last tokens
              read back as rows.
* ``read``    ``kernels.read_rows``: tokens of a cache in all three tiers.
* ``attend``  ``tierkv_hip.tierkv_prefix_attention``: each request sees the
              tokens of its prefix, which others share, then its own.
"""

import math

import numpy as np
import torch

own = False

HOT, WARM, COLD = 0, 1, 2
BS = 16                    # tokens per block, in every configuration of this package
EPS = 1e-6                 # of the norms
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _ceil(a, b):
    return -(-a // b)


# --- cases -------------------------------------------------------------------

def _rotate(name, tokens, heads, kv_heads, head_dim, rot, dtype, norm, pairs, slots, far):
    return dict(name=name, op="rotate", tokens=tokens, heads=heads, kv_heads=kv_heads, head_dim=head_dim, rot=rot,
                dtype=dtype, norm=norm, pairs=pairs, slots=slots, far=far)


def _store(name, batch, ctx, new, pattern, window, kv_heads, head_dim, fmt, dtype):
    return dict(name=name, op="store", batch=batch, ctx=ctx, new=new, pattern=pattern, window=window,
                kv_heads=kv_heads, head_dim=head_dim, fmt=fmt, dtype=dtype)


def _read(name, batch, ctx, window, kv_heads, head_dim, fmt, dtype):
    return dict(name=name, op="read", batch=batch, ctx=ctx, window=window, kv_heads=kv_heads, head_dim=head_dim,
                fmt=fmt, dtype=dtype)


def _attend(name, batch, prefixes, prefix, ctx, new, pattern, heads, kv_heads, head_dim, fmt="absmax_i8", cold="masked",
            dtype="fp16", tiers="mixed", alone=0):
    return dict(name=name, op="attend", batch=batch, prefixes=prefixes, prefix=prefix, ctx=ctx, new=new,
                pattern=pattern, heads=heads, kv_heads=kv_heads, head_dim=head_dim, fmt=fmt, cold=cold, dtype=dtype,
                tiers=tiers, alone=alone)


def listed():
    return [
        # A decode step of 64 requests, 32 / 8 heads of 128, rotated into the cache.
        _rotate("rotate_decode_64", 64, 32, 8, 128, 128, "fp16", False, False, True, 4000),
        # One prefill step's rows with per-head norms, positions of a long context.
        _rotate("rotate_prompts_16384", 16384, 32, 8, 128, 128, "bf16", True, False, True, 120000),
        # A model with half of its dims rotated, in adjacent pairs; the keys come back as rows.
        _rotate("rotate_pairs_1237", 1237, 14, 2, 64, 32, "bf16", True, True, False, 9000),
        # Decoding over a quantized cache: one token each into open blocks, the last block's tokens read back.
        _store("store_decode_96", 96, 700, 1, "ragged", 16, 8, 128, "absmax_i8", "fp16"),
        # A shared prompt of odd length, quantized token by token as it is written, and read back whole.
        _store("store_prompt_8191_ref", 1, 0, 8191, "same", 8191, 8, 128, "ref_u8", "bf16"),
        # The last tokens of many requests of very different lengths, for a program that attends to a window.
        _read("read_windows_24", 24, 1500, 300, 4, 64, "ref_u8", "bf16"),
        # One long context read back whole.
        _read("read_context_32768", 1, 32768, 32768, 8, 128, "absmax_i8", "fp16"),
        # Two requests' next tokens after a short shared prompt.
        _attend("attend_2_prefix_600", 2, 1, 600, 20, 1, "same", 32, 8, 128),
        # A decode step of 64 requests that share a prompt of 8192 tokens.
        _attend("attend_decode_64_prefix_8192", 64, 1, 8192, 250, 1, "ragged", 32, 8, 128),
        # A decode step of 256 requests over four prompts, some of them without one.
        _attend("attend_decode_256_prefix_4x4096", 256, 4, 4096, 180, 1, "ragged", 32, 8, 128, "ref_u8", "masked", "bf16",
                "mixed", 7),
        # Drafted tokens of small-model requests (32 / 4 heads of 64) after a prompt that ends inside a block.
        _attend("attend_verify_24x5_d64", 24, 2, 1501, 90, 5, "ragged", 32, 4, 64, "ref_u8", "zero_logit", "bf16"),
        # Sixteen fresh questions of 512 tokens on one document of 16384.
        _attend("attend_questions_16x512", 16, 1, 16384, 0, 512, "ragged", 32, 8, 128, "absmax_i8", "masked", "fp16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotate", "rotate", "store", "store", "read", "attend", "attend", "attend"])
    kv_heads = rng.choice([1, 2, 4, 8])
    head_dim = rng.choice([64, 128])
    fmt = rng.choice(["absmax_i8", "ref_u8"])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "rotate":
        heads = kv_heads * rng.choice([1, 2, 4, 7, 8])
        head_dim = rng.choice([64, 96, 128])
        rot = head_dim if rng.random() < 0.6 else head_dim // 2
        tokens = _log(rng, 1, 16384 * 48 * 128 // ((heads + 2 * kv_heads) * head_dim))
        case = _rotate("", min(tokens, 40000), heads, kv_heads, head_dim, rot, dtype, rng.random() < 0.5,
                       rng.random() < 0.4, rng.random() < 0.6, _log(rng, 100, 500000))
    elif op == "store":
        batch = _log(rng, 1, 200)
        pattern = rng.choice(["same", "ragged", "one_long"])
        rows = 1 if pattern == "one_long" else batch
        new = _log(rng, 1, max(1, min(8191, 8191 * 1024 // (rows * kv_heads * head_dim))))
        ctx = 0 if rng.random() < 0.3 else _log(rng, 1, max(1, 40000 // batch))
        case = _store("", batch, ctx, new, pattern, _log(rng, 1, min(ctx + new, max(1, 16000 // batch))), kv_heads,
                      head_dim, fmt, dtype)
    elif op == "read":
        batch = _log(rng, 1, 100)
        ctx = _log(rng, 1, max(1, 32768 * 1024 // (batch * kv_heads * head_dim)))
        ctx = min(ctx, 32768)
        case = _read("", batch, ctx, _log(rng, 1, ctx), kv_heads, head_dim, fmt, rng.choice(["fp16", "bf16", "fp32"]))
    else:
        heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
        batch = _log(rng, 2, 256)
        prefixes = min(batch, rng.choice([1, 1, 2, 5]))
        pattern = rng.choice(["same", "ragged", "one_long"])
        rows = 1 if pattern == "one_long" else batch
        new = 1 if rng.random() < 0.5 else _log(rng, 1, max(1, 8192 // rows))
        prefix = _log(rng, 64, 16384)
        ctx = 0 if rng.random() < 0.3 else _log(rng, 1, max(1, 60000 // batch))
        new = min(new, 4096)
        # No dearer than the dearest listed case: 8192 tokens of 32 heads of 128 on 16384.
        while rows * new * (prefix + ctx + new) * heads * head_dim > 3.2e11 and new > 1:
            new = max(1, new // 2)
        case = _attend("", batch, prefixes, prefix, ctx, new, pattern, heads, kv_heads, head_dim, fmt,
                       rng.choice(["masked", "zero_logit"]), dtype, rng.choice(["mixed", "hot"]), rng.choice([0, 0, 3]))
    del case["name"]
    return case


# --- lengths -----------------------------------------------------------------

def _new_tokens(case):
    """New tokens per request."""
    n, batch = case["new"], case["batch"]
    if case["pattern"] == "same" or n == 1:
        return [n] * batch
    if case["pattern"] == "one_long":
        return [n] + [1] * (batch - 1)
    return [max(1, n - (b * 37) % max(1, n // 2)) if b % 5 else n for b in range(batch)]


def _context(case):
    """Tokens of its own that each request holds before the step."""
    ctx, batch = case["ctx"], case["batch"]
    if case.get("pattern") == "same" or ctx < 8:
        return [ctx] * batch
    return [ctx - (b * 131) % (ctx // 2 + 1) for b in range(batch)]


def _fill(tokens):
    """Valid tokens of the blocks that hold this many."""
    return [BS] * (tokens // BS) + ([tokens % BS] if tokens % BS else [])


def _mixed(blocks, rng):
    """Tiers of a context's blocks: the first and the last 4 HOT, of the others
    10 % HOT, 60 % WARM and the rest COLD."""
    states = np.full(blocks, HOT, np.int32)
    if blocks > 5:
        r = rng.random(blocks - 5)
        states[1:blocks - 4] = np.where(r < 0.1, HOT, np.where(r < 0.7, WARM, COLD))
    return states


def _prefix_lengths(case):
    return [max(1, case["prefix"] - 45 * g) for g in range(case["prefixes"])]


def _prefix_of(case):
    """Each request's prefix, -1 where it has none."""
    alone = case["alone"]
    return [-1 if alone and b % alone == alone - 1 else (b * 7 + b // 5) % case["prefixes"] for b in range(case["batch"])]


# --- inputs ------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 6151 + 29)
    return {"rotate": _prepare_rotate, "store": _prepare_store, "read": _prepare_read, "attend": _prepare_attend}[
        case["op"]](case, np.random.default_rng(int(seed)), gen)


def _cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _prepare_rotate(case, rng, gen):
    n, heads, kv, d = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
    dt = DTYPES[case["dtype"]]
    rows = n + 3                                  # a padded step: three rows of no request
    x = (_randn(gen, rows, (heads + 2 * kv) * d) * 1.5).to(dt)
    q = x[:, :heads * d].view(rows, heads, d)
    k = x[:, heads * d:(heads + kv) * d].view(rows, kv, d)
    v = x[:, (heads + kv) * d:].view(rows, kv, d)
    # Requests of any length, each at its own place in its context.
    positions = np.full(rows, -1, np.int32)
    at = 0
    while at < n:
        take = min(n - at, int(rng.integers(1, max(2, n // 4))))
        positions[at:at + take] = int(rng.integers(0, case["far"])) + np.arange(take)
        at += take
    f = 500000.0 ** (-np.arange(0, case["rot"], 2, dtype=np.float64) / case["rot"])
    st = dict(op="rotate", q=q, k=k, v=v, positions=_cuda(positions), inv_freq=_cuda(f.astype(np.float32)),
              pairs=case["pairs"], q_out=torch.zeros((rows, heads, d), dtype=dt, device="cuda"), q_weight=None,
              k_weight=None, k_out=None)
    if case["norm"]:
        st["q_weight"] = (1 + 0.3 * _randn(gen, d)).to(dt)
        st["k_weight"] = (1 + 0.3 * _randn(gen, d)).to(dt)
    if case["slots"]:
        blocks = _ceil(n, BS) + 16
        order = rng.permutation(blocks)[:_ceil(n, BS)]
        slots = np.full(rows, -1, np.int32)
        slots[:n] = (order[:, None] * BS + np.arange(BS)[None]).ravel()[:n]
        pool = _randn(gen, 2, blocks, kv, BS, d).to(torch.float16)
        st.update(slots=_cuda(slots), hot_k=pool[0], hot_v=pool[1])
    else:
        st.update(v=None, slots=None, hot_k=None, hot_v=None, k_out=torch.zeros((rows, kv, d), dtype=dt, device="cuda"))
    return st


def _quantize(x, fmt, filled=None):
    """WARM codes and metadata of tiles [slots, kv, bs, d], of which the first
    ``filled`` [slots] tokens count, in the shapes of the package's pools."""
    xf = x.float()
    if filled is not None:
        xf = xf * (torch.arange(xf.shape[2], device=xf.device)[None] < filled[:, None])[:, None, :, None]
    if fmt == "absmax_i8":
        s = xf.abs().amax(dim=(2, 3)) / 127.0
        q = torch.round(xf / torch.where(s > 0, s, 1.0)[:, :, None, None]).clamp(-127, 127)
        return q.to(torch.int8), s, None
    return _row_codes(xf)


def _row_codes(xf):
    """The reference's codec over the last dim: every operation's result is
    rounded to 16 bits."""
    r = lambda t: t.half().float()
    lo, hi = xf.amin(-1, keepdim=True), xf.amax(-1, keepdim=True)
    s = r(r(hi - lo) / 255.0)
    s = torch.where(s == 0, 1.0, s)
    z = r(-torch.round(r(lo / s)))
    q = r(torch.round(r(xf / s)) + z).clamp(0, 255)
    return q.to(torch.uint8), s.half(), z.half()


def _prepare_store(case, rng, gen):
    batch, kv, d, fmt = case["batch"], case["kv_heads"], case["head_dim"], case["fmt"]
    new, ctx = _new_tokens(case), _context(case)
    total = [c + n for c, n in zip(ctx, new)]
    width = max(_ceil(t, BS) for t in total)
    used = sum(_ceil(t, BS) for t in total)
    slot = rng.permutation(used + 4).astype(np.int32)
    table = np.full((batch, width), -1, np.int32)
    states = np.full((batch, width), COLD, np.int32)
    lengths = np.zeros((batch, width), np.int32)
    held = np.zeros(used + 4, np.int32)           # tokens in each slot before the step
    slots, at = [], 0
    for b in range(batch):
        nb = _ceil(total[b], BS)
        table[b, :nb] = slot[at:at + nb]
        states[b, :nb] = WARM
        lengths[b, :nb] = _fill(total[b])
        before = _fill(ctx[b])
        held[table[b, :len(before)]] = before
        pos = ctx[b] + np.arange(new[b])
        slots.append(table[b, pos // BS] * BS + pos % BS)
        at += nb
    filled = _cuda(held)
    (wk, ks, kz), (wv, vs, vz) = (_quantize(_randn(gen, used + 4, kv, BS, d).half(), fmt, filled) for _ in range(2))
    rows = sum(new)
    scale = torch.exp(0.4 * _randn(gen, 2, rows, 1, 1))           # tokens of different size
    k, v = ((scale[i] * _randn(gen, rows, kv, d)).to(DTYPES[case["dtype"]]) for i in range(2))
    start = np.array([max(0, t - case["window"]) for t in total], np.int32)
    cu = np.concatenate([[0], np.cumsum(np.array(total) - start)]).astype(np.int32)
    return dict(op="store", k=k, v=v, slots=_cuda(np.concatenate(slots).astype(np.int32)), fmt=fmt, warm_k=wk, warm_v=wv,
                k_scale=ks, k_zero=kz, v_scale=vs, v_zero=vz, table=_cuda(table), states=_cuda(states),
                lengths=_cuda(lengths), nblocks=_cuda(np.array([_ceil(t, BS) for t in total], np.int32)),
                hot_k=torch.zeros((1, kv, BS, d), dtype=torch.float16, device="cuda"),
                hot_v=torch.zeros((1, kv, BS, d), dtype=torch.float16, device="cuda"), start=_cuda(start), cu=_cuda(cu),
                rows=int(cu[-1]), begins=start.tolist(), counts=np.diff(cu).tolist(),
                held=[_ceil(t, BS) for t in total], dtype=torch.float16)


def _tiered(tables, kv, d, fmt, rng, gen):
    """Slots and pools for tables given as (states, lengths) rows: returns the
    device tables, one group per list of rows, and the pools."""
    groups = []
    pools = {}
    host = []
    for rows in tables:
        width = max(max((len(s) for s, _ in rows), default=1), 1)
        states = np.full((len(rows), width), COLD, np.int32)
        lengths = np.zeros((len(rows), width), np.int32)
        inside = np.zeros((len(rows), width), bool)
        for b, (s, ln) in enumerate(rows):
            states[b, :len(s)], lengths[b, :len(s)], inside[b, :len(s)] = s, ln, True
        host.append((np.full((len(rows), width), -1, np.int32), states, lengths, inside))
    for tier, name in ((HOT, "hot"), (WARM, "warm")):
        places = [np.nonzero(inside & (states == tier)) for _, states, _, inside in host]
        count = max(1, sum(len(p[0]) for p in places))
        order, at = rng.permutation(count).astype(np.int32), 0
        for (table, _, _, _), p in zip(host, places):
            table[p] = order[at:at + len(p[0])]
            at += len(p[0])
        pools[name] = _randn(gen, 2, count, kv, BS, d).to(torch.float16)
    pools["hot"][0][:, :, :1, :4] *= 3                            # some tokens draw attention
    (wk, ks, kz), (wv, vs, vz) = (_quantize(pools["warm"][i], fmt) for i in (0, 1))
    for (table, states, lengths, _), rows in zip(host, tables):
        groups.append(dict(table=_cuda(table), states=_cuda(states), lengths=_cuda(lengths),
                           nblocks=_cuda(np.array([len(s) for s, _ in rows], np.int32)), held=[len(s) for s, _ in rows]))
    return groups, dict(hot_k=pools["hot"][0], hot_v=pools["hot"][1], warm_k=wk, warm_v=wv, k_scale=ks, k_zero=kz,
                        v_scale=vs, v_zero=vz)


def _read_rows_of(case, rng=None):
    """(states, lengths) of a read case's requests: a prompt, whose last block
    may be partly filled, and the tokens after it."""
    out = []
    for c in _context(case):
        prompt = max(1, (c * 5) // 8)
        ln = _fill(prompt) + _fill(c - prompt)
        out.append((None if rng is None else _mixed(len(ln), rng), ln))
    return out


def _prepare_read(case, rng, gen):
    rows = _read_rows_of(case, rng)
    (g,), pools = _tiered([rows], case["kv_heads"], case["head_dim"], case["fmt"], rng, gen)
    total = np.array([sum(ln) for _, ln in rows])
    start = np.maximum(0, total - case["window"]).astype(np.int32)
    cu = np.concatenate([[0], np.cumsum(total - start)]).astype(np.int32)
    return dict(op="read", start=_cuda(start), cu=_cuda(cu), rows=int(cu[-1]), begins=start.tolist(),
                counts=np.diff(cu).tolist(), dtype=DTYPES[case["dtype"]], **g, **pools)


def _attend_rows_of(case, rng):
    """(states, lengths) of the prefixes and of the requests' own tokens."""
    prefixes = []
    for p in _prefix_lengths(case):
        ln = _fill(p)
        states = _mixed(len(ln), rng)
        if case["tiers"] == "hot":
            states[:] = HOT
        prefixes.append((states, ln))
    mine = []
    for c, n in zip(_context(case), _new_tokens(case)):
        old, ln = _fill(c), _fill(c + n)
        states = np.full(len(ln), HOT, np.int32)
        if len(old) > 5:
            states[:len(old)] = _mixed(len(old), rng)
        mine.append((states, ln))
    return prefixes, mine


def _prepare_attend(case, rng, gen):
    kv, d, heads = case["kv_heads"], case["head_dim"], case["heads"]
    new = _new_tokens(case)
    prefixes, mine = _attend_rows_of(case, rng)
    (shared, g), pools = _tiered([prefixes, mine], kv, d, case["fmt"], rng, gen)
    rows = sum(new) + 2                           # two rows of no request
    q = _randn(gen, rows, heads, d).to(DTYPES[case["dtype"]])
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    member = _prefix_of(case)
    return dict(op="attend", q=q, cu=_cuda(cu), shared=shared, member=_cuda(np.array(member, np.int32)),
                members=member, groups=heads // kv, scaling=d ** -0.5, cold=case["cold"], new=new, max_new=max(new),
                out=torch.zeros_like(q), tokens=[sum(ln) for _, ln in mine], **g, **pools)


# --- one pass ----------------------------------------------------------------

def run(state):
    return {"rotate": _run_rotate, "store": _run_store, "read": _run_read, "attend": _run_attend}[state["op"]](state)


def _run_rotate(st):
    if own:
        from paged_tierkv_amd import kernels

        kernels.rotate_rows(st["q"], st["k"], st["positions"], st["inv_freq"], q_weight=st["q_weight"],
                            k_weight=st["k_weight"], eps=EPS, interleaved=st["pairs"], value=st["v"], slots=st["slots"],
                            hot_k=st["hot_k"], hot_v=st["hot_v"], q_out=st["q_out"], k_out=st["k_out"])
        return (st["q_out"], st["k_out"]) if st["slots"] is None else (st["q_out"], st["hot_k"], st["hot_v"])
    pos = st["positions"]
    keep = pos >= 0
    angle = pos.double()[:, None, None] * st["inv_freq"].double()
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    half = cos.shape[-1]

    def turned(x, weight):
        x = x.float()
        if weight is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
        if st["pairs"]:
            a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
            y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = x[..., :half], x[..., half:2 * half]
            y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([y, x[..., 2 * half:]], -1)

    mask = keep[:, None, None]
    st["q_out"].copy_(torch.where(mask, turned(st["q"], st["q_weight"]).to(st["q_out"].dtype), st["q_out"]))
    k = turned(st["k"], st["k_weight"])
    if st["slots"] is None:
        st["k_out"].copy_(torch.where(mask, k.to(st["k_out"].dtype), st["k_out"]))
        return st["q_out"], st["k_out"]
    put = keep & (st["slots"] >= 0)
    slot, row = st["slots"][put].long() // BS, st["slots"][put].long() % BS
    st["hot_k"][slot, :, row] = k[put].half()
    st["hot_v"][slot, :, row] = st["v"][put].float().half()
    return st["q_out"], st["hot_k"], st["hot_v"]


def _run_store(st):
    meta = [st[x] for x in ("k_scale", "k_zero", "v_scale", "v_zero")]
    if own:
        from paged_tierkv_amd import kernels

        kernels.quantize_rows(st["k"], st["v"], st["slots"], st["warm_k"], st["warm_v"], *meta, warm_format=st["fmt"])
    else:
        _plain_write(st, st["k"], st["warm_k"], st["k_scale"], st["k_zero"])
        _plain_write(st, st["v"], st["warm_v"], st["v_scale"], st["v_zero"])
    return (*_run_read(st), *(t for t in meta if t is not None))


def _plain_write(st, rows, codes, scale, zero):
    at = st["slots"].long()
    slot, pos = at // BS, at % BS
    x = rows.half().float()
    if zero is not None:
        q, s, z = _row_codes(x)
        codes[slot, :, pos] = q
        scale[slot, :, pos] = s
        zero[slot, :, pos] = z
        return
    # The blocks' largest magnitudes and first new rows, then every code of
    # these blocks by its value.
    count, kv, _, d = codes.shape
    peak = x.abs().amax(2)
    top = torch.zeros((count, kv), device=x.device).scatter_reduce_(0, slot[:, None].expand(-1, kv), peak, "amax")
    first = torch.full((count,), BS, device=x.device).scatter_reduce_(0, slot, pos, "amin")
    fresh = first == 0
    s = torch.maximum(torch.where(fresh[:, None], 0.0, scale), top / 127.0)
    value = codes.float() * scale[:, :, None, None]
    held = (torch.arange(BS, device=x.device)[None] < first[:, None]) & (first < BS)[:, None]
    div = torch.where(s > 0, s, 1.0)
    again = torch.round(value / div[:, :, None, None]).clamp(-127, 127).to(torch.int8)
    codes.copy_(torch.where(held[:, None, :, None], again, codes))
    codes[slot, :, pos] = torch.round(x / div[slot][:, :, None]).clamp(-127, 127).to(torch.int8)
    scale.copy_(torch.where((first < BS)[:, None], s, scale))


def _run_read(st):
    if own:
        from paged_tierkv_amd import kernels

        return kernels.read_rows(st["start"], st["cu"], st["rows"], st["table"], st["states"], st["lengths"],
                                 st["nblocks"], st["hot_k"], st["hot_v"], st["warm_k"], st["warm_v"], st["k_scale"],
                                 st["k_zero"], st["v_scale"], st["v_zero"], dtype=st["dtype"])
    k, v = [], []
    for b, (begin, n) in enumerate(zip(st["begins"], st["counts"])):
        slots, states, valid = _row_of(st, b)
        for out, hot, warm, s, z in ((k, "hot_k", "warm_k", "k_scale", "k_zero"), (v, "hot_v", "warm_v", "v_scale", "v_zero")):
            x = _values(slots, states, st[hot], st[warm], st[s], st[z])
            out.append(x[:, valid][:, begin:begin + n].transpose(0, 1).to(st["dtype"]))
    return torch.cat(k), torch.cat(v)


def _row_of(tables, b):
    """Slots, states and, token by token, which places of a table's row hold one."""
    nb = tables["held"][b]
    lens = tables["lengths"][b, :nb]
    valid = (torch.arange(BS, device=lens.device)[None] < lens[:, None]).reshape(-1)
    return tables["table"][b, :nb].long(), tables["states"][b, :nb], valid


def _values(slots, states, hot, warm, scale, zero):
    """K or V of a table's row [kv, places, d] in 32 bits, 0 where evicted."""
    h = hot[slots.clamp(0, hot.shape[0] - 1)].float()
    w = slots.clamp(0, warm.shape[0] - 1)
    if zero is None:
        x = warm[w].float() * scale[w][:, :, None, None]
    else:
        x = (warm[w].float() - zero[w].float()) * scale[w].float()
    tier = states[:, None, None, None]
    x = torch.where(tier == HOT, h, torch.where(tier == WARM, x, 0.0))
    return x.transpose(0, 1).reshape(hot.shape[1], -1, hot.shape[3])


def _run_attend(st):
    if own:
        from paged_tierkv_amd.tierkv_hip import tierkv_prefix_attention

        shared = st["shared"]
        return tierkv_prefix_attention(
            st["q"], st["cu"], st["table"], st["states"], st["lengths"], st["hot_k"], st["hot_v"], st["warm_k"],
            st["warm_v"], st["k_scale"], st["k_zero"], st["v_scale"], st["v_zero"], st["table"].shape[1], st["groups"],
            st["scaling"], st["member"], shared["table"], shared["states"], shared["lengths"],
            prefix_num_blocks=shared["nblocks"], cold_mode=st["cold"], seq_num_blocks=st["nblocks"],
            max_tokens=st["max_new"], out=st["out"])
    shared = {}
    for g in set(st["members"]):
        if g >= 0:
            shared[g] = _plain_tokens(st, st["shared"], g)
    row = 0
    for b, n in enumerate(st["new"]):
        _plain_attend(st, b, row, n, shared.get(st["members"][b]))
        row += n
    return st["out"]


def _plain_tokens(st, tables, b):
    """K, V [kv, tokens, d] that enter the softmax and their ordinals."""
    slots, states, valid = _row_of(tables, b)
    ordinal = valid.long().cumsum(0) - 1
    if st["cold"] == "masked":
        valid = valid & (states != COLD).repeat_interleave(BS)
    k = _values(slots, states, st["hot_k"], st["warm_k"], st["k_scale"], st["k_zero"])
    v = _values(slots, states, st["hot_v"], st["warm_v"], st["v_scale"], st["v_zero"])
    return k[:, valid], v[:, valid], ordinal[valid]


def _plain_attend(st, b, row, n, shared):
    groups = st["groups"]
    k, v, ordinal = _plain_tokens(st, st, b)
    i = torch.arange(n, device=k.device)
    seen = ordinal[None] <= st["tokens"][b] - n + i[:, None]      # [n, own tokens]
    if shared is not None:
        k, v = torch.cat([shared[0], k], 1), torch.cat([shared[1], v], 1)
        seen = torch.cat([seen.new_ones((n, shared[0].shape[1])), seen], 1)
    seen = seen.repeat_interleave(groups, 0)
    q = st["q"][row:row + n].float().view(n, k.shape[0], groups, -1)
    for h in range(k.shape[0]):
        x = (q[:, h].reshape(n * groups, -1) @ k[h].t()) * st["scaling"]
        x = torch.where(seen, x, float("-inf"))
        m = x.amax(1, keepdim=True)
        e = torch.exp(x - torch.where(torch.isinf(m), 0.0, m))
        total = e.sum(1, keepdim=True)
        o = (e @ v[h]) / torch.where(total > 0, total, 1.0)
        st["out"][row:row + n, h * groups:(h + 1) * groups] = o.view(n, groups, -1).to(st["out"].dtype)


# --- work --------------------------------------------------------------------

def _block_bytes(case, states, lengths):
    """K/V bytes and table words of resident blocks."""
    kv, d = case["kv_heads"], case["head_dim"]
    warm = d if case["fmt"] == "absmax_i8" else d + 4
    total = 0
    for s, n in zip(states, lengths):
        total += 12 + (0 if s == COLD else 2 * kv * n * (2 * d if s == HOT else warm))
    return total


def work(case):
    op, kv, d = case["op"], case["kv_heads"], case["head_dim"]
    if op == "rotate":
        n, heads = case["tokens"], case["heads"]
        read = (heads + kv + (kv if case["slots"] else 0)) * d * 2
        turned = n * (heads + kv) * (3 * case["rot"] + (4 * d if case["norm"] else 0))
        return {"bytes": n * (2 * read + 8), "flops": turned}
    if op == "store":
        new, ctx = _new_tokens(case), _context(case)
        total = 0
        code = 1 if case["fmt"] == "absmax_i8" else (d + 4) / d
        for c, n in zip(ctx, new):
            again = c % BS if case["fmt"] == "absmax_i8" else 0   # tokens of the open block whose codes may change
            back = min(c + n, case["window"])
            total += 2 * kv * d * (n * (2 + code) + again * 2 + back * (code + 2)) + n * 4
        return {"bytes": int(total), "flops": 2 * kv * d * 4 * sum(new)}
    rng = np.random.default_rng(0)
    if op == "read":
        size = 4 if case["dtype"] == "fp32" else 2
        total = 0
        for states, lengths in _read_rows_of(case, rng):
            tokens = sum(lengths)
            back = min(tokens, case["window"])
            share = back / tokens
            total += _block_bytes(case, states, lengths) * share + back * 2 * kv * d * size
        return {"bytes": int(total), "flops": 2 * kv * d * sum(min(c, case["window"]) for c in _context(case))}
    prefixes, mine = _attend_rows_of(case, rng)
    member, new = _prefix_of(case), _new_tokens(case)
    resident = [sum(n for s, n in zip(*p) if s != COLD) for p in prefixes]
    total = sum(_block_bytes(case, *p) for g, p in enumerate(prefixes) if g in member)
    pairs = 0
    for g, n, (states, lengths) in zip(member, new, mine):
        total += _block_bytes(case, states, lengths) + 2 * n * case["heads"] * d * 2
        pairs += sum(x for s, x in zip(states, lengths) if s != COLD) * n - n * (n - 1) // 2
        pairs += resident[g] * n if g >= 0 else 0
    return {"bytes": int(total), "flops": int(4 * pairs * case["heads"] * d)}


# --- the definitions in 64 bits ----------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    return {"rotate": _exact_rotate, "store": _exact_store, "read": _exact_read, "attend": _exact_attend}[case["op"]](st)


def _exact_rotate(st):
    """By complex numbers: a pair of dims times e^(i position frequency)."""
    pos = st["positions"].cpu()
    live = (pos >= 0).nonzero()[:, 0]
    turn = torch.polar(torch.ones(1, dtype=torch.float64), pos[live].double()[:, None] * st["inv_freq"].cpu().double()[None])
    half = turn.shape[1]
    order = torch.arange(2 * half)
    if not st["pairs"]:
        order = order.view(2, half).t().reshape(-1)                # pair i is (i, i + half)

    def turned(x, w):
        x = x[live.cuda()].double().cpu()
        if w is not None:
            x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS) * w.double().cpu()
        z = torch.view_as_complex(x[..., order].view(*x.shape[:2], half, 2).contiguous()) * turn[:, None]
        y = x.clone()
        y[..., order] = torch.view_as_real(z).flatten(-2)
        return y

    q = torch.zeros(st["q_out"].shape, dtype=torch.float64)
    q[live] = turned(st["q"], st["q_weight"])
    k = turned(st["k"], st["k_weight"])
    if st["slots"] is None:
        out = torch.zeros(st["k_out"].shape, dtype=torch.float64)
        out[live] = k
        return q, out
    at = st["slots"].cpu()[live].long()
    hk, hv = (st[name].double().cpu().transpose(1, 2).reshape(-1, *k.shape[1:]) for name in ("hot_k", "hot_v"))
    hk[at], hv[at] = k, st["v"][live.cuda()].double().cpu()
    back = lambda x: x.view(-1, BS, *k.shape[1:]).transpose(1, 2)
    return q, back(hk), back(hv)


def _exact_store(st):
    """Block by block on the host."""
    slots = st["slots"].cpu().numpy()
    for rows, name in ((st["k"], "k"), (st["v"], "v")):
        x = rows.cpu().to(torch.float16).numpy()
        codes = st["warm_" + name].cpu().numpy()
        scale = st[name + "_scale"].cpu().numpy()
        zero = st[name + "_zero"]
        if zero is not None:
            zero = zero.cpu().numpy()
            h = np.float16
            lo, hi = x.min(-1).astype(np.float64), x.max(-1).astype(np.float64)
            s = ((hi - lo).astype(h).astype(np.float64) / 255.0).astype(h)
            s[s == 0] = 1
            sd = s.astype(np.float64)
            z = (-np.rint((lo / sd).astype(h).astype(np.float64))).astype(h)
            r = np.rint((x.astype(np.float64) / sd[..., None]).astype(h).astype(np.float64))
            q = np.clip((r + z.astype(np.float64)[..., None]).astype(h), 0, 255).astype(np.uint8)
            codes[slots // BS, :, slots % BS], scale[slots // BS, :, slots % BS, 0] = q, s
            zero[slots // BS, :, slots % BS, 0] = z
            st[name + "_zero"] = torch.from_numpy(zero).cuda()
        else:
            for slot in np.unique(slots // BS):
                mine = np.nonzero(slots // BS == slot)[0]
                pos = slots[mine] % BS
                first = int(pos.min())
                new = x[mine].astype(np.float64)                   # [rows, kv, d]
                old = scale[slot].astype(np.float64) if first else np.zeros(scale.shape[1])
                s = np.maximum(old, (np.abs(new).max((0, 2)) / 127.0).astype(np.float32).astype(np.float64))
                div = np.where(s > 0, s, 1.0)
                value = codes[slot, :, :first].astype(np.float64) * old[:, None, None]
                codes[slot, :, :first] = np.clip(np.rint(value / div[:, None, None]), -127, 127)
                codes[slot][:, pos] = np.clip(np.rint(new / div[None, :, None]), -127, 127).transpose(1, 0, 2)
                scale[slot] = s
        st["warm_" + name], st[name + "_scale"] = torch.from_numpy(codes).cuda(), torch.from_numpy(scale).cuda()
    meta = [st[x] for x in ("k_scale", "k_zero", "v_scale", "v_zero")]
    return (*_exact_read(st), *(t.double() for t in meta if t is not None))


def _token_list(tables, b):
    """Block, place and tier of each of a row's tokens, in order."""
    lens = tables["lengths"][b].cpu().numpy()[:tables["held"][b]]
    blk = np.repeat(np.arange(len(lens)), lens)
    pos = np.concatenate([np.arange(n) for n in lens]) if len(lens) else np.zeros(0, np.int64)
    slot = tables["table"][b].cpu().numpy()[blk].astype(np.int64)
    return slot, pos.astype(np.int64), tables["states"][b].cpu().numpy()[blk]


def _token_values(st, name, slot, pos, tier):
    """[tokens, kv, d] in 64 bits."""
    hot, warm, scale, zero = (st[x] for x in ("hot_" + name, "warm_" + name, name + "_scale", name + "_zero"))
    x = torch.zeros((len(slot), *hot.shape[1::2]), dtype=torch.float64, device="cuda")
    a = _cuda(np.nonzero(tier == HOT)[0])
    s, p = _cuda(slot), _cuda(pos)
    x[a] = hot[s[a], :, p[a]].double()
    a = _cuda(np.nonzero(tier == WARM)[0])
    code = warm[s[a], :, p[a]].double()
    if zero is None:
        x[a] = code * scale[s[a]].double()[:, :, None]
    else:
        x[a] = (code - zero[s[a], :, p[a]].double()) * scale[s[a], :, p[a]].double()
    return x


def _exact_read(st):
    out = ([], [])
    for b, (begin, n) in enumerate(zip(st["begins"], st["counts"])):
        which = [a[begin:begin + n] for a in _token_list(st, b)]
        for rows, name in zip(out, ("k", "v")):
            rows.append(_token_values(st, name, *which))
    return tuple(torch.cat(rows) for rows in out)


def _exact_attend(st):
    """A softmax per request and head over the tokens it sees, listed one by one."""
    out = torch.zeros(st["out"].shape, dtype=torch.float64, device="cuda")
    cu = st["cu"].cpu().tolist()
    masked = st["cold"] == "masked"
    kept = {}

    def tokens(tables, b):
        slot, pos, tier = _token_list(tables, b)
        order = np.arange(len(slot))
        if masked:
            slot, pos, tier, order = (a[tier != COLD] for a in (slot, pos, tier, order))
        return _token_values(st, "k", slot, pos, tier), _token_values(st, "v", slot, pos, tier), order

    for b, g in enumerate(st["members"]):
        n = cu[b + 1] - cu[b]
        k, v, order = tokens(st, b)
        limit = st["tokens"][b] - n + np.arange(n)
        hidden = order[None] > limit[:, None]
        if g >= 0:
            if g not in kept:
                kept[g] = tokens(st["shared"], g)
            k, v = torch.cat([kept[g][0], k]), torch.cat([kept[g][1], v])
            hidden = np.concatenate([np.zeros((n, len(kept[g][2])), bool), hidden], 1)
        hidden = _cuda(hidden)
        for h in range(st["q"].shape[1]):
            x = (st["q"][cu[b]:cu[b + 1], h].double() @ k[:, h // st["groups"]].t()) * st["scaling"]
            out[cu[b]:cu[b + 1], h] = torch.nan_to_num(torch.softmax(x.masked_fill_(hidden, -math.inf), 1)) @ v[:, h // st["groups"]]
    return out
