"""Seeded random steps of any geometry against the oracle: tables, formats,
head layouts, lengths, tiers and bounds drawn together, the outputs between
guard values."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import serving
from paged_tierkv_amd import kernels

from test_gpu_serving_step import COLD, call, check, gpu, logits, step, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed", range(48))
def test_attention_of_any_geometry(device, seed):
    rng = np.random.default_rng(1000 + seed)
    bs = int(rng.choice([1, 3, 8, 15, 16, 16, 17, 31, 32, 48, 64]))
    d = 8 * int(rng.integers(1, 17))
    kv = int(rng.choice([1, 2, 3, 5, 8]))
    groups = int(rng.choice([1, 2, 3, 4, 7, 8, 33]))
    batch = int(rng.integers(1, 7))
    new = [int(x) for x in rng.choice([0, 1, 2, 5, 9, 31, 32, 33, 70, 200], batch)]
    held = [int(n + rng.choice([0, 0, 1, 15, 16, 100, 900])) for n in new]
    if seed % 5 == 0:
        held = [max(0, h - int(rng.integers(0, 4))) for h in held]        # more rows than tokens
    fmt = ("absmax_i8", "ref_u8")[seed % 2]
    cold = ("masked", "zero_logit")[(seed // 2) % 2]
    dtype = (torch.float16, torch.bfloat16)[(seed // 4) % 2]
    if sum(new) == 0:
        new[0], held[0] = 3, held[0] + 3
    s = step(seed, new, held, kv * groups, kv, d, bs, fmt, dtype, cold=float(rng.random() * 0.5), warm=0.4, pad=2,
             holes=seed % 3 == 0)
    inside = np.arange(s["table"].shape[1])[None] < s["nblocks"][:, None]
    s["states"][inside & (rng.random(inside.shape) < 0.1)] = COLD
    print(f"[sweep] {seed}: bs {bs} d {d} kv {kv} groups {groups} new {new} held {held} {fmt} {cold} {dtype}", flush=True)
    shape, guard = tuple(s["q"].shape), 4096
    flat = torch.full((s["q"].numel() + 2 * guard,), 7.0, dtype=dtype, device=device)
    out = flat[guard:-guard].view(shape)
    got = call(s, device, cold, out=out, max_tokens=int(max(new) + rng.integers(0, 3)))
    check(got, s, cold)
    assert (out[s["cu"][-1]:] == 7.0).all() and (flat[:guard] == 7.0).all() and (flat[-guard:] == 7.0).all()


@pytest.mark.parametrize("seed", range(40))
def test_slot_maps_and_writes_of_any_geometry(device, seed):
    rng = np.random.default_rng(2000 + seed)
    batch = int(rng.choice([1, 2, 5, 63, 64, 65, 200, 1024, 1025, 4096]))
    bs = int(rng.choice([1, 5, 16, 33, 64]))
    width = int(rng.choice([1, 3, 12, 40, 300]))
    if batch * width > 200000:
        width = 12
    state = list(tables(rng, batch, width, bs, batch * (width + 1) + 8))
    most = int(rng.choice([0, 1, 2, 40, 200]))
    new = rng.integers(0, most + 1, batch).astype(np.int32)
    if seed % 4 == 0:
        new[rng.integers(0, batch)] = -1 if seed % 8 == 0 else bs * width + 1
    rows = max(0, int(np.maximum(new, 0).sum()) + int(rng.integers(-1, 4)))
    state[6][0] = min(int(state[6][0]), int(rng.choice([0, batch, 10 ** 9])))
    host, dev = [a.copy() for a in state], [gpu(a, device) for a in state]
    print(f"[sweep] {seed}: batch {batch} bs {bs} width {width} most {most} rows {rows}", flush=True)
    exp = serving.build_slot_map(new, *host, bs, rows)
    m = kernels.build_slot_map(gpu(new, device), *dev, bs, rows)
    for g, e in zip((*m, *dev[:6]), (*exp, *host[:6])):
        np.testing.assert_array_equal(g.cpu().numpy(), e)
    assert dev[6][0].item() == host[6][0] and dev[6][3].item() == host[6][3]
    assert (dev[6][2].item() != 0) == (host[6][2] != 0)
    if rows == 0:
        return
    slots = batch * (width + 1) + 8
    kv, d = int(rng.choice([1, 2, 5])), int(rng.choice([8, 20, 64]))
    if slots * kv * bs * d > 3 * 10 ** 7 or rows * kv * d > 10 ** 7:
        kv, d = 1, 8
    x = torch.randn((2, rows, kv, d), dtype=torch.float16, device=device)
    hot = torch.full((2, slots, kv, bs, d), 7.0, dtype=torch.float16, device=device)
    want = hot.clone()
    keep = m.slots >= 0
    at = m.slots[keep].long()
    for p, t in zip(want, x):
        p[at // bs, :, at % bs] = t[keep]
    kernels.write_slots(x[0], x[1], m.slots, hot[0], hot[1])
    assert torch.equal(hot, want)


@pytest.mark.parametrize("seed", range(40))
def test_token_choice_of_any_rows(device, seed):
    rng = np.random.default_rng(3000 + seed)
    vocab = int(np.exp(rng.uniform(0, np.log(150000))))
    batch = int(rng.integers(1, 9))
    dtype = (torch.float16, torch.bfloat16, torch.float32)[seed % 3]
    kind = ("plain", "peaked", "flat", "ties", "masked")[seed % 5]
    x = logits(rng, batch, vocab, dtype, kind)
    u = rng.random(batch).astype(np.float32)
    t = np.where(rng.random(batch) < 0.1, 0, np.exp(rng.uniform(-6, 4, batch))).astype(np.float32)
    k = np.where(rng.random(batch) < 0.4, 0, np.exp(rng.uniform(0, np.log(vocab + 2), batch))).astype(np.int32)
    p = np.where(rng.random(batch) < 0.3, 1.0, rng.random(batch) ** 0.3).astype(np.float32)
    m = np.where(rng.random(batch) < 0.5, 0.0, rng.random(batch) ** 4).astype(np.float32)
    print(f"[sweep] {seed}: batch {batch} vocab {vocab} {dtype} {kind} k {k.tolist()}", flush=True)
    dev = lambda a: torch.from_numpy(a).to(device)   # noqa: E731
    got, prob = kernels.sample_tokens(x.to(device), dev(u), dev(t), dev(k), dev(p), dev(m))
    exp = [serving.sample_row(x[b].float().numpy(), u[b], t[b], int(k[b]), p[b], m[b]) for b in range(batch)]
    assert got.tolist() == [e[0] for e in exp]
    np.testing.assert_allclose(prob.cpu().numpy(), [e[1] for e in exp], rtol=2.0 ** -23)


@pytest.mark.parametrize("fmt", ["absmax_i8", "ref_u8"])
@pytest.mark.parametrize("scaling", [-0.2, 0.0])
@pytest.mark.parametrize("new,held", [([5, 1], [60, 33]), ([70], [200])])
def test_a_scaling_that_is_not_positive(device, fmt, scaling, new, held):
    for dtype in (torch.float16, torch.bfloat16):
        s = step(71, new, held, 4, 2, 64, fmt=fmt, dtype=dtype)
        s["scaling"] = scaling
        check(call(s, device, "zero_logit"), s, "zero_logit")
