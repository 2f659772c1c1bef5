"""The operators of a step whose requests share a prompt, run together as a
serving program would: the prompt's rows rotated and quantized as they are
written, the requests' rows rotated into HOT slots, attention over both, the
prompt read back; and the batched runtime's calls of them."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import shared_prompt
from paged_tierkv_amd import kernels
from paged_tierkv_amd.runtime import BatchedTieredKVRuntime
from paged_tierkv_amd.tierkv_hip import tierkv_prefix_attention, workspace_error_word

pytestmark = pytest.mark.gpu
HOT, WARM, COLD = 0, 1, 2
BS, H, KV, D = 16, 8, 2, 64
EPS = 1e-5


def frequencies(device):
    return torch.from_numpy((10000.0 ** (-np.arange(0, D, 2) / D)).astype(np.float32)).to(device)


def turned(rows, positions, f, weight):
    """Normed and rotated rows in float64."""
    y, _ = shared_prompt.rotate(rows.float().cpu().numpy(), positions, f.cpu().numpy(), weight.float().cpu().numpy(), EPS)
    return torch.from_numpy(y)


@pytest.mark.parametrize("fmt", ["absmax_i8", "ref_u8"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_prompt_for_all_then_two_steps(device, fmt, dtype):
    g = torch.Generator().manual_seed(3)
    f = frequencies(device)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)   # noqa: E731
    wq, wk = (1 + 0.2 * torch.randn(2, D, generator=g)).to(dtype).to(device)
    prompt, batch = 145, 3
    pblocks = -(-prompt // BS)
    qkv = torch.randn((prompt, (H + 2 * KV) * D), generator=g).to(dtype).to(device)
    cut = lambda t, a, n: t[:, a * D:(a + n) * D].view(t.shape[0], n, D)   # noqa: E731
    # The prompt, in two pieces that meet inside a block, into WARM slots of its own.
    i8 = fmt == "absmax_i8"
    codes = [torch.zeros((pblocks + 1, KV, BS, D), dtype=torch.int8 if i8 else torch.uint8, device=device) for _ in range(2)]
    scale = [torch.zeros((pblocks + 1, KV), device=device) if i8 else
             torch.ones((pblocks + 1, KV, BS, 1), dtype=torch.float16, device=device) for _ in range(2)]
    zero = [None if i8 else torch.zeros((pblocks + 1, KV, BS, 1), dtype=torch.float16, device=device) for _ in range(2)]
    warm = (codes[0], codes[1], scale[0], zero[0], scale[1], zero[1])
    order = torch.randperm(pblocks + 1, generator=g)[:pblocks].int().to(device)
    at = torch.arange(prompt, device=device)
    slots = (order[at // BS] * BS + at % BS).int()
    for a, b in ((0, 101), (101, prompt)):
        _, k = kernels.rotate_rows(cut(qkv[a:b], 0, H), cut(qkv[a:b], H, KV), at[a:b].int(), f, q_weight=wq, k_weight=wk, eps=EPS)
        kernels.quantize_rows(k, cut(qkv[a:b], H + KV, KV), slots[a:b], *warm, warm_format=fmt)
    # What the cache holds of it, by the codes.
    pk, pv = kernels.read_rows(i32(0), i32(0, prompt), prompt, order[None], torch.full_like(order[None], WARM),
                               torch.tensor([[BS] * (pblocks - 1) + [prompt - BS * (pblocks - 1)]], dtype=torch.int32, device=device),
                               None, torch.zeros((1, KV, BS, D), dtype=torch.float16, device=device),
                               torch.zeros((1, KV, BS, D), dtype=torch.float16, device=device), *warm, dtype=torch.float32)
    want = turned(cut(qkv, H, KV), np.arange(prompt), f, wk)
    # Within a step of each scale (absmax blocks may have grown once: one and a half).
    size = want.abs().max()
    step = (size / 127 if i8 else 2 * size / 255) * 1.5 + size * torch.finfo(dtype).eps
    assert (pk.double().cpu() - want).abs().max() <= step
    # Two steps of requests that share it, one of them alone; the second is one token each.
    width = 6
    tables = [torch.full((batch, width), x, dtype=torch.int32, device=device) for x in (-1, COLD, 0)]
    nb, opened, free = torch.zeros(batch, dtype=torch.int32, device=device), i32(0, 0, 0), torch.arange(20, dtype=torch.int32, device=device)
    ctl = i32(20, 0, 0, 0)
    hot = torch.zeros((2, 20, KV, BS, D), dtype=torch.float16, device=device)
    member = i32(0, -1, 0)
    own_k, own_v = ([torch.zeros((0, KV, D), dtype=torch.float64) for _ in range(batch)] for _ in range(2))
    held = [0] * batch
    for new in ([20, 7, 33], [1, 1, 1]):
        n = sum(new)
        x = torch.randn((n + 2, (H + 2 * KV) * D), generator=g).to(dtype).to(device)
        m = kernels.build_slot_map(i32(*new), *tables, nb, opened, free, ctl, BS, n + 2)
        # Requests with the prompt stand behind it.
        behind = torch.where(member >= 0, prompt, 0).int()
        of = torch.searchsorted(m.cu_tokens[1:].contiguous(), torch.arange(n + 2, dtype=torch.int32, device=device), right=True)
        positions = torch.where(m.positions >= 0, m.positions + behind[of.clamp(max=batch - 1)], -1).int()
        q, _ = kernels.rotate_rows(cut(x, 0, H), cut(x, H, KV), positions, f, q_weight=wq, k_weight=wk, eps=EPS,
                                   value=cut(x, H + KV, KV), slots=m.slots, hot_k=hot[0], hot_v=hot[1],
                                   q_out=torch.zeros((n + 2, H, D), dtype=dtype, device=device))
        out = tierkv_prefix_attention(
            q, m.cu_tokens, *tables, hot[0], hot[1], *warm, width, H // KV, D ** -0.5, member, order[None],
            torch.full_like(order[None], WARM), torch.tensor([[BS] * (pblocks - 1) + [prompt - BS * (pblocks - 1)]],
                                                             dtype=torch.int32, device=device),
            cold_mode="masked", seq_num_blocks=nb, max_tokens=max(new), out=torch.zeros_like(q))
        row = 0
        for b, c in enumerate(new):
            pos = np.arange(held[b], held[b] + c) + (prompt if int(member[b]) >= 0 else 0)
            kk = turned(cut(x[row:row + c], H, KV), pos, f, wk).half().double()
            own_k[b], own_v[b] = torch.cat([own_k[b], kk]), torch.cat([own_v[b], cut(x[row:row + c], H + KV, KV).half().double().cpu()])
            shared = int(member[b]) >= 0
            ks = torch.cat([pk.double().cpu(), own_k[b]]) if shared else own_k[b]
            vs = torch.cat([pv.double().cpu(), own_v[b]]) if shared else own_v[b]
            limit = len(ks) - c + torch.arange(c)
            hidden = torch.arange(len(ks))[None] > limit[:, None]
            for h in range(H):
                logits = (q[row:row + c, h].double().cpu() @ ks[:, h // (H // KV)].t()) * D ** -0.5
                p = torch.softmax(logits.masked_fill(hidden, -torch.inf), 1)
                ref = p @ vs[:, h // (H // KV)]
                # As test_gpu_prefix_attention.py; keys in the pool are rounded
                # from 32 bits, here from 64, so one may be a step apart: 2^-11
                # of it in a logit, twice in p.
                mass = p @ vs[:, h // (H // KV)].abs()
                biggest = (q[row:row + c, h].double().abs().cpu() @ ks[:, h // (H // KV)].abs().t()).amax(1, keepdim=True) * D ** -0.5
                tol = mass * (2 * 2.0 ** -11 + 2.0 ** -20 + 2 * (2.0 ** -11 + (D + 8) * 2.0 ** -24) * biggest)
                tol = tol + ref.abs() * torch.finfo(dtype).eps / 2 + 2.0 ** -23
                assert ((out[row:row + c, h].double().cpu() - ref).abs() <= tol).all()
            held[b] += c
            row += c
        assert (out[n:] == 0).all() and int(ctl[2]) == 0
    assert workspace_error_word(device) == 0


def runtime(device, **kw):
    return BatchedTieredKVRuntime(1, 2, KV, D, 512, hot_fraction=0.5, warm_fraction=0.5, device=device, extend_tokens=64, **kw)


@pytest.mark.parametrize("interleaved", [False, True])
def test_extend_layer_rotates_on_the_way_into_the_cache(device, interleaved):
    """The same as rows rotated before the call, with the runtime's own keys."""
    g = torch.Generator().manual_seed(5)
    a, b = runtime(device), runtime(device)
    prompt_k, prompt_v = torch.randn((2, 2, KV, 70, D), generator=g).half().to(device)
    for rt in (a, b):
        rt.prefill_layer(0, prompt_k, prompt_v)
    q = torch.randn((2, H, 21, D), generator=g).half().to(device)
    k, v = torch.randn((2, 2, KV, 21, D), generator=g).half().to(device)
    f = frequencies(device)
    w = (1 + 0.2 * torch.randn(D, generator=g)).to(device)
    rotary = dict(inv_freq=f, q_weight=w, k_weight=w, eps=EPS, interleaved=interleaved)
    rows = lambda t: t.transpose(1, 2).reshape(42, -1, D)   # noqa: E731
    back = lambda t: t.view(2, 21, -1, D).transpose(1, 2)   # noqa: E731
    pos = (70 + torch.arange(21, dtype=torch.int32, device=device)).repeat(2)
    rq, rk = kernels.rotate_rows(rows(q), rows(k), pos, **rotary)
    got = a.extend_layer(0, q, k, v, H // KV, 0.125, rotary=rotary)
    want = b.extend_layer(0, back(rq), back(rk), v, H // KV, 0.125)
    assert torch.equal(got, want)
    assert torch.equal(a.layers[0].hot_k, b.layers[0].hot_k) and torch.equal(a.layers[0].hot_v, b.layers[0].hot_v)
    assert torch.equal(a.layers[0].states, b.layers[0].states)
    # Refused before anything changes.
    before = a.layers[0].meta.clone()
    for bad in (dict(inv_freq=f.double()), dict(inv_freq=f, q_weight=w[:8]), dict(inv_freq=f, eps=-1.0)):
        with pytest.raises(ValueError):
            a.extend_layer(0, q, k, v, H // KV, 0.125, rotary=bad)
    with pytest.raises(ValueError):
        a.extend_layer(0, q.bfloat16(), k, v, H // KV, 0.125, rotary=rotary)
    assert torch.equal(a.layers[0].meta, before)


@pytest.mark.parametrize("fmt", ["absmax_i8", "ref_u8"])
def test_read_layer_gives_the_cache_back(device, fmt):
    rt = runtime(device, warm_format=fmt)
    k, v = torch.randn((2, 2, KV, 100, D)).half().to(device)
    rt.prefill_layer(0, k, v)
    rk, rv = rt.read_layer(0, 0, 104, torch.float32)
    assert rk.shape == (2, KV, 104, D) and (rk[:, :, 100:] == 0).all()
    st = rt.layers[0]
    tier = st.states[:, :7].repeat_interleave(BS, 1)[:, :100]
    for got, x in ((rk[:, :, :100], k), (rv[:, :, :100], v)):
        for b in range(2):
            hot, warm, cold = (tier[b] == t for t in (HOT, WARM, COLD))
            assert torch.equal(got[b][:, hot], x[b][:, hot].float()) and (got[b][:, cold] == 0).all()
            # A block's or a row's largest magnitude over 127 codes, half a
            # step (absmax), or its range over 255, one step (ref_u8).
            step = x.abs().max() / 127 / 2 if fmt == "absmax_i8" else (x.max() - x.min()) / 255
            assert (got[b][:, warm] - x[b][:, warm].float()).abs().max() <= step * 1.01 + 2.0 ** -9
    part = rt.read_layer(0, 37, 9)
    assert torch.equal(part[0], rk[:, :, 37:46].half()) and torch.equal(part[1], rv[:, :, 37:46].half())
    with pytest.raises(ValueError):
        rt.read_layer(0, -1, 4)
    assert rt.read_layer(0, 3, 0)[0].shape == (2, KV, 0, D)
