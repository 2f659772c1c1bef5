"""Serving-step calls as programs make them: from several threads, with bounds
below what a step brings, with limits of every kind.  Inputs, bounds of error
and the oracle are those of test_gpu_serving_step."""

from __future__ import annotations

import threading

import numpy as np
import pytest
import torch

from oracle import codec, serving
from paged_tierkv_amd import kernels
from paged_tierkv_amd.tierkv_hip import DecodeWorkspace

from test_gpu_serving_step import call, check, gpu, step, tables

pytestmark = pytest.mark.gpu


def test_threads_on_one_stream_get_their_own_results(device):
    """Three threads on the default stream, each with steps of its own shape:
    every result is the one it gets alone."""
    steps = [step(41, [3, 90], [900, 200], 8, 2, 64), step(42, [60, 2, 5, 1], [70, 1500, 40, 9], 8, 2, 128),
             step(43, [1] * 40, [33 + i for i in range(40)], 4, 4, 64)]
    xs = [torch.randn((b, v), device=device) for b, v in ((8, 40000), (1, 3000), (64, 1000))]
    us = [torch.rand(x.shape[0], device=device) for x in xs]
    maps = [tables(np.random.default_rng(i), b, 30, 16, b * 40) for i, b in enumerate((3, 300, 70))]

    def one(i):
        state = [gpu(a, device) for a in maps[i]]
        new = torch.full((state[0].shape[0],), 7 + i, dtype=torch.int32, device=device)
        m = kernels.build_slot_map(new, *state, 16, state[0].shape[0] * 10)
        return [call(steps[i], device, "masked"), *kernels.sample_tokens(xs[i], us[i], top_p=0.9),
                *kernels.sample_tokens(xs[i], us[i], top_k=30), *m, *state]

    alone = [one(i) for i in range(3)]
    torch.cuda.synchronize()
    results = [[] for _ in range(3)]
    threads = [threading.Thread(target=lambda i=i: results[i].extend(one(i) for _ in range(12))) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(3):
        assert len(results[i]) == 12
        for got in results[i]:
            assert all(torch.equal(g, e) for g, e in zip(got, alone[i]))


@pytest.mark.parametrize("new,held,heads,kv,d,bound,rows", [
    ([9, 5, 0, 20], [60, 300, 4, 20], 8, 2, 64, 6, None),            # narrow tiles
    ([300, 3, 40], [900, 70, 41], 8, 1, 128, 37, None),              # wide tiles, one bound inside a request's second
    ([90, 1], [2500, 3000], 16, 1, 64, 33, None),                    # cut tiles
    ([9, 30], [60, 300], 8, 2, 64, 1, None),
    ([9, 30], [60, 300], 8, 2, 64, None, 20),                        # packed rows that end inside a request
    ([6, 4], [5, 4], 4, 2, 64, 3, None),                             # more new tokens than the request holds
])
@pytest.mark.parametrize("cold", ["masked", "zero_logit"])
def test_rows_within_a_bound_that_is_too_low_are_right(device, new, held, heads, kv, d, bound, rows, cold):
    """Of a request that brings more tokens than max_tokens (or than there are
    rows), the first rows see what they see in any case, the others stay as
    they were, and the error word tells."""
    s = step(51 + len(new), new, held, heads, kv, d)
    count = int(s["cu"][-1]) if rows is None else rows
    done = np.concatenate([s["cu"][b] + np.arange(min(n, bound or n)) for b, n in enumerate(new)])
    done = done[done < count]
    q = s["q"].to(device)[:count]
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device=device)
    ws = DecodeWorkspace(device)
    call(s, device, cold, q=q, out=out, max_tokens=bound, workspace=ws)
    assert ws.error_word() == 4
    left = np.setdiff1d(np.arange(count), done)
    assert (out[torch.from_numpy(left).to(device)] == 7.0).all()
    full = torch.zeros(s["q"].shape, dtype=q.dtype, device=device)
    full[:count] = out
    check(full, s, cold, done)
    call(s, device, cold, out=full, max_tokens=max(new), workspace=ws)
    assert ws.error_word() == 0


def test_a_bound_that_is_too_low_is_raised_when_errors_are_checked(device, monkeypatch):
    s = step(52, [9, 5], [60, 30], 8, 2, 64)
    monkeypatch.setenv("TIERKV_CHECK_ERRORS", "1")
    call(s, device, "masked", max_tokens=9)
    with pytest.raises(RuntimeError, match="max_tokens"):
        call(s, device, "masked", max_tokens=8)


def far_from_zero(s, rng, mean, dev):
    """Keys of a cache in the reference format at ``mean`` +- ``dev`` in every
    dim, HOT ones too: zero points of about -255 mean / (6 dev)."""
    key = lambda a: (mean + dev * rng.standard_normal(a.shape)).astype(np.float16)   # noqa: E731
    s["hot"] = (key(s["hot"][0]), s["hot"][1])
    qk, ks, kz = codec.quantize_ref_u8(key(s["warm"][0]))
    s["warm"], s["meta"] = (qk, s["warm"][1]), (ks, kz, *s["meta"][2:])
    return kz


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("mean,dev", [(10, 0.2), (-30, 0.1), (100, 2.0), (100, 0.3)])
@pytest.mark.parametrize("new,held,heads,kv,d", [([3, 5], [40, 33], 4, 2, 64), ([60, 3], [120, 40], 8, 1, 128),
                                                 ([4], [20], 2, 1, 40)])
def test_reference_format_keys_far_from_zero(device, new, held, heads, kv, d, mean, dev, dtype):
    """|code - zero| well past 2048, where fp16 has no more whole numbers."""
    rng = np.random.default_rng(int(abs(mean) + 10 * dev))
    s = step(61, new, held, heads, kv, d, fmt="ref_u8", dtype=dtype, cold=0.1, warm=0.85)
    assert np.abs(far_from_zero(s, rng, mean, dev).astype(np.float64)).max() > 1500
    check(call(s, device, "masked"), s, "masked")


@pytest.mark.parametrize("zero", [-65504.0, 65504.0, -40000.0, 255.0, 0.0])
def test_reference_format_zero_points_over_their_whole_range(device, zero):
    """code - zero past what fp16 holds; the logits are ordinary numbers."""
    s = step(62, [40, 3], [90, 60], 4, 2, 64, fmt="ref_u8", cold=0, warm=0.8)
    ks, kz, vs, vz = s["meta"]
    scale = np.float16(2.0 ** -11 if abs(zero) > 1000 else 2.0 ** -7)
    s["meta"] = (np.full_like(ks, scale), np.full_like(kz, zero), vs, vz)
    mean = np.float16(-zero * float(scale))
    s["hot"] = ((s["hot"][0].astype(np.float32) * 0.03 + mean).astype(np.float16), s["hot"][1])
    out = call(s, device, "masked")
    assert torch.isfinite(out.float()).all()
    check(out, s, "masked")
