"""Serving-step calls as programs make them: from several threads, with bounds
below what a step brings, with limits of every kind.  Inputs, bounds of error
and the oracle are those of test_gpu_serving_step."""

from __future__ import annotations

import threading

import numpy as np
import pytest
import torch

from oracle import serving
from paged_tierkv_amd import kernels

from test_gpu_serving_step import call, gpu, step, tables

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
