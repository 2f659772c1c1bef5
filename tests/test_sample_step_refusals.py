"""A sampled decode step whose arguments are refused does not run the step
(CPU: the runner's own step is a stand-in)."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from paged_tierkv_amd import _lib, hf_llama


class _OnGpu(torch.Tensor):
    is_cuda = property(lambda self: True)


def on_gpu(t):
    return t.as_subclass(_OnGpu)


@pytest.fixture
def runner(monkeypatch):
    monkeypatch.setattr(_lib, "lib", lambda: None)
    r = hf_llama.DecodeGraphRunner.__new__(hf_llama.DecodeGraphRunner)
    r.rt = SimpleNamespace(batch=3)
    r.ids = torch.zeros((3, 1), dtype=torch.long)
    r.model = SimpleNamespace(config=SimpleNamespace(vocab_size=50))
    r.steps = 0

    def step(ids):
        r.steps += 1
        raise StopIteration

    r.step = step
    return r


U = on_gpu(torch.zeros(3))


@pytest.mark.parametrize("u,limits", [
    (on_gpu(torch.zeros(2)), {}), (on_gpu(torch.zeros(3, dtype=torch.float64)), {}), (torch.zeros(3), {}), (None, {}),
    (U, dict(temperature=-1.0)), (U, dict(temperature=float("nan"))), (U, dict(top_p=-0.1)), (U, dict(min_p=1.5)),
    (U, dict(top_k=torch.zeros(2, dtype=torch.int32))), (U, dict(min_p=torch.zeros((3, 1)))),
])
def test_refused_arguments_run_no_step(runner, u, limits):
    with pytest.raises(ValueError):
        runner.sample_step(torch.zeros((3, 1), dtype=torch.long), u, **limits)
    assert runner.steps == 0


def test_a_vocabulary_past_the_limit_runs_no_step(runner):
    runner.model.config.vocab_size = (1 << 20) + 1
    with pytest.raises(ValueError, match="vocabularies"):
        runner.sample_step(torch.zeros((3, 1), dtype=torch.long), U)
    assert runner.steps == 0


def test_arguments_that_are_taken_run_it(runner):
    for limits in (dict(), dict(temperature=0.0, top_k=5, top_p=0.5, min_p=0.1), dict(top_p=torch.ones(3))):
        with pytest.raises(StopIteration):
            runner.sample_step(torch.zeros((3, 1), dtype=torch.long), U, **limits)
    assert runner.steps == 3
