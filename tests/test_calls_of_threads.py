"""Calls from several host threads on one stream.  A call of more than one
launch hands state from launch to launch through scratch that the stream's
calls share, and a ctypes call gives up the interpreter lock, so each call has
to be enqueued whole.  Here the library is a stand-in (CPU) that notes which
calls are inside it at a time and with which scratch."""

from __future__ import annotations

import threading
import time

import pytest
import torch

from paged_tierkv_amd import _lib, kernels, tierkv_hip


class _AnyDevice:
    def __eq__(self, other):
        return True


class _OnGpu(torch.Tensor):
    """A host tensor that passes for a GPU tensor."""

    is_cuda = property(lambda self: True)


def on_gpu(t):
    return t.as_subclass(_OnGpu)


class _Library:
    """The entry points the calls below use: sizes, and launches that take a while."""

    def __init__(self):
        self.inside, self.most, self.calls, self.lost = 0, 0, 0, 0
        self.guard = threading.Lock()
        self.workspaces = None     # called inside a launch: the scratch that calls share now

    def __getattr__(self, name):
        if name.endswith("_bytes"):
            return lambda *a: 4096 * (1 + a[0])
        return self._launch

    def _launch(self, *args):
        with self.guard:
            self.inside += 1
            self.calls += 1
            self.most = max(self.most, self.inside)
        time.sleep(0.003)
        # The scratch that this call was given is still the one in use.
        if self.workspaces is not None and not any(p in args for p in self.workspaces()):
            self.lost += 1
        with self.guard:
            self.inside -= 1
        return _lib.TIERKV_OK


@pytest.fixture
def library(monkeypatch):
    lib = _Library()
    monkeypatch.setattr(_lib, "lib", lambda: lib)
    monkeypatch.setattr(_lib, "stream_of", lambda device: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: _AnyDevice())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: "stream")
    monkeypatch.setattr(kernels, "_scratch_ws", {})
    monkeypatch.setattr(kernels, "_prefill_ws", {})
    monkeypatch.setattr(tierkv_hip, "_implicit", {})
    monkeypatch.setattr(tierkv_hip, "_REBIND", {})
    monkeypatch.setattr(tierkv_hip, "stream_workspace", lambda device=None: tierkv_hip._implicit.setdefault(
        0, tierkv_hip.DecodeWorkspace("cpu")))
    monkeypatch.delenv("TIERKV_CHECK_ERRORS", raising=False)
    return lib


def sample(batch):
    kernels.sample_tokens(on_gpu(torch.zeros((batch, 50))), on_gpu(torch.zeros(batch)), top_p=0.5)


def slot_map(batch):
    i32 = lambda *shape: on_gpu(torch.zeros(shape, dtype=torch.int32))   # noqa: E731
    kernels.build_slot_map(i32(batch), i32(batch, 4), i32(batch, 4), i32(batch, 4), i32(batch), i32(batch), i32(9), i32(4),
                           16, 8)


def prefill_scores(batch):
    q = on_gpu(torch.zeros((batch, 2, 16, 8), dtype=torch.float16))
    kernels.prefill_block_mass(q, q, 16, 1.0)


def pools():
    f16 = lambda: on_gpu(torch.zeros((2, 1, 16, 64), dtype=torch.float16))          # noqa: E731
    i8 = lambda: on_gpu(torch.zeros((2, 1, 16, 64), dtype=torch.int8))              # noqa: E731
    scale = lambda: on_gpu(torch.ones((2, 1)))                                      # noqa: E731
    return f16(), f16(), i8(), i8(), scale(), None, scale(), None


def tables(batch):
    return [on_gpu(torch.zeros((batch, 4), dtype=torch.int32)) for _ in range(3)]


def extend(batch):
    q = on_gpu(torch.zeros((batch, 2, 64), dtype=torch.float16))
    cu = on_gpu(torch.arange(batch + 1, dtype=torch.int32))
    tierkv_hip.tierkv_extend_attention(q, cu, *tables(batch), *pools(), 4, 2, 1.0)


def decode_with_scores(batch):
    q = on_gpu(torch.zeros((batch, 2, 1, 64), dtype=torch.float16))
    tierkv_hip.tierkv_decode_attention(q, *tables(batch), *pools(), 4, 2, 1.0, True)


def decode_with_scores_again(batch, held={}):
    """The same tables and pools in every call (the short way through the wrapper)."""
    args = held.setdefault(batch, (on_gpu(torch.zeros((batch, 2, 1, 64), dtype=torch.float16)), *tables(batch), *pools()))
    tierkv_hip.tierkv_decode_attention(*args, 4, 2, 1.0, True)


@pytest.mark.parametrize("call", [sample, slot_map, prefill_scores, extend, decode_with_scores, decode_with_scores_again])
def test_two_threads_on_one_stream_enqueue_their_calls_whole(library, call):
    def shared():
        own = [*kernels._scratch_ws.values(), *kernels._prefill_ws.values()]
        return [t.data_ptr() for t in own] + [ws.data_ptr() for ws in tierkv_hip._implicit.values()]

    library.workspaces = shared
    errors = []

    def work(i):
        try:
            for n in range(6):
                call(1 + (i + n) % 3 + n)        # the scratch grows under way
        except Exception as e:                   # (shown by the test, not by the thread)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and library.calls == 18
    assert library.most == 1, "launches of two calls interleave on one stream"
    assert library.lost == 0, "a call's scratch was replaced before its launches were enqueued"


def test_a_call_that_is_refused_lets_the_next_one_in(library):
    done = []
    with pytest.raises(ValueError):
        kernels.sample_tokens(on_gpu(torch.zeros((2, 50))), on_gpu(torch.zeros(2)), min_p=2.0)
    library._launch = lambda *a: _lib.TIERKV_ERR_UNSUPPORTED
    library.tierkv_last_error = lambda: b"refused"
    for call in (sample, extend):
        with pytest.raises(RuntimeError, match="refused"):
            call(2)
    del library._launch
    t = threading.Thread(target=lambda: (sample(1), extend(1), done.append(True)))
    t.start()
    t.join(20)
    assert done
