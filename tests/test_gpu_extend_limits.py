"""What the batched runtime does with several new tokens per sequence that do
not fit, or that it cannot take: it says so before anything changes."""

from __future__ import annotations

import pytest
import torch

from paged_tierkv_amd.runtime import BatchedTieredKVRuntime

pytestmark = pytest.mark.gpu


def runtime(device, **kw):
    a = dict(num_layers=1, batch=3, kv_heads=2, head_dim=64, max_seq_len=1600, hot_fraction=0.1, warm_fraction=0.5,
             policy_interval=16, extend_tokens=48, device=device)
    a.update(kw)
    return BatchedTieredKVRuntime(**a)


def rand(device, seed=0):
    g = torch.Generator().manual_seed(seed)
    return lambda h, T, dtype=torch.float16: torch.randn((3, h, T, 64), generator=g).to(dtype).to(device)


def held(rt, layer=0):
    """Everything that a call may change, on the host and on the device."""
    st = rt.layers[layer]
    host = (list(rt._blocks), list(rt._open_tokens), list(rt._hot_bound), rt.seq_len)
    return host, [t.clone() for t in (st.meta, st.hot_k, st.hot_v, st.warm_k, st.warm_v)]


def same(a, b):
    return a[0] == b[0] and all(torch.equal(x, y) for x, y in zip(a[1], b[1]))


@pytest.mark.parametrize("mode", ["hot_warm", "hot_warm_cold"])
def test_tokens_without_a_free_hot_slot_are_refused_before_anything_changes(device, mode):
    """Calls without a tick use up the HOT slots: the first that does not fit
    raises, at the very count where the stack ends, and a tick makes room."""
    rt, x = runtime(device, policy_mode=mode), rand(device)
    rt.prefill_layer(0, x(2, 200), x(2, 200))
    taken = 0
    while True:
        before = held(rt)
        free = int(rt.layers[0].ctl[0])
        try:
            out = rt.extend_layer(0, x(4, 48), x(2, 48), x(2, 48), 2, 0.125, policy_step=False)
        except RuntimeError as e:
            assert "HOT" in str(e)
            break
        assert torch.isfinite(out.float()).all() and free >= 3 * 3
        taken += 1
        assert taken < 60, "the stack never ended"
    assert taken > 1 and free < 3 * 3
    assert same(held(rt), before)
    rt.check_errors()
    assert rt._blocks[0] == int(rt.layers[0].nblocks[0])
    rt.tick_layer(0, torch.rand((3, 4, rt.max_blocks), device=device), rt._blocks[0])
    rt.extend_layer(0, x(4, 48), x(2, 48), x(2, 48), 2, 0.125)
    rt.check_errors()
    assert rt._blocks[0] == int(rt.layers[0].nblocks[0]) and rt.seq_len == 200 + 48 * (taken + 1)


def test_a_step_that_the_device_refuses_gives_zeros(device):
    """The free stack lost behind the host's back: no row is computed, none is
    left as the allocator gave it, and check_errors tells."""
    rt, x = runtime(device), rand(device, 1)
    rt.prefill_layer(0, x(2, 100), x(2, 100))
    rt.layers[0].ctl[0] = 2
    rows = x(4, 48)
    torch.full((3, 48, 4, 64), float("nan"), dtype=torch.float16, device=device)   # what a reused buffer may hold
    out = rt.extend_layer(0, rows, x(2, 48), x(2, 48), 2, 0.125, policy_step=False)
    assert out.shape == (3, 48, 4, 64) and (out == 0).all()
    with pytest.raises(RuntimeError, match="no free HOT slot"):
        rt.check_errors()


def test_the_bound_on_hot_blocks_holds_over_steps_of_all_kinds(device):
    """Decode steps, follow-up tokens and ticks in turn: no sequence ever holds
    more HOT blocks than the host's bound, and nothing is refused."""
    rt, x = runtime(device, num_layers=2), rand(device, 2)
    for layer in range(2):
        rt.prefill_layer(layer, x(2, 333), x(2, 333))
    for i in range(40):
        T = (1, 1, 48, 7, 1)[i % 5]
        tick = rt.begin_step() if T == 1 else True
        for layer in range(2):
            if T == 1:
                rt.decode_layer(layer, x(4, 1), x(2, 1), x(2, 1), 2, 0.125, policy_step=tick)
            else:
                rt.extend_layer(layer, x(4, T), x(2, T), x(2, T), 2, 0.125)
            hot = (rt.layers[layer].states == 0).sum(1).max()
            assert int(hot) <= rt._hot_bound[layer] <= rt.hot_per_seq
        if T == 1:
            rt.end_step()
    rt.check_errors()


@pytest.mark.parametrize("why", ["query fp32", "query fp64", "heads", "groups", "head_dim", "K bf16, V fp16", "query on the host",
                                 "K/V on the host", "scaling", "tokens", "too long"])
def test_a_call_that_is_refused_changes_nothing(device, why):
    rt, x = runtime(device, max_seq_len=260), rand(device, 3)
    rt.prefill_layer(0, x(2, 230), x(2, 230))
    q, k, v, groups, scaling = x(4, 9), x(2, 9), x(2, 9), 2, 0.125
    if why == "query fp32":
        q = q.float()
    if why == "query fp64":
        q = q.double()
    if why == "heads":
        q = x(6, 9)
    if why == "groups":
        groups = 4
    if why == "head_dim":
        q = q[..., :32]
    if why == "K bf16, V fp16":
        k = k.bfloat16()
    if why == "query on the host":
        q = q.cpu()
    if why == "K/V on the host":
        k, v = k.cpu(), v.cpu()
    if why == "scaling":
        scaling = float("nan")
    if why == "tokens":
        q, k, v = x(4, 49), x(2, 49), x(2, 49)
    if why == "too long":
        q, k, v = x(4, 33), x(2, 33), x(2, 33)
    before = held(rt)
    with pytest.raises(RuntimeError if why == "too long" else ValueError):
        rt.extend_layer(0, q, k, v, groups, scaling)
    assert same(held(rt), before)
    rt.extend_layer(0, x(4, 9), x(2, 9), x(2, 9), 2, 0.125)
    rt.check_errors()


def test_a_capture_is_refused(device):
    rt, x = runtime(device), rand(device, 4)
    rt.prefill_layer(0, x(2, 100), x(2, 100))
    q, k, v = x(4, 9), x(2, 9), x(2, 9)
    rt.extend_layer(0, q, k, v, 2, 0.125)
    before = held(rt)
    torch.cuda.synchronize()
    graph, seen = torch.cuda.CUDAGraph(), None
    with torch.cuda.graph(graph):
        try:
            rt.extend_layer(0, q, k, v, 2, 0.125)
        except RuntimeError as e:
            seen = str(e)
        q.add(0)
    assert seen and "captured" in seen and same(held(rt), before)


def test_geometry_that_the_attention_does_not_take_is_refused_at_once(device):
    for kw in (dict(head_dim=256), dict(head_dim=68), dict(block_size=128)):
        with pytest.raises(ValueError, match="extend_tokens"):
            runtime(device, **kw)
    runtime(device, head_dim=256, extend_tokens=0)


def test_keys_and_values_in_32_bits_become_fp16(device):
    outs = []
    for k_type, v_type in ((torch.float16,) * 2, (torch.float32,) * 2, (torch.float32, torch.float16)):
        rt, x = runtime(device), rand(device, 5)
        rt.prefill_layer(0, x(2, 100), x(2, 100))
        q, k, v = x(4, 9), x(2, 9), x(2, 9)
        outs.append(rt.extend_layer(0, q, k.to(k_type), v.to(v_type), 2, 0.125))
        rt.check_errors()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
