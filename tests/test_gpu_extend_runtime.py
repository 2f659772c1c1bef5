"""Several new tokens on a cache that holds some, through the batched runtime
and the HF hooks, and sampled decode steps through the graph runner."""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytest.importorskip("transformers")

from oracle import serving  # noqa: E402
from paged_tierkv_amd import hf_llama, kernels, tierkv_policy as tp  # noqa: E402
from paged_tierkv_amd.runtime import BatchedTieredKVRuntime  # noqa: E402

pytestmark = pytest.mark.gpu


def runtime(device, **kw):
    a = dict(num_layers=1, batch=3, kv_heads=2, head_dim=64, max_seq_len=400, hot_fraction=0.2, warm_fraction=0.5,
             policy_interval=16, extend_tokens=48, device=device)
    a.update(kw)
    return BatchedTieredKVRuntime(**a)


def rand(g, *shape):
    return torch.randn(shape, generator=g).half()


@pytest.mark.parametrize("fmt,cold", [("absmax_i8", "masked"), ("ref_u8", "zero_logit")])
def test_extend_layer_matches_oracle(device, fmt, cold):
    g = torch.Generator().manual_seed(1)
    rt = runtime(device, warm_format=fmt, cold_mode=cold)
    B, kv, H, d = 3, 2, 8, 64
    rt.prefill_layer(0, rand(g, B, kv, 101, d).to(device), rand(g, B, kv, 101, d).to(device))
    st = rt.layers[0]
    for T in (5, 48, 1, 11):
        q, k, v = (rand(g, B, h, T, d).to(device) for h in (H, kv, kv))
        # V as a projection's view, K contiguous: both layouts the hooks produce.
        v = v.transpose(1, 2).contiguous().transpose(1, 2)
        before = [t.cpu().numpy().copy() for t in (st.table, st.states, st.lengths, st.nblocks, st.open, st.hot_free,
                                                   st.ctl)]
        out = rt.extend_layer(0, q, k, v, H // kv, d ** -0.5, policy_step=False)
        slots, _, cu, _ = serving.build_slot_map(np.full(B, T, np.int32), *before, 16, B * T)
        for t, e in zip((st.table, st.states, st.lengths, st.nblocks, st.open, st.ctl),
                        (*before[:5], before[6])):
            np.testing.assert_array_equal(t.cpu().numpy(), e)
        hk, hv = st.hot_k.cpu().numpy(), st.hot_v.cpu().numpy()
        for pool, x in ((hk, k), (hv, v)):
            rows = x.transpose(1, 2).reshape(B * T, kv, d).cpu().numpy()
            np.testing.assert_array_equal(pool[slots // 16, :, slots % 16], rows)
        meta = [None if t is None else t.cpu().numpy() for t in (st.k_scale, st.k_zero, st.v_scale, st.v_zero)]
        exp, mass, _ = serving.extend_attention(
            q.transpose(1, 2).reshape(B * T, H, d).float().cpu().numpy(), cu, before[0], before[1], before[2], before[3],
            hk, hv, st.warm_k.cpu().numpy(), st.warm_v.cpu().numpy(), *meta, H // kv, d ** -0.5, fmt, cold)
        got = out.reshape(B * T, H, d).float().cpu().numpy()
        # Two roundings of at most 2^-11 of what is added, the logits' (2^-12 here) and the output's.
        assert (np.abs(got - exp) <= mass * (2 * 2.0 ** -11 + 2.0 ** -12) + np.abs(exp) * 2.0 ** -11 + 2.0 ** -23).all()
        rt.tick_layer(0, torch.rand((B, H, rt.max_blocks), generator=g).to(device), rt._blocks[0])
    rt.check_errors()
    assert rt._blocks[0] == int(st.nblocks[0]) and rt.seq_len == 101 + 65


def test_extend_layer_retiers_to_the_budgets(device):
    g = torch.Generator().manual_seed(2)
    rt = runtime(device)
    rt.prefill_layer(0, rand(g, 3, 2, 200, 64).to(device), rand(g, 3, 2, 200, 64).to(device))
    for _ in range(3):
        q, k, v = (rand(g, 3, h, 48, 64).to(device) for h in (4, 2, 2))
        rt.extend_layer(0, q, k, v, 2, 0.125)
        hot, warm = rt.budgets(rt._blocks[0])
        states = rt.layers[0].states.cpu().numpy()[:, :rt._blocks[0]]
        assert ((states == 0).sum(1) <= hot).all() and ((states == 1).sum(1) <= warm).all()
    rt.check_errors()


def test_extend_layer_refusals(device):
    g = torch.Generator().manual_seed(3)
    rt = runtime(device, max_seq_len=160)
    x = lambda h, T: rand(g, 3, h, T, 64).to(device)   # noqa: E731
    rt.prefill_layer(0, x(2, 100), x(2, 100))
    with pytest.raises(ValueError, match="extend_tokens"):
        rt.extend_layer(0, x(4, 49), x(2, 49), x(2, 49), 2, 0.125)
    with pytest.raises(ValueError, match="geometry"):
        rt.extend_layer(0, x(4, 8), x(2, 9), x(2, 9), 2, 0.125)
    rt.extend_layer(0, x(4, 40), x(2, 40), x(2, 40), 2, 0.125)
    with pytest.raises(RuntimeError, match="max_seq_len"):
        rt.extend_layer(0, x(4, 30), x(2, 30), x(2, 30), 2, 0.125)
    assert not runtime(device, extend_tokens=0).extends(8)
    with pytest.raises(ValueError, match="extend_tokens"):
        runtime(device, extend_tokens=-1)


@pytest.fixture(scope="module")
def model(device):
    from transformers import LlamaConfig, LlamaForCausalLM

    cfg = LlamaConfig(hidden_size=512, intermediate_size=1024, num_hidden_layers=2, num_attention_heads=8,
                      num_key_value_heads=2, head_dim=64, vocab_size=1000, max_position_embeddings=1024)
    cfg._attn_implementation = "sdpa"
    torch.manual_seed(0)
    m = LlamaForCausalLM(cfg).to(device=device, dtype=torch.float16).eval()
    hf_llama.install()
    yield m
    hf_llama.uninstall()
    tp.reset_global_tierkv()


def test_follow_up_prompts_through_the_model_match_dense(model, device):
    """Prompt, two follow-up prompts and single steps in between, all HOT: the
    logits of stock dense attention over the same tokens."""
    cfg = model.config
    ids = torch.randint(0, 1000, (3, 160), generator=torch.Generator().manual_seed(5)).to(device)
    rt = BatchedTieredKVRuntime(cfg.num_hidden_layers, 3, cfg.num_key_value_heads, cfg.head_dim, 240, hot_fraction=1.0,
                                warm_fraction=0.0, policy_mode="hot_warm", policy_interval=8, device=device,
                                extend_tokens=64)
    with torch.no_grad():
        ref = model(input_ids=ids, use_cache=False).logits
        at, got = 0, []
        for n in (70, 1, 1, 50, 1, 7, 30):
            got.append(model(input_ids=ids[:, at:at + n], past_key_values=rt.cache, use_cache=True).logits)
            at += n
    rt.check_errors()
    assert at == 160 == rt.cache.get_seq_length() == rt.seq_len
    torch.testing.assert_close(torch.cat(got, 1), ref, atol=2e-2, rtol=2e-2)


def test_without_extend_tokens_a_prompt_replaces_the_cache(model, device):
    """What a multi-token forward did before stays: a new prompt."""
    cfg = model.config
    ids = torch.randint(0, 1000, (2, 90), generator=torch.Generator().manual_seed(6)).to(device)
    rt = BatchedTieredKVRuntime(cfg.num_hidden_layers, 2, cfg.num_key_value_heads, cfg.head_dim, 240, device=device)
    with torch.no_grad():
        for n in (40, 50):
            rt.cache.reset()
            model(input_ids=ids[:, :n], past_key_values=rt.cache, use_cache=True)
    assert int(rt.layers[0].nblocks[0]) == 4 and rt._blocks[0] == 4


def test_sampled_steps_of_the_graph_runner(model, device):
    """Greedy limits give the argmax chain; top-k 1 the same; a draw is
    ``sample_tokens`` of the step's logits."""
    cfg = model.config

    def make():
        return BatchedTieredKVRuntime(cfg.num_hidden_layers, 2, cfg.num_key_value_heads, cfg.head_dim, 200,
                                      policy_interval=8, device=device)

    ids = torch.randint(0, 1000, (2, 60), generator=torch.Generator().manual_seed(7)).to(device)
    u = torch.rand((12, 2), generator=torch.Generator().manual_seed(8)).to(device)

    def run(step):
        rt = make()
        with torch.no_grad():
            tok = model(input_ids=ids, past_key_values=rt.cache, use_cache=True).logits[:, -1].argmax(-1, keepdim=True)
        runner, out = hf_llama.DecodeGraphRunner(model, rt), []
        for i in range(12):
            tok = step(runner, tok, u[i])
            out.append(tok)
        rt.check_errors()
        return torch.cat(out, 1)

    greedy = run(lambda r, t, _: r.step(t)[:, -1].argmax(-1, keepdim=True))
    assert torch.equal(run(lambda r, t, v: r.sample_step(t, v, temperature=0.0)[0]), greedy)
    assert torch.equal(run(lambda r, t, v: r.sample_step(t, v, top_k=1)[0]), greedy)
    limits = dict(temperature=0.8, top_k=40, top_p=0.9)
    drawn = run(lambda r, t, v: r.sample_step(t, v, **limits)[0])
    byhand = run(lambda r, t, v: kernels.sample_tokens(r.step(t)[:, -1], v, **limits)[0][:, None])
    assert torch.equal(drawn, byhand) and ((drawn >= 0) & (drawn < 1000)).all()
