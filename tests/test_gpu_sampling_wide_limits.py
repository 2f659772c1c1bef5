"""Token choice with a top-k in the hundreds and thousands (the lists of more
than 512 tokens, and the rows that one workgroup walks by digits), handed on
to top-p and min-p, and the largest vocabularies: exactly the oracle's tokens."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import serving
from paged_tierkv_amd import kernels

from test_gpu_serving_step import logits

pytestmark = pytest.mark.gpu


def compare(device, x, rng, **kw):
    batch = x.shape[0]
    u = rng.random(batch).astype(np.float32)
    tok, prob = kernels.sample_tokens(x.to(device), torch.from_numpy(u).to(device), **kw)
    exp = [serving.sample_row(x[b].float().numpy(), u[b], **kw) for b in range(batch)]
    assert tok.tolist() == [e[0] for e in exp], kw
    np.testing.assert_allclose(prob.cpu().numpy(), [e[1] for e in exp], rtol=2.0 ** -23)


@pytest.mark.parametrize("kind", ["plain", "ties", "masked"])
@pytest.mark.parametrize("vocab,dtype", [(1500, torch.float32), (32000, torch.float16), (128256, torch.float32),
                                         (50257, torch.bfloat16)])
@pytest.mark.parametrize("top_k", [400, 512, 513, 700, 1000, 1024, 1025, 3000])
def test_many_tokens_kept(device, kind, vocab, dtype, top_k):
    rng = np.random.default_rng(vocab + top_k)
    x = logits(rng, 3, vocab, dtype, kind)
    for kw in (dict(), dict(top_p=0.9), dict(top_p=0.9, min_p=0.002), dict(temperature=2.5, top_p=0.97),
               dict(temperature=0.3, top_p=0.6), dict(temperature=50.0, top_p=0.5)):
        compare(device, x, rng, top_k=top_k, **kw)


@pytest.mark.parametrize("kind", ["plain", "ties"])
@pytest.mark.parametrize("vocab,dtype", [((1 << 20) - 3, torch.float32), (1 << 20, torch.float16), (600001, torch.bfloat16)])
def test_vocabularies_up_to_the_largest(device, kind, vocab, dtype):
    rng = np.random.default_rng(vocab)
    x = logits(rng, 2, vocab, dtype, kind)
    for kw in (dict(), dict(top_k=40), dict(top_k=2000, top_p=0.9), dict(top_p=0.9), dict(top_p=0.999, temperature=2.0),
               dict(min_p=0.01)):
        compare(device, x, rng, **kw)


def test_rows_with_limits_of_their_own_over_the_whole_range(device):
    rng = np.random.default_rng(9)
    batch, vocab = 60, 20000
    x = torch.cat([logits(rng, 20, vocab, torch.float32, kind) for kind in ("plain", "ties", "masked")])
    u = rng.random(batch).astype(np.float32)
    t = (0.3 + 2 * rng.random(batch)).astype(np.float32)
    k = rng.choice([0, 1, 30, 512, 513, 900, 1024, 1025, 2500, 19999, 20000], batch).astype(np.int32)
    p = rng.choice([1.0, 0.95, 0.5], batch).astype(np.float32)
    m = rng.choice([0.0, 0.01], batch).astype(np.float32)
    dev = lambda a: torch.from_numpy(a).to(device)   # noqa: E731
    got, _ = kernels.sample_tokens(x.to(device), dev(u), dev(t), dev(k), dev(p), dev(m))
    assert got.tolist() == [serving.sample_row(x[b].numpy(), u[b], t[b], int(k[b]), p[b], m[b])[0] for b in range(batch)]
