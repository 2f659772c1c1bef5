"""The cache object's crop hook: the drop-in runtime's is a no-op as the
reference's (tierkv_policy.py:1518-1528); the batched runtime has no way to
take tokens back and says so (CPU)."""

from __future__ import annotations

from types import SimpleNamespace

import pytest

from paged_tierkv_amd.tierkv_policy import TieredKVCache


def cache(batched, tokens=40):
    c = TieredKVCache(SimpleNamespace(is_batched=batched, num_layers=1, begin_forward=lambda n: None,
                                      finish_forward=lambda: None))
    c.begin_forward(tokens)
    c.finish_forward()
    return c


@pytest.mark.parametrize("length", [39, 1, 0, -1, -40])
def test_the_batched_runtime_refuses_to_shorten_the_cache(length):
    c = cache(True)
    with pytest.raises(NotImplementedError, match="shorten"):
        c.crop(length)
    assert c.get_seq_length() == 40


@pytest.mark.parametrize("length", [40, 41, 10 ** 9])
def test_a_crop_that_shortens_nothing_is_taken(length):
    assert cache(True).crop(length) is None
    assert cache(True, 0).crop(0) is None


def test_the_drop_in_runtime_s_hook_is_a_no_op():
    c = cache(False)
    assert c.crop(3) is None and c.get_seq_length() == 40
