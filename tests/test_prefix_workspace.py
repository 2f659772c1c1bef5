"""Workspace sizes of attention with shared prefixes, and the calls that they
are refused or taken for, before any launch (CPU)."""

from __future__ import annotations

import pytest

from paged_tierkv_amd import _lib
from test_shared_prompt_refusals import prefix

MB = 1 << 20


def size(batch, prefixes, rows, most, heads, kv, blocks, pblocks, bs, d):
    return _lib.lib().tierkv_prefix_workspace_bytes(batch, prefixes, rows, most, heads, kv, blocks, pblocks, bs, d)


def call(batch, prefixes, rows, most, heads, kv, blocks, pblocks, bs, d, nbytes):
    return prefix(batch=batch, prefixes=prefixes, rows=rows, most=most, heads=heads, kv=kv, blocks=blocks, stride=blocks,
                  pblocks=pblocks, pstride=pblocks, bs=bs, d=d, qt=heads * d, qh=d, nbytes=nbytes)


# Rows per request up to 64 (tokens times heads of a kv head) are a step, above that a plan.
@pytest.mark.parametrize("batch", [1, 16, 64, 256, 1024, 2000])
@pytest.mark.parametrize("blocks,bs", [(16, 16), (1024, 16), (16384, 16), (32768, 64)])
def test_sizes_do_not_jump_between_the_two_ways(batch, blocks, bs):
    """A step's partials follow the tables' width; they take no more than twice
    what the plan of the same rows takes, however wide the tables are."""
    step, plan = (size(batch, 1, 16 * batch, most, 32, 8, blocks, 512, bs, 128) for most in (16, 17))
    assert 0 < step <= 2 * plan, (step / MB, plan / MB)


def test_steps_whose_launch_is_too_large_are_planned():
    """2000 requests of 16 tokens in tables of 32768 blocks of 64: 10 million
    workgroups as a step, past a launch's 2^32 threads."""
    geometry = (2000, 1, 32000, 16, 32, 8, 32768, 512, 64, 128)
    need = size(*geometry)
    assert 0 < need < 9000 * MB
    assert call(*geometry, need - 1) == 4                    # too small, and not "grid too large"


def test_ordinary_steps_keep_their_way():
    """Sizes of steps as they were: single tokens and drafts of ordinary tables."""
    assert size(64, 1, 64, 1, 32, 8, 17, 512, 16, 128) < 64 * MB
    assert size(256, 4, 256, 1, 32, 8, 13, 256, 16, 128) < 64 * MB
    assert size(24, 2, 120, 5, 32, 4, 6, 94, 16, 64) < 16 * MB
    assert size(2, 1, 2, 1, 32, 8, 2, 38, 16, 128) < MB


OK = dict(batch=2, prefixes=1, rows=8, most=8, heads=8, kv=2, blocks=8, pblocks=8, bs=16, d=64)


@pytest.mark.parametrize("kw", [
    dict(d=20), dict(d=4), dict(d=132), dict(bs=65),
    dict(batch=4096), dict(batch=5000, rows=5000, most=1), dict(prefixes=4095), dict(batch=2000, prefixes=2097),
    dict(blocks=(1 << 27)), dict(pblocks=(1 << 27)), dict(pblocks=(1 << 27) - 1, rows=1 << 20),
    dict(rows=1 << 28), dict(rows=1 << 27, heads=2), dict(batch=1 << 30, rows=1 << 30), dict(prefixes=1 << 30),
    dict(blocks=(1 << 31) - 1, pblocks=(1 << 31) - 1),
])
def test_sizes_that_no_call_takes_have_no_workspace(kw):
    """Whatever the call refuses for its sizes has no workspace, and the other
    way round."""
    a = {**OK, **kw}
    assert size(*a.values()) == -1
    assert call(*a.values(), 1 << 62) in (1, 2) and _lib.last_error()


@pytest.mark.parametrize("kw", [dict(), dict(d=8), dict(d=128), dict(bs=64), dict(batch=4095), dict(prefixes=4094),
                                dict(blocks=(1 << 27) - 2), dict(rows=1 << 26, heads=2)])
def test_sizes_at_the_limits_have_one(kw):
    a = {**OK, **kw}
    need = size(*a.values())
    assert need > 0 and call(*a.values(), need - 1) == 4


def test_a_prefix_and_own_tokens_that_are_walked_together_count_together():
    """A request of 512 rows per kv head and more walks its prefix and its own
    tokens as one row, whose places are 32-bit numbers."""
    half = dict(OK, blocks=1 << 26, pblocks=1 << 26, rows=600)
    for most, taken in ((600, False), (128, False), (127, True), (16, True)):
        a = dict(half, most=most)
        need = size(*a.values())
        assert (need > 0) == taken, most
        assert call(*a.values(), need - 1 if taken else 1 << 62) == (4 if taken else 2)
    a = dict(half, most=600, pblocks=(1 << 26) - 64)      # 1024 tokens fewer
    assert size(*a.values()) > 0
