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
