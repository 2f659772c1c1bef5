"""Steps of few tokens per request whose tables are so wide that their parts'
workspace would pass twice the plan's: they are planned on the device, and give
what the oracle gives (bounds as in test_gpu_prefix_attention.py)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from paged_tierkv_amd import _lib
from paged_tierkv_amd.tierkv_hip import DecodeWorkspace
from test_gpu_prefix_attention import HOT, check, launch, step, tensors

pytestmark = pytest.mark.gpu


def widen(s, width):
    """The requests' tables with entries behind the counts up to ``width``,
    which name slots that are not there."""
    for k, fill in enumerate((10 ** 6, HOT, 7)):
        a = s["own"][k]
        wide = np.full((len(a), width), fill, np.int32)
        wide[:, :a.shape[1]] = a
        s["own"][k] = wide
    return s


CASES = [
    # width, copies of (prefixes, member, new, held), heads, kv, d, bs, what a step's parts would take in MB
    (12000, 60, ([30, 400], [0, 1, 1, 1, -1], [1, 1, 1, 0, 1], [20, 50, 64, 9, 300]), 16, 4, 64, 64, 1178),      # single tokens
    (60000, 8, ([30, 400], [0, 1, 1, 1, -1], [1, 5, 3, 0, 2], [20, 50, 64, 9, 300]), 16, 2, 64, 64, 781),        # drafts, two tiles
    (2400000, 2, ([30, 400], [0, 1, 1, -1], [1, 1, 1, 1], [20, 500, 64, 300]), 4, 1, 128, 64, 3072),            # no tile of more than 32 rows
]


@pytest.mark.parametrize("width,many,rows,heads,kv,d,bs,step_mb", CASES)
@pytest.mark.parametrize("fmt,cold,dtype", [("absmax_i8", "zero_logit", torch.float16), ("ref_u8", "masked", torch.bfloat16)])
def test_steps_of_very_wide_tables(device, width, many, rows, heads, kv, d, bs, step_mb, fmt, cold, dtype):
    prefixes, member, new, held = rows
    print(f"[prefix] {many} x {new} in tables of {width} blocks of {bs}, {heads}/{kv} x {d}, {fmt} {cold}", flush=True)
    s = widen(step(width % 97, prefixes, member * many, new * many, held * many, heads, kv, d, bs, fmt, dtype), width)
    rows, most = int(s["cu"][-1]) + 2, max(new)
    nbytes = _lib.lib().tierkv_prefix_workspace_bytes(len(s["member"]), 2, rows, most, heads, kv, width,
                                                      s["pre"][0].shape[1], bs, d)
    assert 0 < nbytes < step_mb * 1e6 / 2
    t = tensors(s, device)
    ws = DecodeWorkspace(device)
    out = torch.full_like(t["q"], 7.0)
    launch(t, s, cold, workspace=ws, max_tokens=most, out=out)
    assert ws.error_word() == 0
    check(out, s, cold)
    assert (out[-2:] == 7.0).all()
    assert torch.equal(launch(t, s, cold, workspace=ws, max_tokens=most)[:-2], out[:-2])
