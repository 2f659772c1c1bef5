"""A sampling limit given as a tensor of any numeric type (CPU: what the
launch is given)."""

from __future__ import annotations

import pytest
import torch

from paged_tierkv_amd import kernels

MAX = kernels.SAMPLE_MAX_VOCAB


def limit(x):
    t, _ = kernels._limit(x, "top_k", x.numel(), x.device, torch.int32)
    assert t.dtype == torch.int32 and t.is_contiguous()
    return t.tolist()


@pytest.mark.parametrize("dtype,values,want", [
    (torch.int32, [7, 0, 2 ** 31 - 1], [7, 0, 2 ** 31 - 1]),
    (torch.int64, [7, -2 ** 40, 2 ** 32 + 1], [7, 0, MAX]),
    (torch.int16, [7, -3, 32767], [7, 0, 32767]),
    (torch.int8, [7, -3, 127], [7, 0, 127]),
    (torch.uint8, [7, 0, 255], [7, 0, 255]),
    (torch.bool, [True, False, True], [1, 0, 1]),
    (torch.float32, [7.0, float("nan"), float("inf")], [7, 0, MAX]),
    (torch.float16, [7.0, -1.0, 60000.0], [7, 0, 60000]),
    (torch.bfloat16, [7.0, float("-inf"), 1e30], [7, 0, MAX]),
])
def test_top_k_tensors_of_any_type(dtype, values, want):
    assert limit(torch.tensor(values, dtype=dtype)) == want


def test_top_k_tensors_of_any_stride():
    assert limit(torch.arange(12, dtype=torch.int64)[::4]) == [0, 4, 8]
