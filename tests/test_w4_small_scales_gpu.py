"""Quantising groups whose scale is next to the smallest normal number."""
from __future__ import annotations

import pytest
import torch

import w4_util

DEV = "cuda"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_scales_next_to_the_smallest_normal_number(dtype, group):
    """A scale is an eighth of the largest magnitude in five significant bits, or 0 where that is below 2^-126: 7.75 * 2^-126 makes 31/32 of it, which is
    below, 7.875 * 2^-126 is a tie that rounds to it."""
    from fellm_b200 import ops
    g = torch.Generator(device=DEV).manual_seed(group)
    tops = torch.arange(7 * 32, 9 * 32 + 1, device=DEV, dtype=torch.float64) / 32 * 2.0 ** -126               # (all of at most eight bits or one more)
    tops = tops.to(dtype)
    if dtype == torch.float32:
        tops = torch.cat([tops, torch.nextafter(tops, torch.zeros_like(tops)), torch.nextafter(tops, torch.ones_like(tops))])
    w = (torch.rand(2 * tops.numel(), group, generator=g, device=DEV).double() * 2 - 1) * 6.9 * 2.0 ** -126
    w = w.to(dtype)
    at = torch.randint(0, group, (2 * tops.numel(), 1), generator=g, device=DEV)
    w.scatter_(1, at, torch.cat([tops, -tops])[:, None])
    q, s = w4_util.plain_quantize(w, group)
    assert (s == 0).any() and (s != 0).any()
    got = ops.quantize_w4(w, group)
    assert torch.equal(ops.dequantize_w4(got, torch.float32).double(), w4_util.plain_values(q, s, group))
