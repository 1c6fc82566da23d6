"""Matrices in four bits: what is refused, on the CPU, and the form's arithmetic."""
from __future__ import annotations

import pytest
import torch

import w4_util
from fellm_b200 import ops
from fellm_b200.config.errors import KernelError


def test_level_times_scale_is_a_bfloat16_number():
    levels = torch.arange(-8, 8, dtype=torch.float64)
    for m in range(16, 32):
        for e in (-126 - 4, -40, 0, 118):
            v = levels * (m * 2.0 ** e)
            assert torch.equal(v.to(torch.bfloat16).double(), v)


def test_plain_quantizing_takes_the_extreme_to_minus_eight():
    g = torch.Generator().manual_seed(3)
    w = torch.randn(64, 96, generator=g)
    q, s = w4_util.plain_quantize(w, 32)
    at = w.reshape(64, 3, 32).abs().argmax(-1, keepdim=True)
    assert (q.reshape(64, 3, 32).gather(-1, at) == -8).all()
    # nothing is further off than half a step, but what would be level +8 (an extreme of the other sign: one step, and the
    # scale's rounding of 2^-5 of eight steps, a quarter)
    off = (w4_util.plain_values(q, s, 32) - w.double()).abs().reshape(64, 3, 32)
    assert (off <= s.abs().unsqueeze(-1) * 1.25).all()


def _fake(N=32, K=64, group=32):
    q, s = ops._w4_room(N, K, group, "cpu")
    return ops.W4(q, s, N, K, group)


@pytest.mark.parametrize("group", [0, 16, 48, 256, -32])
def test_groups_that_are_none(group):
    with pytest.raises(KernelError, match="group"):
        ops.quantize_w4(torch.zeros(16, 64), group)
    with pytest.raises(KernelError, match="group"):
        ops.pack_w4(torch.zeros(16, 64, dtype=torch.int8), torch.ones(16, 1), group)


def test_matrices_that_are_none():
    for w in (torch.zeros(64), torch.zeros(4, 4, 4), torch.zeros(0, 64), torch.zeros(64, 0), torch.zeros(64, 32).T, torch.zeros(1, 2 ** 20 + 1)):
        with pytest.raises(KernelError):
            ops.quantize_w4(w, 32)
    with pytest.raises(KernelError, match="CUDA"):
        ops.quantize_w4(torch.zeros(16, 64), 32)
    with pytest.raises(KernelError, match="int8"):
        ops.pack_w4(torch.zeros(16, 64), torch.ones(16, 2), 32)
    with pytest.raises(KernelError, match="scales"):
        ops.pack_w4(torch.zeros(16, 64, dtype=torch.int8), torch.ones(16, 3), 32)
    with pytest.raises(KernelError, match="dtype"):
        ops.pack_w4(torch.zeros(16, 64, dtype=torch.int8), torch.ones(16, 2, dtype=torch.float16), 32)


@pytest.mark.parametrize("kw", [
    dict(x=torch.zeros(2, 63)), dict(x=torch.zeros(64)), dict(x=torch.zeros(2, 64, dtype=torch.float16)), dict(x=torch.zeros(64, 2).T),
    dict(accumulate=True), dict(swiglu=True, act="relu2"), dict(act="gelu"), dict(out=torch.zeros(2, 31)), dict(out=torch.zeros(3, 32)),
    dict(out=torch.zeros(32, 2).T), dict(out=torch.zeros(1, 32).expand(2, 32)), dict(out=torch.zeros(2, 32, dtype=torch.float16)),
    dict(out=torch.zeros(2, 32, dtype=torch.bfloat16)), dict(x=torch.zeros(2, 64, dtype=torch.bfloat16), out=torch.zeros(2, 32, dtype=torch.bfloat16), accumulate=True),
    dict(x=torch.zeros(2, 64, dtype=torch.bfloat16), out=torch.zeros(2, 32), out_dtype=torch.bfloat16),
    dict(bias=torch.zeros(31)), dict(bias=torch.zeros(32, dtype=torch.bfloat16)), dict()])
def test_products_that_are_refused(kw):
    with pytest.raises(KernelError):
        ops.gemm_w4(**{**dict(x=torch.zeros(2, 64), w=_fake()), **kw})


def test_gated_rows_come_in_sixteens():
    with pytest.raises(KernelError, match="16"):
        ops.gemm_w4(torch.zeros(2, 64), _fake(N=24), swiglu=True)


def test_rows_of_a_table_that_are_refused():
    tok = torch.zeros(3, dtype=torch.int32)
    for out in (torch.zeros(3, 63), torch.zeros(2, 64), torch.zeros(3, 64, dtype=torch.bfloat16), torch.zeros(64, 3).T, torch.zeros(3, 64)):
        with pytest.raises(KernelError):
            ops.embed_rows_w4(tok, _fake(), out)
    with pytest.raises(KernelError):
        ops.embed_rows_w4(tok.long(), _fake(), torch.zeros(3, 64))
    with pytest.raises(KernelError):
        ops.dequantize_w4(_fake(), out=torch.zeros(32, 63))
    with pytest.raises(KernelError, match="over one another"):
        ops.dequantize_w4(_fake(), out=torch.zeros(1, 64).expand(32, 64))
