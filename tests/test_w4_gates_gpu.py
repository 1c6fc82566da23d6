"""The gated epilogue of products with matrices in four bits over the whole range of a gate."""
from __future__ import annotations

import pytest
import torch

DEV = "cuda"


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 16, 17, 64, 200])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_gates_from_minus_102_to_102(M, out):
    """Two elements a row, so that nothing is summed: gate = -x0 (1 and -1 as weights) and up = x1 exactly; silu(gate) * up at the bottom is as small as
    a number gets, and far from 0 where exp(-gate) has no float32 number or 1 + exp(-gate) no reciprocal."""
    from fellm_b200 import ops
    g = torch.Generator(device=DEV).manual_seed(M)
    levels = torch.zeros(16 * 9, 64, dtype=torch.int8, device=DEV)
    scales = torch.ones(16 * 9, 1, device=DEV)
    for block in range(9):
        rows = torch.arange(8, device=DEV) + 16 * block
        levels[rows, block] = -1                              # gate: minus element `block`
        levels[rows + 8, 9 + block] = 1                       # up: element 9 + `block`
    w4 = ops.pack_w4(levels, scales, 64)
    gates = torch.tensor([0.0, -20.0, -60.0, -80.0, -86.0, -87.5, -88.5, -95.0, 95.0], device=DEV)
    x = torch.zeros(M, 64, device=DEV)
    x[:, :9] = -(gates + (torch.rand(M, 9, generator=g, device=DEV) * 8 - 4).mul(gates.abs().clamp(max=1)) + torch.linspace(-3, 3, M, device=DEV)[:, None])
    x[:, 9:18] = torch.rand(M, 9, generator=g, device=DEV) + 0.5
    x[:, 12:18:2] *= -1
    x = x.bfloat16()
    got = ops.gemm_w4(x, w4, swiglu=True, out_dtype=out).double()
    ops.check_umma_status(DEV)
    gate, up = -x[:, :9].double(), x[:, 9:18].double()
    want = (gate * torch.sigmoid(gate) * up).repeat_interleave(8, 1)
    size = gate.abs().repeat_interleave(8, 1)
    if out == torch.bfloat16:
        # half a step, and the approximate exponential's two units and 1.18 units for every unit of its argument, |gate| / 2, whose square is taken,
        # behind it the reciprocal and four products (units of 2^-23: 4 + 1.18 |gate| + 2 + 4)
        room = 2.0 ** -8 * 1.001 * want.abs() + (10 + 1.2 * size) * 2.0 ** -23 * want.abs() + 2.0 ** -133
    else:
        # float32: the exponential (a unit of 2^-23, or of 2^-149 where it is that small), a sum, a quotient, two products
        room = 8 * 2.0 ** -24 * want.abs() + 2 * size * 2.0 ** -149 + 2.0 ** -148
    assert ((got - want).abs() <= room).all(), float(((got - want).abs() / room).max())
    assert (want[gate.repeat_interleave(8, 1) < -88] != 0).any() or M < 16


@pytest.mark.gpu
@pytest.mark.parametrize("M", [2, 40])
def test_gates_that_are_no_numbers(M):
    from fellm_b200 import ops
    levels = torch.zeros(16, 64, dtype=torch.int8, device=DEV)
    levels[:8, 0], levels[8:, 1] = 1, 1
    levels[:, 2:] = 1
    w4 = ops.pack_w4(levels, torch.ones(16, 1, device=DEV), 64)
    for value, up in ((float("inf"), float("inf")), (float("nan"), float("nan"))):
        x = torch.zeros(M, 64, device=DEV, dtype=torch.bfloat16)
        x[0, 2] = value                                       # (gate and up)
        for out in (torch.bfloat16, torch.float32):
            got = ops.gemm_w4(x, w4, swiglu=True, out_dtype=out)
            assert torch.equal(got[0].float(), torch.full((8,), up, device=DEV)) or (up != up and got[0].isnan().all())
            assert (got[1:] == 0).all()
