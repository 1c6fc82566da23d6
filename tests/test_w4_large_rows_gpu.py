"""Products with matrices in four bits at the ends of the numbers' range: a result that is finite comes out, whatever a group's sum of x times
levels would be."""
from __future__ import annotations

import pytest
import torch

import w4_util

DEV = "cuda"


@pytest.mark.gpu
@pytest.mark.parametrize("N,K,group", [(272, 1024, 64), (1008, 136, 32), (144, 4104, 128), (5200, 520, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M", [1, 3, 8, 9, 16, 17, 130])
@pytest.mark.parametrize("rows,scale", [(124, -24), (-110, 90), (-100, -24)])
def test_large_rows_of_small_scales_and_the_other_way_round(N, K, group, dtype, M, rows, scale, monkeypatch):
    """Elements of up to some 2^127: at most K 8 2^-24 times that, below 2^119.  An extreme element meets the largest levels of its group.  Results down to
    the smallest numbers: what is lost there is a last place of 2^-149 for every addition of the tensor cores, and of 2^-140 for every group and every
    warp's share where up to 16 rows are summed in units of 2^10; bfloat16's last place is 2^-133."""
    from fellm_b200 import ops
    g = torch.Generator(device=DEV).manual_seed(N + K + M)
    levels, scales = w4_util.random_matrix(N, K, group, g, DEV)
    levels[::3] = -8
    scales = scales.float().mul(2.0 ** scale).bfloat16()
    x = torch.randn(M, K, generator=g, device=DEV).clamp(-7.9, 7.9).mul(2.0 ** rows).to(dtype)
    x[:, :min(K, 128)] = x[:, :min(K, 128)].abs().clamp(min=2.0 ** rows)
    w4, values = ops.pack_w4(levels, scales, group), w4_util.plain_values(levels, scales, group)
    want, mags = x.double() @ values.T, x.double().abs() @ values.abs().T
    for first in (1 << 24, 0):                               # float32 rows cut by every warp, and cut first
        monkeypatch.setattr(ops, "W4_CUT_FIRST", first)
        for out in (torch.float32,) if dtype == torch.float32 else (torch.float32, torch.bfloat16):
            got = ops.gemm_w4(x, w4, out_dtype=out)
            ops.check_umma_status(DEV)
            # (K additions that truncate, 17 terms aligned in an MMA of 16 products; half a step of the result's type)
            room = 1.25 * K * 2.0 ** -23 * mags + (2.0 ** -24 if out == torch.float32 else 2.0 ** -8) * 1.001 * want.abs()
            room = room + K * 2.0 ** -149 + (K // group + 17) * 2.0 ** -140 + (2.0 ** -134 if out == torch.bfloat16 else 0.0)
            assert got.isfinite().all() and ((got.double() - want).abs() <= room).all()


@pytest.mark.gpu
@pytest.mark.parametrize("M", [2, 8, 16, 40])
def test_large_rows_that_come_with_a_norm(M):
    from fellm_b200 import ops
    g, K, N = torch.Generator(device=DEV).manual_seed(M), 1024, 272
    levels, scales = w4_util.random_matrix(N, K, 64, g, DEV)
    scales = scales.float().mul(2.0 ** -24).bfloat16()
    x = torch.randn(M, K, generator=g, device=DEV).clamp(-7.9, 7.9).abs().mul(2.0 ** 124).bfloat16()
    values = w4_util.plain_values(levels, scales, 64)
    ssq = torch.full((M * 4,), K * 2.0 ** 78, device=DEV)
    factor = 2.0 ** -40                                        # 1 / sqrt(4 ssq / K + 0)
    got = ops.gemm_w4(x, ops.pack_w4(levels, scales, 64), out_dtype=torch.float32, row_scale=(ssq, 4, 0.0)).double()
    want, mags = x.double() @ values.T * factor, x.double().abs() @ values.abs().T * factor
    room = 1.25 * K * 2.0 ** -23 * mags + 4 * 2.0 ** -24 * want.abs()           # (the quotient, the square root, the product)
    assert got.isfinite().all() and ((got - want).abs() <= room).all()
