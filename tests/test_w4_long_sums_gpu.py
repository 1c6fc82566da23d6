"""Products with matrices in four bits over a long K whose results are bfloat16: the sums are those of a float32 result."""
from __future__ import annotations

import pytest
import torch

import w4_util

DEV = "cuda"


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(16, 512, 8192), (17, 512, 4104), (40, 1536, 8192), (128, 272, 40000), (200, 512, 16384), (1029, 2056, 8192), (17, 48, 2 ** 20)])
@pytest.mark.parametrize("act", [None, "relu2"])
def test_a_bfloat16_result_is_the_float32_one_rounded(M, N, K, act):
    from fellm_b200 import ops
    g = torch.Generator(device=DEV).manual_seed(M + N + K)
    w4 = ops.pack_w4(*w4_util.random_matrix(N, K, 128, g, DEV), 128)
    x = torch.randn(M, K, generator=g, device=DEV).bfloat16()
    bias = torch.randn(N, generator=g, device=DEV)
    wide = torch.empty(M, N, device=DEV)
    ops.gemm_w4(x, w4, bias, out=wide, act=act)
    assert torch.equal(ops.gemm_w4(x, w4, bias, act=act), wide.bfloat16())
    ops.check_umma_status(DEV)


def _waves(M, N, K, gen):
    """Rows and a matrix whose sums rise to a peak and come back to nearly nothing eight times over K (so that every share of K, of up to
    eight, holds a rise and a fall): products of one sign in the first half of a period, in the second the negative of as many, one in 64 of
    them a quarter larger."""
    half = K // 16
    levels = torch.randint(1, 8, (N, half), generator=gen, device=DEV, dtype=torch.int8).repeat(1, 16)
    scales = (torch.randint(16, 32, (N, half // 128), generator=gen, device=DEV).float() * 2.0 ** -16).bfloat16().repeat(1, 16)
    up = (torch.rand(M, 8, half, generator=gen, device=DEV) + 0.5).bfloat16()
    more = torch.rand(up.shape, generator=gen, device=DEV) < 1 / 64
    x = torch.stack([up, -torch.where(more, up * 1.25, up)], 2).reshape(M, K)
    return x, levels, scales


@pytest.mark.gpu
@pytest.mark.parametrize("M,K", [(17, 2 ** 18), (200, 2 ** 18), (17, 2 ** 20), (8, 2 ** 20)])
def test_sums_that_rise_and_fall(M, K):
    """Added one by one in float32, rounding to nearest, a sum that rises to S and falls again in even steps is off by 2^-24 / sqrt(3) of its size
    each time, whose mean square is S^2 / 3: 2^-24 S sqrt(K) / 3 together.  Over a whole result the kernel's sums are no further off."""
    from fellm_b200 import ops
    g = torch.Generator(device=DEV).manual_seed(M + K)
    x, levels, scales = _waves(M, 48, K, g)
    w4, values = ops.pack_w4(levels, scales, 128), w4_util.plain_values(levels, scales, 128)
    exact = x.double() @ values.T
    peak = x.double().abs() @ values.abs().T / 16
    room = 2.0 ** -24 * K ** 0.5 / 3 * peak.norm()
    for out in (torch.bfloat16, torch.float32):
        off = (ops.gemm_w4(x, w4, out_dtype=out).double() - exact).norm()
        assert off <= room + (2.0 ** -8 if out == torch.bfloat16 else 2.0 ** -24) * exact.norm(), (out, float(off / room))


@pytest.mark.gpu
@pytest.mark.parametrize("M", [17, 8])
def test_gates_whose_sums_rise_and_fall(M):
    """Element by element, three times the mean."""
    from fellm_b200 import ops
    g, K = torch.Generator(device=DEV).manual_seed(M), 2 ** 20
    x, levels, scales = _waves(M, 48, K, g)
    values = w4_util.plain_values(levels, scales, 128)
    bias = torch.full((48,), 6.0, device=DEV)                  # (gates above 0, where the function is as steep as its argument)
    want = w4_util.plain_product(x, values, bias, "swiglu")
    y, peak = x.double() @ values.T + 6, x.double().abs() @ values.abs().T / 16
    gate, up = (t.reshape(M, -1) for t in y.reshape(M, -1, 2, 8).unbind(2))
    eg, eu = (t.reshape(M, -1) * 2.0 ** -24 * K ** 0.5 for t in peak.reshape(M, -1, 2, 8).unbind(2))
    got = ops.gemm_w4(x, ops.pack_w4(levels, scales, 128), bias, swiglu=True).double()
    # |silu'| <= 1.1; half a step of bfloat16 and 2^-16 for the function
    room = 1.1 * eg * (up.abs() + eu) + gate.abs() * eu + (2.0 ** -8 + 2.0 ** -16) * 1.001 * want.abs()
    assert ((got - want).abs() <= room).all(), float(((got - want).abs() / room).max())


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(8, 1024, 16384), (17, 1024, 8192), (64, 2048, 16384), (128, 96, 40000)])
def test_a_norm_handed_on_behind_a_long_sum(M, N, K):
    """What is handed on are the rows as they are written, whatever the sums are put together from."""
    from fellm_b200 import ops
    g = torch.Generator(device=DEV).manual_seed(M + N + K)
    ops.reserve_norm_handoff(DEV, N)
    w4 = ops.pack_w4(*w4_util.random_matrix(N, K, 64, g, DEV), 64)
    x = torch.randn(M, K, generator=g, device=DEV).bfloat16()
    stream, weight = torch.randn(M, N, generator=g, device=DEV), torch.rand(N, generator=g, device=DEV) + 0.5
    plain = stream.clone()
    ops.gemm_w4(x, w4, out=plain, accumulate=True)
    ops.forget_norm_handoff()
    ops.expect_norm(stream, weight)
    ops.gemm_w4(x, w4, out=stream, accumulate=True)
    h = ops.norm_handoff(stream, weight)
    assert torch.equal(stream, plain) and torch.equal(h.xg, (stream * weight).bfloat16())
    want = stream.double().view(M, h.parts, -1).pow(2).sum(-1)
    assert ((h.ssq[:M * h.parts].view(M, -1).double() - want).abs() <= 20 * 2.0 ** -24 * want).all()        # (squares and at most 16 sums of positive numbers)
    ops.forget_norm_handoff()


@pytest.mark.gpu
@pytest.mark.parametrize("M", [40, 200, 600])
def test_long_sums_in_a_replayed_graph_and_on_two_streams(M):
    from fellm_b200 import ops
    g = torch.Generator(device=DEV).manual_seed(M)
    w4 = ops.pack_w4(*w4_util.random_matrix(1536, 8192, 64, g, DEV), 64)
    xs = [torch.randn(M, 8192, generator=g, device=DEV).bfloat16() for _ in range(4)]
    want = [ops.gemm_w4(x, w4) for x in xs]
    held, y, side = xs[0].clone(), torch.empty(M, 1536, device=DEV, dtype=torch.bfloat16), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.gemm_w4(held, w4, out=y)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.gemm_w4(held, w4, out=y)
    for i in range(4):
        held.copy_(xs[i])
        graph.replay()
        with torch.cuda.stream(side):
            beside = [ops.gemm_w4(x, w4) for x in xs]
        torch.cuda.synchronize()
        assert torch.equal(y, want[i]) and all(torch.equal(a, b) for a, b in zip(beside, want))
    ops.check_umma_status(DEV)
