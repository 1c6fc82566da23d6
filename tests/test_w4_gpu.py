"""Matrices in four bits on the GPU, against plain forms in 64 bits."""
from __future__ import annotations

import zlib

import pytest
import torch

import w4_util

DEV = "cuda"
SIZES = [(16, 64, 32), (1, 1, 32), (17, 33, 32), (40, 200, 64), (129, 130, 128), (1003, 1357, 32), (256, 1024, 64), (272, 2056, 128), (2064, 64, 64),
         (48, 8200, 128), (2100, 200, 32), (4100, 520, 128), (40000, 136, 32), (4104, 4104, 64)]


def _gen(*seed):
    return torch.Generator(device=DEV).manual_seed(zlib.crc32(repr(seed).encode()))


def _room(x, w, bias, out_bf16):
    """K products summed in float32 in any order, each addition truncating: at most 1.25 K 2^-23 of the sum of magnitudes (17
    terms aligned in an MMA of 16 products), half a step of the output's type."""
    K = x.shape[1]
    mags = x.double().abs() @ w.abs().T + (bias.double().abs() if bias is not None else 0.0)
    return 1.25 * K * 2.0 ** -23 * mags, (2.0 ** -8 if out_bf16 else 2.0 ** -24) * 1.001


# ---------------------------------------------------------------------------------------------- into the form and out of it

@pytest.mark.gpu
@pytest.mark.parametrize("N,K,group", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantized_values(N, K, group, dtype):
    from fellm_b200 import ops
    g = _gen(N, K, group)
    held = torch.randn(N, K + 5, generator=g, device=DEV) * torch.exp(3 * torch.randn(N, 1, generator=g, device=DEV))
    w = held.to(dtype)[:, :K]                                    # (rows that start anywhere)
    for t in (w, w.contiguous()):
        got = ops.quantize_w4(t, group)
        q, s = w4_util.plain_quantize(t, group)
        want = w4_util.plain_values(q, s, group)
        assert got.shape == (N, K) and got.group == group
        assert torch.equal(ops.dequantize_w4(got).double(), want)
        assert torch.equal(ops.dequantize_w4(got, torch.float32).double(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
def test_halves_ties_and_ends(group):
    """Elements on and next to every half step, groups of zeros, extremes of both signs and equal, tiny and huge magnitudes."""
    from fellm_b200 import ops
    rows = []
    for unit in (1.0, 2.0 ** -7 * 17, 2.0 ** -60 * 31, 2.0 ** 100):
        for sign in (1.0, -1.0):
            base = torch.zeros(group)
            base[0] = -8 * sign * unit                            # the scale: sign * unit
            half = torch.arange(-15, 15, dtype=torch.float32) / 2 * unit
            base[1:31] = half
            up, down = base.clone(), base.clone()
            up[1:31] = torch.nextafter(half, torch.full_like(half, float("inf")))
            down[1:31] = torch.nextafter(half, torch.full_like(half, -float("inf")))
            rows += [base, up, down]
    rows += [torch.zeros(group), torch.full((group,), 3.0), torch.full((group,), -3.0), torch.full((group,), 2.0 ** -149), torch.full((group,), 2.0 ** -123),
             torch.full((group,), 2.0 ** -122), torch.full((group,), 3.4028234663852886e38), -torch.full((group,), 3.4028234663852886e38)]
    both = torch.zeros(group); both[3], both[9] = 5.0, -5.0
    rows.append(both)
    w = torch.stack(rows).to(DEV)
    w = torch.cat([w, w.flip(0)], 1)
    q, s = w4_util.plain_quantize(w, group)
    got = ops.quantize_w4(w, group)
    assert torch.equal(ops.dequantize_w4(got, torch.float32).double(), w4_util.plain_values(q, s, group))


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_group_with_an_element_that_is_not_finite_is_nan(bad, dtype):
    from fellm_b200 import ops
    w = torch.randn(40, 200, generator=_gen(1), device=DEV).to(dtype)
    w[21, 70] = bad
    out = ops.dequantize_w4(ops.quantize_w4(w, 64))
    assert out[21, 64:128].isnan().all()
    out[21, 64:128] = 0
    assert out.isfinite().all()
    y = ops.gemm_w4(torch.zeros(2, 200, device=DEV, dtype=torch.bfloat16), ops.quantize_w4(w, 64))
    assert y[:, 21].isnan().all() and y[:, :21].isfinite().all() and y[:, 22:].isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("N,K,group", SIZES)
def test_packed_levels_come_back(N, K, group):
    from fellm_b200 import ops
    levels, scales = w4_util.random_matrix(N, K, group, _gen(N, K), DEV)
    want = w4_util.plain_values(levels, scales, group)
    wide = torch.zeros(N, K + 3, dtype=torch.int8, device=DEV)
    wide[:, :K] = levels
    for lv, sc in ((levels, scales), (wide[:, :K], scales.float()), (levels, scales.T.contiguous().T)):
        assert torch.equal(ops.dequantize_w4(ops.pack_w4(lv, sc, group)).double(), want)
    out = torch.full((N, K + 3), 7.0, device=DEV)
    ops.dequantize_w4(ops.pack_w4(levels, scales, group), out=out[:, :K])
    assert torch.equal(out[:, :K].double(), want) and (out[:, K:] == 7).all()


@pytest.mark.gpu
def test_levels_and_scales_that_are_refused():
    from fellm_b200 import ops
    from fellm_b200.config.errors import KernelError
    levels, scales = w4_util.random_matrix(33, 100, 32, _gen(5), DEV)
    for v in (-9, 8, 127, -128):
        lv = levels.clone(); lv[32, 99] = v
        with pytest.raises(KernelError, match="levels"):
            ops.pack_w4(lv, scales, 32)
    for v in (33 / 32, 257 / 256, float("inf"), float("nan"), 2.0 ** 123, 2.0 ** -127):
        sc = scales.float(); sc[32, 3] = v
        with pytest.raises(KernelError, match="scales"):
            ops.pack_w4(levels, sc, 32)
    for v in (0.0, -0.0, 31 * 2.0 ** 118, 2.0 ** -126, -1.9375):
        sc = scales.float(); sc[32, 3] = v
        assert torch.equal(ops.dequantize_w4(ops.pack_w4(levels, sc, 32)).double(), w4_util.plain_values(levels, sc, 32))


# ------------------------------------------------------------------------------------------------------------ embedding

@pytest.mark.gpu
@pytest.mark.parametrize("N,K,group", SIZES)
@pytest.mark.parametrize("T", [1, 5, 300])
def test_embedding_rows(N, K, group, T):
    from fellm_b200 import ops
    g = _gen(N, K, T)
    levels, scales = w4_util.random_matrix(N, K, group, g, DEV)
    table = ops.pack_w4(levels, scales, group)
    tokens = torch.randint(0, N, (T,), generator=g, device=DEV, dtype=torch.int32)
    tokens[-1] = N - 1
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    held = torch.full((T + 1, K), 7.0, device=DEV)
    ops.embed_rows_w4(tokens, table, held[:T], status, 0.25)
    assert torch.equal(held[:T].double(), w4_util.plain_values(levels, scales, group)[tokens.long()] * 0.25)
    assert (held[T:] == 7).all() and int(status) == 0
    if T > 1:
        tokens[0], tokens[2] = N, -1
        ops.embed_rows_w4(tokens, table, held[:T], status, 0.25)
        assert int(status) == 1 and (held[[0, 2]] == 0).all()
        assert torch.equal(held[3:T].double(), w4_util.plain_values(levels, scales, group)[tokens[3:].long()] * 0.25)


@pytest.mark.gpu
def test_no_tokens_and_no_rows():
    from fellm_b200 import ops
    w = ops.quantize_w4(torch.randn(32, 64, device=DEV), 32)
    assert ops.embed_rows_w4(torch.zeros(0, dtype=torch.int32, device=DEV), w, torch.empty(0, 64, device=DEV)).shape == (0, 64)
    assert ops.gemm_w4(torch.zeros(0, 64, device=DEV, dtype=torch.bfloat16), w).shape == (0, 32)


# ------------------------------------------------------------------------------------------------------------- products

ROWS = [1, 2, 5, 8, 9, 16, 17, 31, 33, 64, 65, 128, 130, 256, 300, 521]


@pytest.mark.gpu
@pytest.mark.parametrize("N,K,group", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M", ROWS)
def test_whole_numbers_come_out_exactly(N, K, group, dtype, M):
    """Sums that are float32 numbers in every order: any element left out, doubled or in a wrong place shows."""
    from fellm_b200 import ops
    g = _gen(N, K, M)
    levels, scales = w4_util.random_matrix(N, K, group, g, DEV)
    x = w4_util.whole_rows(M, K, dtype, g, DEV)
    got = ops.gemm_w4(x, ops.pack_w4(levels, scales, group), out_dtype=torch.float32)
    ops.check_umma_status(DEV)
    assert torch.equal(got.double(), w4_util.plain_product(x, w4_util.plain_values(levels, scales, group)))


@pytest.mark.gpu
@pytest.mark.parametrize("N,K,group", [(16, 16, 32), (1008, 136, 32), (272, 1024, 64), (2064, 72, 128), (144, 4104, 128), (16, 333, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M", [1, 3, 8, 16, 23, 48, 100, 129, 400])
@pytest.mark.parametrize("epi", ["store", "f32", "acc", "relu2", "swiglu"])
def test_products(N, K, group, dtype, M, epi):
    """Every epilogue, with a bias, from rows that lie apart into rows that lie apart, beside what has to stay."""
    from fellm_b200 import ops
    g = _gen(N, K, M, epi)
    levels, scales = w4_util.random_matrix(N, K, group, g, DEV)
    w4, w = ops.pack_w4(levels, scales, group), w4_util.plain_values(levels, scales, group)
    for shift, pad in ((0, 0), (3, 7), (8, 8)):
        xs = torch.randn(shift + M * (K + pad), generator=g, device=DEV).to(dtype)
        x = xs[shift:].view(M, K + pad)[:, :K]
        bias = torch.randn(N, generator=g, device=DEV) if pad else None
        out_bf16 = dtype == torch.bfloat16 and epi not in ("f32", "acc")
        cols = N // 2 if epi == "swiglu" else N
        held = torch.randn(shift + (M + 1) * (cols + pad), generator=g, device=DEV).to(torch.bfloat16 if out_bf16 else torch.float32)
        before = held.clone()
        view = lambda t: t[shift:shift + M * (cols + pad)].view(M, cols + pad)[:, :cols]  # noqa: E731,B023
        ops.gemm_w4(x, w4, bias, out=view(held), accumulate=epi == "acc", swiglu=epi == "swiglu", act="relu2" if epi == "relu2" else None)
        ops.check_umma_status(DEV)
        sums, step = _room(x, w, bias, out_bf16)
        want = w4_util.plain_product(x, w, bias, epi if epi in ("relu2", "swiglu") else "store")
        if epi == "acc":
            want = want + view(before).double()
            room = sums + 2.0 ** -23 * (view(before).double().abs() + want.abs())
        elif epi == "relu2":
            y = w4_util.plain_product(x, w, bias)
            room = (2 * y.abs() + sums) * sums + (step + 2.0 ** -24) * want.abs()
        elif epi == "swiglu":
            y = w4_util.plain_product(x, w, bias).reshape(M, -1, 2, 8)
            gate, up = y[:, :, 0].reshape(M, -1), y[:, :, 1].reshape(M, -1)
            es = sums.reshape(M, -1, 2, 8)
            eg, eu = es[:, :, 0].reshape(M, -1), es[:, :, 1].reshape(M, -1)
            # |silu'| <= 1.1; the exponential, the sum, the quotient and the product: 8 roundings of float32 at most
            room = 1.1 * eg * (up.abs() + eu) + gate.abs() * eu + (step + 8 * 2.0 ** -24) * want.abs() + 2.0 ** -126
        else:
            room = sums + step * want.abs()
        off = (view(held).double() - want).abs()
        assert (off <= room).all(), float((off / room.clamp(min=1e-300)).max())
        view(held).copy_(view(before))
        assert torch.equal(held, before), "something beside the product's rows was written"


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 4, 20, 200])
def test_float32_rows_keep_all_their_bits(M):
    """One element a row, so that nothing is summed: x q s in float32, correctly rounded twice at most."""
    from fellm_b200 import ops
    g = _gen(M)
    levels, scales = w4_util.random_matrix(40, 200, 64, g, DEV)
    x = torch.zeros(M, 200, device=DEV)
    at = torch.randint(0, 200, (M, 1), generator=g, device=DEV)
    x.scatter_(1, at, torch.randn(M, 1, generator=g, device=DEV) * torch.exp(8 * torch.randn(M, 1, generator=g, device=DEV)))
    got = ops.gemm_w4(x, ops.pack_w4(levels, scales, 64))
    want = x.double() @ w4_util.plain_values(levels, scales, 64).T
    assert ((got.double() - want).abs() <= 2.0 ** -22 * want.abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M", [2, 33, 300])
def test_infinities_stay_in_their_rows(dtype, M):
    from fellm_b200 import ops
    g = _gen(M, 9)
    levels, scales = w4_util.random_matrix(144, 136, 32, g, DEV)
    levels[levels == 0] = 1
    x = torch.randn(M, 136, generator=g, device=DEV).to(dtype)
    w4 = ops.pack_w4(levels, scales, 32)
    clean = ops.gemm_w4(x, w4)
    x[0, 77], x[1, 5] = float("inf"), float("nan")
    got = ops.gemm_w4(x, w4)
    w = w4_util.plain_values(levels, scales, 32)
    assert torch.equal(got[0].double(), w[:, 77].sign() * float("inf")) and got[1].isnan().all()
    assert torch.equal(got[2:], clean[2:])


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 8, 16, 40, 128, 300])
def test_the_same_bits_every_time(M):
    from fellm_b200 import ops
    g = _gen(M, 2)
    w4 = ops.quantize_w4(torch.randn(1024, 2048, generator=g, device=DEV), 64)
    x = torch.randn(M, 2048, generator=g, device=DEV).bfloat16()
    first = ops.gemm_w4(x, w4, out_dtype=torch.float32)
    for _ in range(5):
        assert torch.equal(ops.gemm_w4(x, w4, out_dtype=torch.float32), first)


@pytest.mark.gpu
def test_a_result_cannot_take_the_place_of_x():
    from fellm_b200 import ops
    from fellm_b200.config.errors import KernelError
    w4 = ops.quantize_w4(torch.randn(64, 64, device=DEV), 32)
    for M in (2, 40):
        x = torch.randn(M, 64, device=DEV)
        with pytest.raises(KernelError, match="place"):
            ops.gemm_w4(x, w4, out=x)
        with pytest.raises(KernelError, match="place"):
            ops.gemm_w4(x, w4, out=x, accumulate=True)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 7, 16, 40, 200])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_captured_products_and_products_on_two_streams(M, dtype):
    """The same matrix read by a replayed graph, by this stream and by another one at once; new rows of x for every replay."""
    from fellm_b200 import ops
    g = _gen(M, 11)
    levels, scales = w4_util.random_matrix(2064, 520, 64, g, DEV)
    w4, w = ops.pack_w4(levels, scales, 64), w4_util.plain_values(levels, scales, 64)
    xs = [w4_util.whole_rows(M, 520, dtype, g, DEV) for _ in range(6)]
    want = [w4_util.plain_product(x, w) for x in xs]
    held = xs[0].clone()
    y = torch.empty(M, 2064, device=DEV)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.gemm_w4(held, w4, out=y)                       # (loads the kernels before the capture)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        half = ops.gemm_w4(held, w4, out_dtype=torch.float32) if M > 16 else None
        ops.gemm_w4(held, w4, out=y)
    for i in range(1, 6):
        held.copy_(xs[i])
        graph.replay()
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            beside = [ops.gemm_w4(xs[j], w4, out_dtype=torch.float32) for j in range(6)]
        here = [ops.gemm_w4(xs[j], w4, out_dtype=torch.float32) for j in range(6)]
        torch.cuda.synchronize()
        assert torch.equal(y.double(), want[i]) and (half is None or torch.equal(half.double(), want[i]))
        for got in (beside, here):
            assert all(torch.equal(a.double(), b) for a, b in zip(got, want))
    ops.check_umma_status(DEV)


@pytest.mark.gpu
def test_laying_out_is_refused_inside_a_capture():
    from fellm_b200 import ops
    from fellm_b200.config.errors import KernelError
    w = torch.randn(64, 64, device=DEV)
    ops.quantize_w4(w, 32)
    lv, sc = torch.zeros(64, 64, dtype=torch.int8, device=DEV), torch.ones(64, 2, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(KernelError, match="captured"):
            ops.quantize_w4(w, 32)
        with pytest.raises(KernelError, match="captured"):
            ops.pack_w4(lv, sc, 32)
        w.add_(1)


@pytest.mark.gpu
def test_a_matrix_of_zeros_and_rows_of_zeros():
    from fellm_b200 import ops
    zero = ops.quantize_w4(torch.zeros(40, 200, device=DEV), 64)
    assert (ops.dequantize_w4(zero) == 0).all()
    for M in (1, 9, 40):
        assert (ops.gemm_w4(torch.randn(M, 200, device=DEV).bfloat16(), zero) == 0).all()
        assert (ops.gemm_w4(torch.zeros(M, 200, device=DEV), ops.quantize_w4(torch.randn(40, 200, device=DEV), 64)) == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(M, N, K) for M in (1, 3, 8, 9, 16) for N, K in ((64, 200), (1024, 1024), (2000, 64), (48, 2048))]
                         + [(M, N, K) for M in (17, 32, 33, 64, 100, 128) for N, K in ((64, 200), (1024, 1024), (2016, 64), (96, 2048), (2048, 520))])
def test_a_norm_handed_on(M, N, K):
    """What an accumulate product leaves for the RMSNorm behind it, and the product that reads that."""
    from fellm_b200 import ops
    g, part = _gen(M, N, K), 16 if M <= 16 else 32
    ops.reserve_norm_handoff(DEV, N)
    levels, scales = w4_util.random_matrix(N, K, 64, g, DEV)
    w4 = ops.pack_w4(levels, scales, 64)
    x = torch.randn(M, K, generator=g, device=DEV).bfloat16()
    stream, weight = torch.randn(M, N, generator=g, device=DEV), torch.rand(N, generator=g, device=DEV) + 0.5
    plain = stream.clone()
    ops.gemm_w4(x, w4, out=plain, accumulate=True)
    ops.forget_norm_handoff()
    ops.expect_norm(stream, weight)
    ops.gemm_w4(x, w4, out=stream, accumulate=True)
    assert torch.equal(stream, plain)
    h = ops.norm_handoff(stream, weight)
    assert h is not None and h.parts == N // part and h.rows == M
    assert torch.equal(h.xg, (stream * weight).bfloat16())
    sums = h.ssq[:M * h.parts].view(M, h.parts).double()
    want = stream.double().view(M, h.parts, part).pow(2).sum(-1)
    assert ((sums - want).abs() <= 20 * 2.0 ** -24 * want).all()         # squares and sums of positive numbers: 16 roundings one by one, 6 in pairs
    next_levels, next_scales = w4_util.random_matrix(144, N, 64, g, DEV)
    bias = torch.randn(144, generator=g, device=DEV)
    w = w4_util.plain_values(next_levels, next_scales, 64)
    got = ops.gemm_w4(h.xg, ops.pack_w4(next_levels, next_scales, 64), bias, out_dtype=torch.float32, row_scale=(h.ssq, h.parts, 1e-5))
    factor = 1 / (want.sum(-1, keepdim=True) / N + 1e-5).sqrt()
    exact = h.xg.double() @ w.T * factor + bias.double()
    room = 1.25 * N * 2.0 ** -23 * (h.xg.double().abs() @ w.abs().T) * factor + (20 + N / 16) * 2.0 ** -24 * (exact.abs() + bias.double().abs())
    assert ((got.double() - exact).abs() <= room).all()
    gate = w4_util.random_matrix(160, N, 64, g, DEV)
    w = w4_util.plain_values(*gate, 64)
    got = ops.gemm_w4(h.xg, ops.pack_w4(*gate, 64), swiglu=True, out_dtype=torch.float32, row_scale=(h.ssq, h.parts, 1e-5)).double()
    exact = (h.xg.double() @ w.T * factor).view(M, -1, 2, 8)
    room = (1.25 * N * 2.0 ** -23 * (h.xg.double().abs() @ w.abs().T) * factor).view(M, -1, 2, 8) + (20 + N / 16) * 2.0 ** -24 * exact.abs()
    silu = exact[:, :, 0] * torch.sigmoid(exact[:, :, 0])
    # |d silu| <= 1.1 |d gate|; the function itself in float32: some 2^-20 of it
    room = (1.1 * room[:, :, 0] * (exact[:, :, 1].abs() + room[:, :, 1]) + silu.abs() * room[:, :, 1] + 2.0 ** -20 * (silu * exact[:, :, 1]).abs()).reshape(M, -1)
    assert ((got - (silu * exact[:, :, 1]).reshape(M, -1)).abs() <= room).all()
    stream.add_(1)
    assert ops.norm_handoff(stream, weight) is None
    ops.forget_norm_handoff()


@pytest.mark.gpu
def test_a_norm_that_is_not_handed_on():
    from fellm_b200 import ops
    from fellm_b200.config.errors import KernelError
    w4 = ops.quantize_w4(torch.randn(64, 64, device=DEV), 32)
    ssq = torch.ones(129 * 4, device=DEV)
    for x in (torch.zeros(129, 64, device=DEV, dtype=torch.bfloat16), torch.zeros(2, 64, device=DEV), torch.zeros(130, device=DEV, dtype=torch.bfloat16)[1:129].view(2, 64)):
        with pytest.raises(KernelError, match="handed-on"):
            ops.gemm_w4(x, w4, row_scale=(ssq, 4, 1e-5))
    x = torch.zeros(40, 64, device=DEV, dtype=torch.bfloat16)
    for sums, parts in ((ssq[:40 * 4 - 1], 4), (ssq, 0), (ssq, 129), (ssq.double(), 4), (ssq[1:], 4), (ssq.cpu(), 4), (ssq[::2], 2)):
        for rows in (x, x[:2]):
            if rows is x or sums.numel() > 4 * 40 or sums.dtype != torch.float32:
                with pytest.raises(KernelError, match="handed-on"):
                    ops.gemm_w4(rows, w4, row_scale=(sums, parts, 1e-5))


@pytest.mark.gpu
def test_a_norm_of_another_width_or_of_too_many_rows_is_not_handed_on():
    """A view that begins where the announced rows do is not those rows."""
    from fellm_b200 import ops
    ops.reserve_norm_handoff(DEV, 128)
    weight = torch.ones(128, device=DEV)
    w64, w128 = (ops.quantize_w4(torch.randn(n, 64, device=DEV), 32) for n in (64, 128))
    stream = torch.zeros(200, 128, device=DEV)
    for rows, w, out in ((1, w64, stream[:1, :64]), (200, w128, stream), (40, w64, stream.view(-1, 64)[:40])):
        ops.forget_norm_handoff()
        ops.expect_norm(stream[:100], weight)
        x = torch.randn(rows, 64, device=DEV).bfloat16()
        want = out + ops.gemm_w4(x, w, out_dtype=torch.float32)
        ops.expect_norm(stream[:100], weight)
        ops.gemm_w4(x, w, out=out, accumulate=True)
        assert torch.equal(out, want) and ops._handoff is None
    ops.forget_norm_handoff()


@pytest.mark.gpu
@pytest.mark.parametrize("M", [4, 40])
def test_rows_that_came_with_a_norm_are_not_written_over(M):
    """A product that reads a handed-on norm's rows hands none on: its rows lie where it would write."""
    from fellm_b200 import ops
    g = _gen(M, 7)
    ops.reserve_norm_handoff(DEV, 256)
    w4 = ops.pack_w4(*w4_util.random_matrix(256, 256, 64, g, DEV), 64)
    x, weight = torch.randn(M, 256, generator=g, device=DEV).bfloat16(), torch.rand(256, generator=g, device=DEV) + 0.5
    stream = torch.randn(M, 256, generator=g, device=DEV)
    ops.forget_norm_handoff()
    ops.expect_norm(stream, weight)
    ops.gemm_w4(x, w4, out=stream, accumulate=True)
    h = ops.norm_handoff(stream, weight)
    rows = h.xg.clone()
    other = torch.zeros(M, 256, device=DEV)
    ops.expect_norm(other, weight)
    ops.gemm_w4(h.xg, w4, out=other, accumulate=True, row_scale=(h.ssq, h.parts, 1e-5))
    assert torch.equal(h.xg, rows) and ops.norm_handoff(other, weight) is None and ops.norm_handoff(stream, weight) is h
    want = ops.gemm_w4(h.xg, w4, out_dtype=torch.float32, row_scale=(h.ssq, h.parts, 1e-5))
    assert torch.equal(other, want)
    ops.forget_norm_handoff()


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K,dtype", [(17, 65536, 64, "bfloat16"), (40, 65536, 128, "bfloat16"), (128, 65536, 256, "bfloat16"), (64, 65536, 512, "bfloat16"),
                                         (300, 40000, 32, "bfloat16"), (20, 60000, 64, "float32"), (300, 30000, 64, "float32")])
def test_more_tiles_than_stages(M, N, K, dtype):
    """Of a short K the warps that make weights are tiles ahead of the products when they come to finish the last one with the others."""
    from fellm_b200 import ops
    g = _gen(M, N, K)
    levels, scales = w4_util.random_matrix(N, K, 64, g, DEV)
    w4, values = ops.pack_w4(levels, scales, 64), w4_util.plain_values(levels, scales, 64)
    x = torch.randn(M, K, generator=g, device=DEV).to(getattr(torch, dtype))
    exact, room = x.double() @ values.T, 1.25 * K * 2.0 ** -23 * (x.double().abs() @ values.abs().T)
    for _ in range(10):
        assert ((ops.gemm_w4(x, w4, out_dtype=torch.float32) - exact).abs() <= room).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("M,K", [(17, 8192), (40, 16384), (200, 40000), (600, 20000), (1100, 16384), (300, 70000)])
def test_long_sums_are_as_near_as_float32_sums(M, K, dtype):
    """Of n numbers of one size added one by one in float32, rounding to nearest, the k-th sum is off by 2^-24 / sqrt(3) of itself in the mean, and has
    sqrt(k / n) of the last one's size: 2^-24 sqrt(n / 6) together.  Over a whole result the kernel's sums, by the type's rules and any order,
    are no further off."""
    from fellm_b200 import ops
    g = _gen(M, K)
    levels, scales = w4_util.random_matrix(512, K, 64, g, DEV)
    w4, values = ops.pack_w4(levels, scales, 64), w4_util.plain_values(levels, scales, 64)
    x = torch.randn(M, K, generator=g, device=DEV).to(getattr(torch, dtype))
    exact = x.double() @ values.T
    for kind in ("store", "accumulate"):
        out = torch.zeros(M, 512, device=DEV)
        ops.gemm_w4(x, w4, out=out, accumulate=kind == "accumulate")
        assert (out - exact).norm() <= 2.0 ** -24 * (K / 6) ** 0.5 * exact.norm()

