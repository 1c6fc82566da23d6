"""Plain forms of the operators on matrices in four bits, in 64 bits, and inputs whose products are exact."""
from __future__ import annotations

import torch


def plain_scale(piece):
    """The scale of one group [N, <= G] (float64), [N, 1]."""
    big = piece.abs().amax(1, keepdim=True)
    mant, expo = torch.frexp(big / 8)
    s = torch.ldexp(torch.round(mant * 32), expo - 5).clamp(max=31 * 2.0 ** 118)
    s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
    return torch.where(piece.amax(1, keepdim=True) > -piece.amin(1, keepdim=True), -s, s)


def plain_quantize(w, group):
    """(levels int8 [N, K], scales float64 [N, groups]); w / s in exact arithmetic: a float64 quotient of a float32 number by
    five bits is correctly rounded and cannot fall on a half that it is not."""
    w = w.double()
    levels, scales = torch.empty(w.shape, dtype=torch.int8, device=w.device), []
    for at in range(0, w.shape[1], group):
        piece = w[:, at:at + group]
        s = plain_scale(piece)
        q = torch.round(piece / torch.where(s == 0, torch.ones_like(s), s)).clamp(-8, 7)
        levels[:, at:at + group] = torch.where(s == 0, torch.zeros_like(q), q).to(torch.int8)
        scales.append(s)
    return levels, torch.cat(scales, 1)


def plain_values(levels, scales, group):
    return levels.double() * scales.double().repeat_interleave(group, 1)[:, :levels.shape[1]]


def interleave(t):
    """Rows [gate | up] -> 8 gate, 8 up, ..."""
    gate, up = t.chunk(2, 0)
    F = gate.shape[0]
    return torch.stack([gate.reshape(F // 8, 8, -1), up.reshape(F // 8, 8, -1)], 1).reshape(2 * F, -1).contiguous()


def plain_product(x, w, bias=None, epi="store"):
    """epi: store | relu2 | swiglu (rows of w: 8 gate, 8 up, ...), float64."""
    y = x.double() @ w.T
    if bias is not None:
        y = y + bias.double()
    if epi == "relu2":
        return y.clamp(min=0) ** 2
    if epi == "swiglu":
        z = y.reshape(y.shape[0], -1, 2, 8)
        gate, up = z[:, :, 0].reshape(y.shape[0], -1), z[:, :, 1].reshape(y.shape[0], -1)
        return gate * torch.sigmoid(gate) * up
    return y


def random_matrix(N, K, group, gen, device):
    """Levels and scales (bfloat16) of every kind: both signs, all of -8..7, five significant bits."""
    levels = torch.randint(-8, 8, (N, K), generator=gen, device=device, dtype=torch.int8)
    m = torch.randint(16, 32, (N, -(-K // group)), generator=gen, device=device).float()
    sign = torch.randint(0, 2, m.shape, generator=gen, device=device).float() * 2 - 1
    return levels, (m * sign / 32).bfloat16()


def whole_rows(M, K, dtype, gen, device):
    """Rows of whole numbers with which every product and every sum of products is a float32 number exactly, in any order
    and however an addition rounds: a product is a multiple of 2^-5 and below 8 |x|, a sum of K of them below 8 K max|x|.
    bfloat16: |x| <= 4, 2^5 * 8 K * 4 <= 2^24 for K <= 16384.  float32: whole numbers up to 1025 (11 bits: two of the three
    bfloat16 pieces), at most 16 in a row: 2^5 * 16 * 8 * 1025 < 2^23."""
    if dtype == torch.bfloat16:
        return torch.randint(-4, 5, (M, K), generator=gen, device=device).to(dtype)
    x = torch.zeros(M, K, device=device)
    for _ in range(min(K, 16)):
        at = torch.randint(0, K, (M, 1), generator=gen, device=device)
        x.scatter_(1, at, torch.randint(-2 ** 10, 2 ** 10 + 1, (M, 1), generator=gen, device=device).float() + 1)
    return x
