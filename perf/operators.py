"""The operators on matrices in four bits, as cases to time and compare.

A matrix [n, k] is held as levels of -8..7 and a scale for every `group` consecutive elements of a row; a scale has at
most five significant bits, so that level * scale is a bfloat16 number exactly.  Four operators: a matrix is brought
into that form and read back (`quantize`), multiplied with rows of activations (`product`), multiplied with the gated
activation of a feed-forward behind it (`gated`; its rows are eight of the gate, eight of the up projection, and so
on), and looked up row by row as a token embedding (`embed`).

Widths, feed-forwards and the vocabulary are those of the benchmark's shapes (width 1024, 1536, 2048; feed-forward
4608, 7168, 8192; vocabulary 65,536) or generic ones.
"""
from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
VOCAB = 65536
MOST_FLOPS = 2 * 2048 * 16384 * 2048
MOST_WEIGHTS = 65536 * 2048


# ----------------------------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # one token through a layer's smallest projection: launch and latency
        dict(name="token_small", op="product", rows=1, n=1024, k=1024, group=64, dtype="bfloat16", out="bfloat16", bias=False),
        # one token's logits: the widest matrix of a decode step
        dict(name="token_head", op="product", rows=1, n=VOCAB, k=2048, group=32, dtype="bfloat16", out="float32", bias=False),
        # a small batch decoding through a large square projection with a bias
        dict(name="batch_square", op="product", rows=8, n=8192, k=8192, group=128, dtype="bfloat16", out="bfloat16", bias=True),
        # the 32-bit engine: float32 rows, sizes that are multiples of nothing
        dict(name="rows_float32", op="product", rows=5, n=1003, k=1357, group=32, dtype="float32", out="float32", bias=False),
        # a server's batch decoding: the feed-forward's second projection
        dict(name="batch_down", op="product", rows=48, n=1536, k=7168, group=64, dtype="bfloat16", out="float32", bias=False),
        # the ragged rest of several prompts in one step, an output width that is no multiple of a tile
        dict(name="prompt_down", op="product", rows=1029, n=2056, k=8192, group=128, dtype="bfloat16", out="bfloat16", bias=True),
        # one token through a gated feed-forward's first two projections
        dict(name="token_gated", op="gated", rows=1, n=28672, k=4096, group=64, dtype="bfloat16", out="bfloat16", bias=False),
        # a long prompt's portion through the same: the largest share of a prompt's arithmetic
        dict(name="prompt_gated", op="gated", rows=2048, n=16384, k=2048, group=64, dtype="bfloat16", out="bfloat16", bias=False),
        # a model being loaded: the embedding matrix
        dict(name="load_head", op="quantize", n=VOCAB, k=2048, group=64, dtype="bfloat16"),
        # a matrix stored in 32 bits, of odd sizes
        dict(name="load_float32", op="quantize", n=1003, k=1357, group=32, dtype="float32"),
        # a prompt's tokens
        dict(name="embed_prompt", op="embed", rows=2048, n=VOCAB, k=2048, group=64),
        # a decode step of one request
        dict(name="embed_token", op="embed", rows=1, n=VOCAB, k=1024, group=32),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("product", "product", "product", "gated", "gated", "quantize", "embed"))
    group = rng.choice((32, 64, 128))
    k = _log_int(rng, 16, 16384)
    if rng.random() < 0.7:                       # most models' widths are whole vectors
        k = max(8, k // 8 * 8)
    if op == "quantize":
        return dict(op=op, n=_log_int(rng, 1, min(VOCAB, MOST_WEIGHTS // k)), k=k, group=group, dtype=rng.choice(("bfloat16", "float32")))
    if op == "embed":
        return dict(op=op, rows=_log_int(rng, 1, min(2048, 2048 * 2048 // k)), n=_log_int(rng, 16, min(VOCAB, MOST_WEIGHTS // k)), k=k, group=group)
    # a third decode steps of few requests, a third larger batches, a third portions of prompts
    rows = _log_int(rng, *rng.choice(((1, 16), (17, 128), (129, 2048))))
    n = _log_int(rng, 16, min(VOCAB, MOST_WEIGHTS // k, MOST_FLOPS // (2 * rows * k)))
    dtype = "float32" if rng.random() < 0.2 else "bfloat16"
    if dtype == "float32":
        rows = min(rows, 300)                    # (a yardstick engine: portions of prompts are short there)
    out = "float32" if dtype == "float32" else rng.choice(("bfloat16", "float32"))
    if op == "gated":
        return dict(op=op, rows=rows, n=max(16, n // 16 * 16), k=k, group=group, dtype=dtype, out=dtype, bias=rng.random() < 0.2)
    return dict(op=op, rows=rows, n=n, k=k, group=group, dtype=dtype, out=out, bias=rng.random() < 0.3)


# ---------------------------------------------------------------------------------------------------------- the inputs

def _inputs(case, seed):
    """The case's data from the seed alone."""
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    n, k, group = case["n"], case["k"], case["group"]
    if case["op"] == "quantize":
        w = torch.randn(n, k, generator=g, device=DEV) * 0.02
        return dict(w=w.to(getattr(torch, case["dtype"])))
    got = dict(levels=(torch.randn(n, k, generator=g, device=DEV) * 2.7).round().clamp(-8, 7).to(torch.int8))
    m = torch.randint(16, 32, (n, -(-k // group)), generator=g, device=DEV).float()
    sign = torch.randint(0, 2, m.shape, generator=g, device=DEV).float() * 2 - 1
    got["scales"] = (m * sign * 2.0 ** -12).bfloat16()         # matrices of random weights of 0.02: groups' maxima of some 0.05
    if case["op"] == "embed":
        got["tokens"] = torch.randint(0, n, (case["rows"],), generator=g, device=DEV, dtype=torch.int32)
        return got
    got["x"] = torch.randn(case["rows"], k, generator=g, device=DEV).to(getattr(torch, case["dtype"]))
    got["bias"] = torch.randn(n, generator=g, device=DEV) if case["bias"] else None
    return got


def prepare(case, seed):
    state = dict(case=case, **_inputs(case, seed))
    if own and "levels" in state:
        from fellm_b200 import ops
        state["w4"] = ops.pack_w4(state.pop("levels"), state.pop("scales"), case["group"])
    if case["op"] == "embed":
        state["y"] = torch.empty(case["rows"], case["k"], dtype=torch.float32, device=DEV)
    return state


# ------------------------------------------------------------------------------------------------------------ one pass

def _silu(z):
    return z / (1 + torch.exp(-z))


def _gated(z):
    """Columns are eight of the gate, eight of the up projection, and so on."""
    z = z.reshape(z.shape[0], -1, 2, 8)
    return (_silu(z[:, :, 0]) * z[:, :, 1]).reshape(z.shape[0], -1)


def _plain_quantize(w, group):
    """The scale: an eighth of the group's largest magnitude, rounded to five significant bits, negative where that
    magnitude is a positive element's, so that the extreme becomes level -8.  In 64 bits: a level is a rounded quotient."""
    n, k = w.shape
    v = torch.zeros(n, -(-k // group) * group, dtype=torch.float64, device=w.device)
    v[:, :k] = w
    v = v.reshape(n, -1, group)
    hi, lo = v.amax(-1, keepdim=True), v.amin(-1, keepdim=True)
    mant, expo = torch.frexp(torch.maximum(hi, -lo) / 8)
    s = torch.ldexp(torch.round(mant * 32), expo - 5)
    s = torch.where(hi > -lo, -s, s)
    q = torch.where(s == 0, torch.zeros_like(v), torch.round(v / s)).clamp(-8, 7)
    return (q * s).reshape(n, -1)[:, :k].to(torch.bfloat16)


def _plain(state):
    case = state["case"]
    if case["op"] == "quantize":
        return _plain_quantize(state["w"], case["group"])
    q, s = state["levels"], state["scales"]
    if case["op"] == "embed":
        at = state["tokens"].long()
        q, s = q[at], s[at]
    w = q.float() * s.float().repeat_interleave(case["group"], 1)[:, :case["k"]]
    if case["op"] == "embed":
        return w
    y = state["x"].float() @ w.T
    if state["bias"] is not None:
        y = y + state["bias"]
    if case["op"] == "gated":
        y = _gated(y)
    return y.to(getattr(torch, case["out"]))


def run(state):
    if not own:
        return _plain(state)
    from fellm_b200 import ops
    case = state["case"]
    if case["op"] == "quantize":
        return ops.dequantize_w4(ops.quantize_w4(state["w"], case["group"]))
    if case["op"] == "embed":
        return ops.embed_rows_w4(state["tokens"], state["w4"], state["y"])
    return ops.gemm_w4(state["x"], state["w4"], state["bias"], out_dtype=getattr(torch, case["out"]), swiglu=case["op"] == "gated")


def exact(case, seed):
    """The definitions, in 64 bits."""
    d = _inputs(case, seed)
    group, k = case["group"], case["k"]
    if case["op"] == "quantize":
        w = d["w"].double()
        out = torch.empty_like(w)
        for at in range(0, k, group):
            piece = w[:, at:at + group]
            big = piece.abs().max(1).values
            unit = torch.exp2(torch.floor(torch.log2(big.clamp(min=1e-300))) - 4)      # the fifth significant bit of the magnitude
            scale = torch.round(big / unit) * unit / 8
            scale = torch.where((piece == big[:, None]).any(1) & ~(piece == -big[:, None]).any(1), -scale, scale)[:, None]
            level = torch.round(piece / torch.where(scale == 0, torch.ones_like(scale), scale))
            out[:, at:at + group] = torch.minimum(torch.maximum(level, torch.full_like(level, -8)), torch.full_like(level, 7)) * scale
        return out
    rows = slice(None) if case["op"] != "embed" else d["tokens"].long()
    w = d["levels"][rows].double()
    for i in range(-(-k // group)):
        w[:, i * group:(i + 1) * group] *= d["scales"][rows][:, i:i + 1].double()
    if case["op"] == "embed":
        return w
    y = torch.mm(d["x"].double(), w.t())
    if d["bias"] is not None:
        y += d["bias"].double()
    if case["op"] == "gated":
        at = torch.arange(case["n"], device=DEV).reshape(-1, 16)
        gate, up = y[:, at[:, :8].reshape(-1)], y[:, at[:, 8:].reshape(-1)]
        y = gate * torch.sigmoid(gate) * up
    return y


def work(case):
    n, k, groups = case["n"], case["k"], -(-case["k"] // case["group"])
    size = {"bfloat16": 2, "float32": 4}
    if case["op"] == "quantize":                 # the matrix in, its values out
        return dict(bytes=n * k * (size[case["dtype"]] + 2), flops=4 * n * k)
    row = k / 2 + 2 * groups
    if case["op"] == "embed":
        return dict(bytes=int(case["rows"] * (row + 4 + 4 * k)), flops=case["rows"] * k)
    y = case["rows"] * (n // 2 if case["op"] == "gated" else n) * size[case["out"]]
    x = case["rows"] * k * size[case["dtype"]]
    return dict(bytes=int(n * row + x + y + (4 * n if case["bias"] else 0)), flops=2 * case["rows"] * n * k)
