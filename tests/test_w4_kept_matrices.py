"""Which of a model's matrices are held in four bits and which stay, by the tensors' names: every tensor is filled with a number of its own, and what
is brought into the form is asked which numbers it holds."""
from __future__ import annotations

import re

import pytest
import torch

import meresun_util
import nalizen_util
import petelix_util
import robazen_util
import samusun_util
import tiny
import vofezen_util
from fellm_b200 import ops
from fellm_b200.config.registry import config_from_dict
from fellm_b200.models.model import build_model
from fellm_b200.weights.loader import bind_tensors
from fellm_b200.weights.random_init import random_tensors

# routers and experts, convolutions, side inputs and tables of vectors; the logits of a write strength (b), of a decay (a, or the factors a1 a2, w1 w2) and
# of a gate a head (left.g); the factors of a gate (g1, g2); what a latent's keys and values are made with
STAY = {
    "tiny": r"conv\.conv",
    "robazen": r"mix\.[qkv]\.conv|mix\.b$|mix\.a$|mix\.[ag][12]$|mix\.left\.g$|mix\.right\.(u|w1|w2)$|loop\.step",
    "samusun": r"mlp\.e\d+\.|mlp\.router|loop\.step",
    "meresun": r"mix\.u[kv]$|mlp\.e\d+\.|mlp\.router|side\.",
    "nalizen": r"mlp\.e\d+\.|mlp\.router|side\.",
    "vofezen": r"mix\.u[kv]$|mlp\.e\d+\.|mlp\.router",
    "petelix": r"mlp\.e\d+\.|mlp\.router",
}
DESIGNS = [(u, n) for u in (tiny, robazen_util, samusun_util, meresun_util, nalizen_util, vofezen_util, petelix_util) for n in sorted(u.CONFIGS) if n not in "WM"]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("util,name", DESIGNS, ids=[f"{u.__name__.replace('_util', '')}-{n}" for u, n in DESIGNS])
def test_matrices_that_stay(util, name, dtype, monkeypatch):
    arch, config = config_from_dict(util.CONFIGS[name][0])
    model = build_model(arch.build_spec(config), dtype)
    tensors = random_tensors(model, 3, torch.float32)
    matrices = [n for n, t in tensors.items() if t.dim() == 2]
    held = {}
    number = {n: 0.25 + i // 128 + (i % 128) * 2.0 ** -7 if i < 128 else 2.0 ** (1 + i // 128) * (1 + (i % 128) * 2.0 ** -7) for i, n in enumerate(matrices)}
    by_number = {torch.tensor(v).to(torch.bfloat16).item(): n for n, v in number.items()}
    assert len(by_number) == len(matrices)
    for n in matrices:
        tensors[n].fill_(torch.tensor(number[n]).to(torch.bfloat16).item())
    bind_tensors(model, tensors, "cpu")

    def quantize(w, group):
        rows = [by_number[v] for v in w[:, 0].tolist() if v]
        assert all(len(set(r.tolist())) == 1 for r in w)
        for n in rows:
            held[n] = held.get(n, 0) + 1
        q, s = ops._w4_room(w.shape[0], w.shape[1], group, "cpu")
        return ops.W4(q, s, w.shape[0], w.shape[1], group)

    monkeypatch.setattr(ops, "quantize_w4", quantize)
    model.quantize(32)
    stay = re.compile(STAY[util.__name__.replace("_util", "")])
    assert {n for n in matrices if n not in held} == {n for n in matrices if stay.search(n)}
    assert all(held[n] == tensors[n].shape[0] for n in held), "every row once"


@pytest.mark.parametrize("decay,gate", [("head", "silu"), ("channel", "silu"), ("head", "sigmoid_lowrank"), ("channel", "sigmoid_lowrank")])
def test_the_rows_of_a_delta_mixer_that_stay(decay, gate, monkeypatch):
    """They are there as they were, bit by bit, and where the mixer looks for them."""
    from fellm_b200.parts.gated_delta import GatedDelta
    part = GatedDelta(dtype="bfloat16", size=40, heads=6, kv_heads=3, key_dim=5, value_dim=7, taps=3, norm_eps=1e-6, decay=decay, gate=gate)
    g = torch.Generator().manual_seed(1)
    tensors = {n: torch.randn(d.made_shape(), generator=g).to(torch.bfloat16 if len(d.made_shape()) == 2 and "conv" not in n else torch.float32)
               for n, d in part.decls.items()}
    part.bind(dict(tensors))
    whole, off, rows = part.w["in.weight"].clone(), dict(part.off), dict(part.rows)
    taken = []
    monkeypatch.setattr(ops, "quantize_w4", lambda w, group: (taken.append(w.clone()), ops.W4(*ops._w4_room(*w.shape, group, "cpu"), *w.shape, group))[1])
    part.quantize(64)
    first = torch.cat([tensors[f"{n}.weight"] for n in ("qkvg" if gate == "silu" else "qkv")])
    padded = torch.cat([first, first.new_zeros(-first.shape[0] % 16, 40)])
    assert len(taken) == 2 and torch.equal(taken[0], padded) and torch.equal(taken[1], tensors["o.weight"])
    kept = part.w["logits.weight"]
    assert kept.untyped_storage().nbytes() == kept.numel() * 2, "the whole matrix's memory is held by the rows that stay"
    assert kept.dtype == torch.bfloat16 and kept.shape[0] % 16 == 0 and "in.weight" not in part.w
    for name in ("b", "a") + (("g",) if gate != "silu" else ()):
        at = part.logits_off[name]
        assert torch.equal(kept[at:at + rows[name]], whole[off[name]:off[name] + rows[name]])
