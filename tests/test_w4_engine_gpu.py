"""Whole models with their matrices in four bits.

A level times its scale is a bfloat16 number, so a model in four bits means the same numbers as one whose matrices hold the
values of the four-bit ones: an engine with `weights="int4"` is compared with an engine of kept matrices into which those
values were written.  Both follow the plain implementation of that model within its design's limit (the tests of each design),
so they are within twice that of each other."""
from __future__ import annotations

import numpy as np
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
from fellm_b200.engine import GenParams, StepItem

DESIGNS = [(tiny, "A"), (tiny, "B"), (tiny, "C"), (robazen_util, "P"), (robazen_util, "R"), (samusun_util, "A"), (samusun_util, "C"),
           (meresun_util, "A"), (meresun_util, "B"), (nalizen_util, "A"), (nalizen_util, "B"), (vofezen_util, "A"), (vofezen_util, "B"),
           (petelix_util, "A"), (petelix_util, "B")]
IDS = [f"{u.__name__.replace('_util', '')}-{n}" for u, n in DESIGNS]


def _limit(util, dtype):
    return 2 * getattr(util, "LIMIT", {"float32": 2e-5, "bfloat16": 2.5e-2})[dtype]


def _hold_four_bit_values(eng, group):
    """Every matrix that the int4 engine would keep in four bits, as those values."""
    for part in eng.model.all_parts():
        for name in part.four_bit:
            w = part.w.get(name)
            if isinstance(w, torch.Tensor) and not getattr(w, "_held", False):
                w.copy_(ops.dequantize_w4(ops.quantize_w4(w.contiguous(), group), w.dtype))
                w._held = True                             # (a tied head's matrix is the embedding's)


def _engines(util, name, dtype, group, **opts):
    kept = util.make_engine(name, dtype, **opts)
    _hold_four_bit_values(kept, group)
    return kept, util.make_engine(name, dtype, weights="int4", weight_group=group, **opts)


def _rows(eng, toks, first):
    """Logits of every token: a portion, another beside a second request's, then one token at a time."""
    eng.add_request("a")
    eng.add_request("b")
    rows = [eng.step([StepItem("a", toks[:first], list(range(first)))])]
    rows.append(eng.step([StepItem("b", toks[:3], [2]), StepItem("a", toks[first:first + 9], list(range(9)))]))
    for t in range(first + 9, len(toks)):
        rows.append(eng.step([StepItem("a", [toks[t]], [0]), StepItem("b", [toks[t]], [0])]))
    eng.check_status()
    return torch.cat(rows).double()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,group", [("float32", 32), ("bfloat16", 64), ("bfloat16", 128)])
@pytest.mark.parametrize("util,name", DESIGNS, ids=IDS)
def test_every_design_with_its_matrices_in_four_bits(util, name, dtype, group):
    kept, four = _engines(util, name, dtype, group)
    names = [n for part in four.model.all_parts() for n in part.four_bit if isinstance(part.w.get(n), ops.W4)]
    assert len(names) >= 4 and isinstance(four.model.head.w["weight"], ops.W4) and isinstance(four.model.embedding.w["weight"], ops.W4)
    if getattr(four.model.head, "tied", False):
        assert four.model.head.w["weight"] is four.model.embedding.w["weight"]
    toks = [int(t) for t in np.random.default_rng(77).integers(0, four.spec.vocab_size, 38)]
    got, want = _rows(four, toks, 21), _rows(kept, toks, 21)
    got, want = got - got.mean(-1, keepdim=True), want - want.mean(-1, keepdim=True)
    scale = want.pow(2).mean().sqrt()
    off = (got - want).pow(2).mean(-1).sqrt() / scale
    assert float(off.max()) <= _limit(util, dtype), float(off.max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("util,name", [(tiny, "A"), (tiny, "C"), (meresun_util, "A")], ids=["lfm2-A", "lfm2-C", "meresun-A"])
def test_replayed_steps_are_the_launched_ones(util, name, dtype):
    """Decode steps from CUDA graphs, several requests together, through the scheduler."""
    outs = []
    for graphs in (False, True):
        eng = util.make_engine(name, dtype, weights="int4", weight_group=32, cuda_graphs=graphs, n_ubatch=16)
        rng = np.random.default_rng(5)
        prompts = [[int(t) for t in rng.integers(0, eng.spec.vocab_size, n)] for n in (30, 5, 17)]
        outs.append(eng.generate_batch(prompts, GenParams.greedy(12))[0])
        outs.append(eng.generate_batch(prompts, GenParams.greedy(12))[0])
    assert outs[0] == outs[1] == outs[2] == outs[3]


@pytest.mark.gpu
@pytest.mark.parametrize("requests", [24, 70, 128, 150])
@pytest.mark.parametrize("util,name", [(tiny, "A"), (tiny, "B"), (tiny, "C"), (meresun_util, "A")], ids=["lfm2-A", "lfm2-B", "lfm2-C", "meresun-A"])
def test_a_step_of_many_requests(util, name, requests, monkeypatch):
    """Decode steps of up to 128 requests, whose products hand norms on where the widths are multiples of 32, and of more."""
    opts = dict(max_requests=requests, max_tokens=requests * 64)
    kept, four = _engines(util, name, "bfloat16", 64, **opts)
    taken = []
    product = ops.gemm_w4
    monkeypatch.setattr(ops, "gemm_w4", lambda *a, **k: (taken.append(k.get("row_scale") is not None), product(*a, **k))[1])
    rng = np.random.default_rng(requests)
    first = rng.integers(0, four.spec.vocab_size, (requests, 3))
    then = rng.integers(0, four.spec.vocab_size, (4, requests))
    rows = []
    for eng in (four, kept):
        for r in range(requests):
            eng.add_request(f"r{r}")
        for lo in range(0, requests, 16):
            eng.step([StepItem(f"r{r}", [int(t) for t in first[r]], []) for r in range(lo, min(lo + 16, requests))])
        taken.clear()
        rows.append(torch.cat([eng.step([StepItem(f"r{r}", [int(step[r])], [0]) for r in range(requests)]) for step in then]).double())
        eng.check_status()
        if eng is four and util is tiny:                     # (the other designs' blocks norm their own inputs)
            assert any(taken) == (requests <= 128 and four.spec.hidden_size % 32 == 0)
    got, want = (x - x.mean(-1, keepdim=True) for x in rows)
    off = (got - want).pow(2).mean(-1).sqrt() / want.pow(2).mean().sqrt()
    assert float(off.max()) <= _limit(util, "bfloat16"), float(off.max())


@pytest.mark.gpu
def test_a_portion_is_the_same_tokens_one_by_one():
    eng = tiny.make_engine("B", "float32", weights="int4")
    toks = tiny.tokens("B", 40, 3)
    eng.add_request("whole"), eng.add_request("single")
    whole = eng.step([StepItem("whole", toks, list(range(40)))])
    single = torch.cat([eng.step([StepItem("single", [t], [0])]) for t in toks])
    ok, err, tol = tiny.close(whole, single, "float32")
    assert ok, (err, tol)


@pytest.mark.gpu
def test_the_command_line_runs_a_model_in_four_bits(capsys):
    from fellm_b200 import cli
    folder = tiny.model_folder("A")
    assert cli.main(["run", folder, "--prompt", "5,17,3", "--max-tokens", "6", "--temperature", "0", "--repetition-penalty", "1", "--weights", "int4",
                     "--weight-group", "32", "--page-tokens", "16", "--ctx-size", "256"]) == 0
    said = [int(t) for t in capsys.readouterr().out.split()]
    eng = tiny.make_engine("A", "bfloat16", weights="int4", weight_group=32)
    assert said == list(eng.generate([5, 17, 3], GenParams.greedy(6)))


def test_options_that_are_refused():
    from fellm_b200.config import ConfigError, EngineOptions
    for bad in (dict(weights="int3"), dict(weight_group=48), dict(weights="int4", weight_group=0)):
        with pytest.raises(ConfigError):
            EngineOptions(**bad).validate()
    EngineOptions(weights="int4", weight_group=128).validate()
