"""Models with gated delta mixers whose matrices are in four bits: two products for a mixer's input."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import robazen_util
from fellm_b200.engine import GenParams, StepItem


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["P", "R", "S"])
def test_replayed_steps_are_the_launched_ones(name, dtype):
    outs = []
    for graphs in (False, True):
        eng = robazen_util.make_engine(name, dtype, weights="int4", weight_group=32, cuda_graphs=graphs, n_ubatch=16)
        rng = np.random.default_rng(5)
        prompts = [[int(t) for t in rng.integers(0, eng.spec.vocab_size, n)] for n in (30, 5, 17)]
        for _ in range(2):
            outs.append(eng.generate_batch(prompts, GenParams.greedy(12))[0])
    assert outs[0] == outs[1] == outs[2] == outs[3]


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["P", "R"])
def test_a_portion_is_the_same_tokens_one_by_one(name):
    eng = robazen_util.make_engine(name, "float32", weights="int4", weight_group=32)
    toks = robazen_util.tokens(name, 40, 3)
    eng.add_request("whole"), eng.add_request("single")
    whole = eng.step([StepItem("whole", toks, list(range(40)))])
    single = torch.cat([eng.step([StepItem("single", [t], [0])]) for t in toks])
    # both follow the plain implementation within the design's limit
    assert robazen_util.distance(whole, single) <= 2 * robazen_util.LIMIT["float32"]
