"""Options given by position keep their places."""
from __future__ import annotations

from dataclasses import fields

from fellm_b200.config import EngineOptions


def test_options_by_position():
    opts = EngineOptions("float32", 4096, 1024, 256, True, 32, 8, 512, 0.5, 1 << 20, False, "cuda:1").validate()
    assert (opts.dtype, opts.n_ctx, opts.n_batch, opts.n_ubatch, opts.ctx_past_model, opts.page_tokens, opts.max_requests, opts.max_tokens,
            opts.kv_memory_fraction, opts.kv_device_budget, opts.cuda_graphs, opts.device) == (
        "float32", 4096, 1024, 256, True, 32, 8, 512, 0.5, 1 << 20, False, "cuda:1")
    assert (opts.weights, opts.weight_group) == ("kept", 64)
    assert [f.name for f in fields(EngineOptions)][-2:] == ["weights", "weight_group"]
