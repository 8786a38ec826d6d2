"""Loading with weights in 8 bits gives back what the weights took before."""

from __future__ import annotations

import gc

import pytest
import torch

import tiny_configs
from liteinfer_b200.config.engine_config import EngineConfig
from liteinfer_b200.engine.core import EngineCore
from liteinfer_b200.weights.random_init import write_random_model

pytestmark = pytest.mark.gpu


def test_weights_in_8_bits_leave_more_memory_for_pages(tmp_path, monkeypatch):
    config = dict(tiny_configs.TINY_D, hidden_size=1024, intermediate_size=4096, num_hidden_layers=6, num_attention_heads=16, num_key_value_heads=8)
    folder = write_random_model(config, tmp_path / "model", 1)
    held = {}

    def pages(core, model):
        held[core.config.weight_dtype] = (torch.cuda.memory_reserved(), model.weight_bytes())
        return 8

    monkeypatch.setattr(EngineCore, "_num_pages", pages)
    for kind in (None, "int8"):
        gc.collect()
        torch.cuda.empty_cache()
        before = torch.cuda.memory_reserved()
        core = EngineCore(EngineConfig(model=str(folder), dtype="bfloat16", block_size=16, max_num_seqs=2, max_model_len=64, weight_dtype=kind))
        core.load()
        held[kind] = (held[kind][0] - before, held[kind][1])
        del core
    (wide, wide_bytes), (narrow, narrow_bytes) = held[None], held["int8"]
    # Six layers of 15.7 million numbers.  The memory that is taken from the device when pages are counted falls with the weights, up to what the
    # allocator's pieces (20 MB) leave unused.
    assert narrow_bytes < wide_bytes - 90e6 and narrow < wide - 60e6, held
