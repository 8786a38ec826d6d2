"""How many pages of 8 bits memory affords: what a step needs beside them is left free."""

from __future__ import annotations

import pytest
import torch

from liteinfer_b200 import ops
from liteinfer_b200.cache.manager import CacheManager
from liteinfer_b200.config.engine_config import EngineConfig
from liteinfer_b200.engine.core import EngineCore
from liteinfer_b200.weights.loader import load_model


@pytest.mark.parametrize("int8", [True, False])
def test_pages_leave_room_for_the_attentions_work_space(model_dirs, monkeypatch, int8):
    """A device of 12 GB, 256 requests of up to 32,768 tokens: a step may spread as many contexts as its work space holds, and graphs keep one of their
    own."""
    model, _ = load_model(model_dirs["tiny_d"], torch.bfloat16, "cpu")
    model.hold_in_int8(False, int8)
    total = 12 << 30
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda device=None: (total, total))
    core = EngineCore(EngineConfig(model=str(model_dirs["tiny_d"]), dtype="bfloat16", device="cpu", max_num_seqs=256, max_model_len=32768, block_size=16,
                                   gpu_memory_utilization=0.5, max_num_batched_tokens=512))
    core.device = torch.device("cuda:0")
    pages = core._num_pages(model)
    per_page = CacheManager.bytes_per_page_for(model.cache_needs(), model.schedule, 16, torch.bfloat16)
    assert pages < 256 * 2048                    # memory decides
    left = total // 2 - pages * per_page
    heads, kv_heads, dim = 4, 2, 64
    work = ops.attention_int8_work(256, 32768, 512, heads, kv_heads, dim, 16, torch.bfloat16)
    assert work > 1 << 29
    # Without an 8-bit cache nothing is held back beyond the activations' allowance.
    assert (left >= 2 * work) if int8 else (left < work)
