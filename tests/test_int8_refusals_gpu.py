"""Arguments that would have a kernel over pages of 8 bits read behind their ends are refused before anything is launched."""

from __future__ import annotations

import pytest
import torch

from liteinfer_b200 import ops
from liteinfer_b200.ops import kernels
from test_int8_gpu import DEVICE, _pages

pytestmark = pytest.mark.gpu


def test_attention_refuses_what_is_too_short():
    pages = _pages(4, 2, 16, 64, 1)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEVICE)
    q = torch.zeros((3, 4 * 64), device=DEVICE)
    good = dict(q=q, q_row_stride=256, out=q.clone(), pages=pages, block_table=ints(0, 1)[None], query_start_loc=ints(0, 3), context_lens=ints(3),
                num_seqs=1, max_q_len=3, heads=4, kv_heads=2, head_dim=64, scale=0.1)
    ops.paged_attention_int8(**good)
    before = kernels.launch_count
    for bad in (dict(q=q[:, :192]), dict(q=q[:, :128], q_row_stride=128), dict(num_seqs=2), dict(query_start_loc=ints(0)),
                dict(context_lens=ints()), dict(num_seqs=2, context_lens=ints(3, 3), query_start_loc=ints(0, 3, 3)), dict(block_table=ints(0, 1)[None][:0])):
        with pytest.raises(ValueError):
            ops.paged_attention_int8(**dict(good, **bad))
    assert kernels.launch_count == before
