"""What a plan says of a step's contexts, and what it does not, in the attention over pages of 8 bits."""

from __future__ import annotations

import pytest
import torch

from liteinfer_b200 import ops
from liteinfer_b200.parts.context import AttentionPlan
from test_int8_gpu import DEVICE, _batch, _generator, _pages

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("prefill,decode", [(0, 1338), (131, 0)])
def test_a_bound_that_is_not_known_bounds_nothing(prefill, decode):
    """A plan that knows the longest context of its single tokens alone, or of its portions alone, in a step of both that reads its pages back."""
    sequences = [(100, 31), (1337, 1)]
    heads, kv_heads, dim, page = 8, 2, 64, 8
    positions, seq, table, starts, context, total = _batch(sequences, page, 1)
    pages = _pages(total, kv_heads, page, dim, 1)
    q = torch.randn((32, heads * dim), generator=_generator(2), device=DEVICE)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEVICE)
    outs = []
    for bounds in ((prefill, decode), (131, 1338)):
        plan = AttentionPlan(1, ints(1), ints(31), None, 1, ints(0), 31, bounds[1], bounds[0])
        out = torch.empty_like(q)
        ops.paged_attention_int8(q, q.stride(0), out, pages, table, starts, context, 2, 31, heads, kv_heads, dim, dim ** -0.5, plan=plan)
        outs.append(out)
    assert torch.equal(*outs)
