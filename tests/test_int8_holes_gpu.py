"""Blocks of a table that name no page (-1), among those that a query sees: their keys are not there, whichever kernel takes the call."""

from __future__ import annotations

import math

import pytest
import torch

import int8_bounds
from liteinfer_b200 import ops
from liteinfer_b200.parts.context import AttentionPlan
from test_int8_gpu import DEVICE, TYPES, _batch, _generator, _pages

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [0.125, 12.0])
@pytest.mark.parametrize("mask", [dict(), dict(softcap=3.0), dict(sink=True)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (32, 8, 128)])
def test_pages_that_there_are_none_of(heads, kv_heads, dim, mask, scale, dtype):
    """Blocks in the middle, whole steps of 128 keys, the first ones, every other one, and all behind the queries."""
    page = 16
    sequences = [(700, 90), (700, 1), (4000, 3), (300, 40), (64, 1), (64, 2), (48, 33)]
    holes = [range(3, 7), range(0, 30), range(16, 200), range(1, 18, 2), range(0, 4), range(0, 4), ()]
    positions, seq, table, starts, context, total = _batch(sequences, page, 1)
    pages = _pages(total, kv_heads, page, dim, 1)
    q = torch.randn((positions.numel(), heads * dim), generator=_generator(3), device=DEVICE).to(dtype)
    if mask.get("sink"):
        mask = dict(sink=torch.randn(heads, generator=_generator(5), device=DEVICE))
    given = table.clone()
    for b, gone in enumerate(holes):
        given[b, list(gone)] = -1
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEVICE)
    single, several = [b for b, s in enumerate(sequences) if s[1] == 1], [b for b, s in enumerate(sequences) if s[1] > 1]
    plan = AttentionPlan(len(single), ints(single), starts[ints(single).long()], None, len(several), ints(several), 90, 701, 4003)
    out = torch.full_like(q, math.nan)
    scale = scale / math.sqrt(dim)
    ops.paged_attention_int8(q, q.stride(0), out, pages, given, starts, context, len(sequences), 90, heads, kv_heads, dim, scale, plan=plan, **mask)
    for b, (held, new) in enumerate(sequences):
        # All holes lie behind the queries, so the formula over what is left, that much further ahead, is the formula.
        ids = torch.tensor([int(p) for p in given[b, :-(-(held + new) // page)] if p >= 0], device=DEVICE)
        dropped = page * len(list(holes[b]))
        k, v = ((pool[ids].double() * s[ids].double()[..., None, None]).transpose(1, 2).flatten(0, 1)[:held + new - dropped]
                for pool, s in ((pages.k, pages.k_scale), (pages.v, pages.v_scale)))
        at = int(starts[b])
        want, bound = int8_bounds.attention("single" if new == 1 else "portion", dtype, q[at:at + new].double().view(new, heads, dim), k, v, scale, heads,
                                            kv_heads, held - dropped, v_scales=pages.v_scale[ids], **mask)
        off = (out[at:at + new].double().view(new, heads, dim) - want).abs() / bound
        assert bool((off <= 1).all()), (b, float(off.max()))


@pytest.mark.parametrize("dtype", TYPES)
def test_a_sequence_without_any_page_is_zeros(dtype):
    sequences = [(700, 90), (700, 1), (4000, 3)]
    positions, seq, table, starts, context, total = _batch(sequences, 16, 1)
    pages = _pages(total, 2, 16, 64, 1)
    q = torch.randn((positions.numel(), 8 * 64), generator=_generator(3), device=DEVICE).to(dtype)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEVICE)
    plan = AttentionPlan(1, ints(1), ints(90), None, 2, ints(0, 2), 90, 701, 4003)
    out = torch.full_like(q, math.nan)
    ops.paged_attention_int8(q, q.stride(0), out, pages, torch.full_like(table, -1), starts, context, 3, 90, 8, 2, 64, 0.125, plan=plan)
    assert int(out.count_nonzero()) == 0
