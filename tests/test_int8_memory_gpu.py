"""What serving in 8 bits asks of the device's memory."""

from __future__ import annotations

import pytest
import torch

import int8_bounds
from liteinfer_b200 import ops
from liteinfer_b200.ops import int8, kernels
from liteinfer_b200.parts.context import AttentionPlan
from test_int8_gpu import DEVICE, MIXED, SINGLES, TYPES, _batch, _check_attention, _generator, _pages

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("planned", [True, False])
def test_a_long_context_beside_short_ones_takes_a_bounded_work_space(planned):
    """One portion behind 40,000 tokens and forty behind a few: spread out as wide as the longest they would be 6.7 GB."""
    heads, kv_heads, dim, page, dtype = 8, 8, 128, 16, torch.bfloat16
    sequences = [(7, 3)] * 20 + [(40000, 5)] + [(30 + i, 4) for i in range(20)]
    positions, seq, table, starts, context, total = _batch(sequences, page, 1)
    pages = _pages(total, kv_heads, page, dim, 1)
    q = torch.randn((positions.numel(), heads * dim), generator=_generator(2), device=DEVICE).to(dtype)
    out = torch.full_like(q, float("nan"))
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEVICE)
    plan = AttentionPlan(0, ints([]), ints([]), None, len(sequences), ints(list(range(len(sequences)))), 5, 0, 40005) if planned else None
    kernels.scratch_for(DEVICE)                 # (the process's, made at the first call of all)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    ops.paged_attention_int8(q, q.stride(0), out, pages, table, starts, context, len(sequences), 5, heads, kv_heads, dim, dim ** -0.5, plan=plan)
    most = ops.attention_int8_work(len(sequences), 40005, q.shape[0], heads, kv_heads, dim, page, dtype)
    assert torch.cuda.max_memory_allocated() - before <= most + (1 << 21) and most <= int8.WORK_BYTES + 4096
    for b, (held, new) in enumerate(sequences):
        ids = table[b, :-(-(held + new) // page)].long()
        k, v = ((pool[ids].double() * s[ids].double()[..., None, None]).transpose(1, 2).flatten(0, 1)[:held + new]
                for pool, s in ((pages.k, pages.k_scale), (pages.v, pages.v_scale)))
        at = int(starts[b])
        want, bound = int8_bounds.attention("portion", dtype, q[at:at + new].double().view(new, heads, dim), k, v, dim ** -0.5, heads, kv_heads, held)
        assert bool(((out[at:at + new].double().view(new, heads, dim) - want).abs() <= bound).all()), b


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("room", [1, 200_000])
@pytest.mark.parametrize("layout", [(8, 2, 64, 16), (7, 1, 128, 32), (9, 3, 80, 16), (2, 1, 64, 5), (40, 2, 64, 8)])
def test_as_many_sequences_at_a_time_as_there_is_room_for(monkeypatch, layout, room, dtype):
    """Sequences one by one, or a few at a time: portions and single tokens, spread out or read back, with a plan and without."""
    monkeypatch.setattr(int8, "WORK_BYTES", room)
    _check_attention(MIXED + SINGLES, *layout, dtype)
    _check_attention(MIXED, *layout, dtype, planned=False)
    _check_attention(MIXED + SINGLES, *layout, dtype, window=40, keep_first=7)


def test_portions_and_single_tokens_take_their_work_spaces_in_turn(monkeypatch):
    """Behind kept first keys a step's portions are spread out and its single tokens' pages read back: one work space at a time."""
    monkeypatch.setattr(int8, "WORK_BYTES", 200_000_000)
    heads, kv_heads, dim, page, dtype = 8, 8, 128, 16, torch.bfloat16
    sequences = [(20000, 5)] * 6 + [(20000, 1)] * 6
    positions, seq, table, starts, context, total = _batch(sequences, page, 1)
    pages = _pages(total, kv_heads, page, dim, 1)
    q = torch.randn((positions.numel(), heads * dim), generator=_generator(2), device=DEVICE).to(dtype)
    out = torch.empty_like(q)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEVICE)
    plan = AttentionPlan(6, ints(list(range(6, 12))), ints(list(range(30, 36))), None, 6, ints(list(range(6))), 5, 20001, 20005)
    kernels.scratch_for(DEVICE)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    ops.paged_attention_int8(q, q.stride(0), out, pages, table, starts, context, 12, 5, heads, kv_heads, dim, dim ** -0.5, window=15000, keep_first=4, plan=plan)
    most = ops.attention_int8_work(12, 20005, q.shape[0], heads, kv_heads, dim, page, dtype)
    assert torch.cuda.max_memory_allocated() - before <= most + (1 << 23), (torch.cuda.max_memory_allocated() - before, most)
