"""What is no number stays visible in the attention over pages of 8 bits, however many blocks share a tile's keys."""

from __future__ import annotations

import math

import pytest
import torch

import int8_bounds
from liteinfer_b200 import ops
from liteinfer_b200.parts.context import AttentionPlan
from test_int8_gpu import DEVICE, _batch, _generator, _pages

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float32]
HEADS, KV_HEADS, PAGE = 8, 2, 16


def _attend(held, new, dim, dtype, change, splits=None, sink=None):
    """`new` queries behind `held` keys (bad numbers by `change(q, pages, table)`) -> ([new, kv heads, group * dim], the formula and how far
    from it numbers may be)."""
    positions, seq, table, starts, context, total = _batch([(held, new)], PAGE, 3)
    pages = _pages(total, KV_HEADS, PAGE, dim, 3)
    q = torch.randn((new, HEADS * dim), generator=_generator(4), device=DEVICE).to(dtype)
    change(q, pages, table[0].long())
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEVICE)
    single = new == 1
    plan = AttentionPlan(int(single), ints(0), ints(0), None, int(not single), ints(0), 0 if single else new, held + 1 if single else 0,
                         0 if single else held + new)
    out = torch.full_like(q, 7.0)
    ops.paged_attention_int8(q, q.stride(0), out, pages, table, starts, context, 1, new, HEADS, KV_HEADS, dim, dim ** -0.5, plan=plan,
                             decode_splits=splits, sink=sink)
    ids = table[0].long()
    k, v = ((pool[ids].double() * s[ids].double()[..., None, None]).transpose(1, 2).flatten(0, 1)[:held + new]
            for pool, s in ((pages.k, pages.k_scale), (pages.v, pages.v_scale)))
    mask = {} if sink is None else dict(sink=sink)
    want, bound = int8_bounds.attention("single" if single else "portion", dtype, q.nan_to_num().double().view(new, HEADS, dim), k.nan_to_num(), v.nan_to_num(),
                                        dim ** -0.5, HEADS, KV_HEADS, held, v_scales=pages.v_scale[ids].nan_to_num(), **mask)
    return out.view(new, KV_HEADS, -1), want.reshape(new, KV_HEADS, -1), bound.reshape(new, KV_HEADS, -1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("with_sink", [False, True])
@pytest.mark.parametrize("held,new", [(4000, 5), (4000, 1), (100, 5), (100, 1), (1500, 60)])
def test_a_query_that_is_no_number(held, new, dim, dtype, with_sink):
    sink = torch.randn(HEADS, generator=_generator(5), device=DEVICE) if with_sink else None

    def change(q, pages, table):
        q[new - 1, 2 * dim + 3] = math.nan              # the third head's, of the first KV head
    out, want, bound = _attend(held, new, dim, dtype, change, sink=sink)
    spoilt = torch.zeros(out.shape, dtype=torch.bool, device=DEVICE)
    spoilt[new - 1, 0, 2 * dim:3 * dim] = True
    assert bool((out.isnan() == spoilt).all()) and bool(((out.double() - want).abs() <= bound)[~spoilt].all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("with_sink", [False, True])
@pytest.mark.parametrize("new", [5, 1])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("share", [(0, 0.25), (0.25, 0.5), (0.75, 1), (0.5, 1), (0, 1), (0.1, 0.11)])
def test_pages_that_are_no_numbers_over_a_whole_share(share, which, new, dim, dtype, with_sink):
    """Of one KV head, the scales of a part of the sequence's pages (all that one block of those that share the keys sees, or two)."""
    held = 4096 - new
    sink = torch.randn(HEADS, generator=_generator(5), device=DEVICE) if with_sink else None

    def change(q, pages, table):
        first, last = (int(f * table.numel()) for f in share)
        getattr(pages, which + "_scale")[table[first:last], 1] = math.nan
    out, want, bound = _attend(held, new, dim, dtype, change, sink=sink)
    assert bool(out[:, 1].isnan().all()) and bool(((out.double() - want).abs() <= bound)[:, 0].all())
