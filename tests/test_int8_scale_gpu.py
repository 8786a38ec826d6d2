"""Scores scaled by numbers of either sign, and by none, in the attention over pages of 8 bits."""

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
@pytest.mark.parametrize("scale", [-0.125, 0.0, 0.125])
@pytest.mark.parametrize("mask", [dict(), dict(window=100), dict(softcap=3.0), dict(chunk=64)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (32, 8, 128)])
def test_scales_of_either_sign(heads, kv_heads, dim, mask, scale, dtype):
    sequences, page = [(0, 300), (700, 1), (4000, 3), (130, 1), (700, 90)], 16
    positions, seq, table, starts, context, total = _batch(sequences, page, 1)
    pages = _pages(total, kv_heads, page, dim, 1)
    q = (torch.randn((positions.numel(), heads * dim), generator=_generator(3), device=DEVICE) * 1.5).to(dtype)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEVICE)
    plan = AttentionPlan(2, ints(1, 3), starts[ints(1, 3).long()], None, 3, ints(0, 2, 4), 300, 701, 4003)
    out = torch.full_like(q, math.nan)
    ops.paged_attention_int8(q, q.stride(0), out, pages, table, starts, context, len(sequences), 300, heads, kv_heads, dim, scale, plan=plan, **mask)
    for b, (held, new) in enumerate(sequences):
        ids = table[b, :-(-(held + new) // page)].long()
        k, v = ((pool[ids].double() * s[ids].double()[..., None, None]).transpose(1, 2).flatten(0, 1)[:held + new]
                for pool, s in ((pages.k, pages.k_scale), (pages.v, pages.v_scale)))
        at = int(starts[b])
        want, bound = int8_bounds.attention("single" if new == 1 else "portion", dtype, q[at:at + new].double().view(new, heads, dim), k, v, scale, heads,
                                            kv_heads, held, v_scales=pages.v_scale[ids], **mask)
        off = (out[at:at + new].double().view(new, heads, dim) - want).abs() / bound
        assert bool((off <= 1).all()), (b, float(off.max()))
