"""What the operators over pages of 8 bits read of one another's results: calls one behind the other on a stream, without anything between
them, against the same calls with the device waited for after each."""

from __future__ import annotations

import pytest
import torch

import plain_int8 as plain
from liteinfer_b200 import ops
from liteinfer_b200.parts.context import AttentionPlan
from test_int8_gpu import DEVICE, _batch, _copy, _generator, _pages

pytestmark = pytest.mark.gpu


def _ints(*values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("planned", [False, True])
@pytest.mark.parametrize("between", ["nothing", "a reading", "a product"])
@pytest.mark.parametrize("held,new", [(30, 40), (15, 2), (700, 2500)])
def test_the_last_of_several_appended_tokens_sees_all_of_them(held, new, between, planned, dtype):
    """Several tokens of a sequence are appended, over a page's end, and the last of them alone is attended: every page that it sees has been
    written by the append ahead."""
    heads, kv_heads, dim, page = 8, 8, 64, 16
    positions, seq, table, _, context, total = _batch([(held, new)], page, 1)
    plan = AttentionPlan(1, _ints(0), _ints(0), None, 0, None, 0, held + new, 0) if planned else None
    x = torch.randn((2, 64), generator=_generator(7), device=DEVICE).to(dtype)
    weight = ops.quantise_weight(torch.randn((96, 64), generator=_generator(8), device=DEVICE).to(dtype))
    read = [torch.empty((1, table.shape[1], kv_heads, page, dim), dtype=dtype, device=DEVICE) for _ in range(2)]

    def run(qkv, pages, wait):
        out = torch.empty((1, heads * dim), dtype=dtype, device=DEVICE)
        ops.rope_kv_write_int8(qkv, positions, seq, table, pages, None, heads, kv_heads, dim, 0)
        if wait:
            torch.cuda.synchronize()
        if between == "a reading":
            ops.read_pages_int8(pages, table, context, *read)
        if between == "a product":
            ops.linear_int8(x, weight)
        ops.paged_attention_int8(qkv[-1:], qkv.stride(0), out, pages, table, _ints(0, 1), context, 1, 1, heads, kv_heads, dim, dim ** -0.5, plan=plan)
        return out

    for turn in range(6):
        start = _pages(total, kv_heads, page, dim, turn)
        qkv = torch.randn((new, (heads + 2 * kv_heads) * dim), generator=_generator(100 + turn), device=DEVICE).to(dtype)
        together, apart = _copy(start), _copy(start)
        torch.cuda.synchronize()
        got, want = run(qkv.clone(), together, False), run(qkv.clone(), apart, True)
        assert torch.equal(got, want) and torch.equal(together.k, apart.k) and torch.equal(together.v_scale, apart.v_scale)
        ids = table[0].long()
        k, v = ((pool[ids].double() * s[ids].double()[..., None, None]).transpose(1, 2).flatten(0, 1)[:held + new]
                for pool, s in ((apart.k, apart.k_scale), (apart.v, apart.v_scale)))
        formula, _ = plain.attention(qkv[-1:, :heads * dim].double().view(1, heads, dim), k, v, dim ** -0.5, heads, kv_heads, held + new - 1)
        # (rounded to 8 bits, or sums of 32; what is rounded on the way is held more closely by the tests of the attention)
        assert float((got.double().view(1, heads, dim) - formula).norm() / formula.norm()) <= (2.0 ** -7 if dtype is torch.bfloat16 else 1e-5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_single_tokens_right_behind_their_append(dtype):
    """`after_append`, where it holds: one token of each sequence was appended, in new pages and old ones."""
    heads, kv_heads, dim, page = 8, 2, 64, 16
    sequences = [(0, 1), (15, 1), (16, 1), (4000, 1), (0, 1), (47, 1), (800, 1)]
    positions, seq, table, starts, context, total = _batch(sequences, page, 2)
    rows = _ints(*range(len(sequences)))
    plan = AttentionPlan(len(sequences), rows, rows, None, 0, None, 0, 4001, 0)
    for turn in range(6):
        start = _pages(total, kv_heads, page, dim, turn)
        qkv = torch.randn((len(sequences), (heads + 2 * kv_heads) * dim), generator=_generator(50 + turn), device=DEVICE).to(dtype)
        outs = []
        for ahead in (True, False):
            pages, mine = _copy(start), qkv.clone()
            out = torch.empty((len(sequences), heads * dim), dtype=dtype, device=DEVICE)
            torch.cuda.synchronize()
            ops.rope_kv_write_int8(mine, positions, seq, table, pages, None, heads, kv_heads, dim, 0)
            if not ahead:
                torch.cuda.synchronize()
            ops.paged_attention_int8(mine, mine.stride(0), out, pages, table, starts, context, len(sequences), 1, heads, kv_heads, dim, 0.125,
                                     plan=plan, after_append=ahead)
            outs.append(out)
        assert torch.equal(*outs)
