"""Single tokens over pages of 8 bits to the error of what their kernel rounds, and steps of portions and single tokens as the engine launches
them: an append, and both attentions behind it."""

from __future__ import annotations

import math

import pytest
import torch

import int8_bounds
from liteinfer_b200 import ops
from liteinfer_b200.parts.context import AttentionPlan
from test_int8_gpu import DEVICE, SINGLES, TYPES, _batch, _copy, _generator, _pages, _with_sink

pytestmark = pytest.mark.gpu


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _plan(sequences, starts):
    single, several = [b for b, s in enumerate(sequences) if s[1] == 1], [b for b, s in enumerate(sequences) if s[1] > 1]
    longest = lambda which: max([sum(sequences[b]) for b in which], default=0)
    return AttentionPlan(len(single), _ints(single), starts[_ints(single).long()], None, len(several), _ints(several),
                         max([sequences[b][1] for b in several], default=0), longest(single), longest(several))


def _hold(out, q, pages, table, starts, sequences, heads, kv_heads, dim, page, scale, dtype, **mask):
    """Every sequence's rows of `out` to the formula's bound."""
    for b, (held, new) in enumerate(sequences):
        ids = table[b, :-(-(held + new) // page)].long()
        k, v = ((pool[ids].double() * s[ids].double()[..., None, None]).transpose(1, 2).flatten(0, 1)[:held + new]
                for pool, s in ((pages.k, pages.k_scale), (pages.v, pages.v_scale)))
        at = int(starts[b])
        want, bound = int8_bounds.attention("single" if new == 1 else "portion", dtype, q[at:at + new, :heads * dim].double().view(new, heads, dim), k, v,
                                            scale, heads, kv_heads, held, v_scales=pages.v_scale[ids], **mask)
        off = (out[at:at + new].double().view(new, heads, dim) - want).abs() / bound
        assert bool((off <= 1).all()), (b, float(off.max()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mask", [dict(), dict(window=40), dict(chunk=48), dict(softcap=3.0), dict(sink=True), dict(window=100, softcap=2.0, sink=True)])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 4, 64, 16), (32, 8, 128, 16), (7, 1, 128, 32), (16, 1, 64, 64), (24, 2, 64, 48), (8, 1, 128, 16)])
def test_single_tokens(heads, kv_heads, dim, page, mask, dtype):
    """A few numbers of every query are large, so that the others are few of its whole steps."""
    sequences = SINGLES + [(5000, 1)]
    positions, seq, table, starts, context, total = _batch(sequences, page, 1)
    pages = _pages(total, kv_heads, page, dim, 1)
    q = torch.randn((len(sequences), heads * dim), generator=_generator(3), device=DEVICE)
    q[:, 5::32] *= 6.0
    q, mask, scale = q.to(dtype), _with_sink(mask, heads), dim ** -0.5
    for splits in (None, 1, 8):
        out = torch.full_like(q, math.nan)
        ops.paged_attention_int8(q, q.stride(0), out, pages, table, starts, context, len(sequences), 1, heads, kv_heads, dim, scale,
                                 plan=_plan(sequences, starts), decode_splits=splits, **mask)
        _hold(out, q, pages, table, starts, sequences, heads, kv_heads, dim, page, scale, dtype, **mask)


STEPS = {"a portion and single tokens": [(500, 60), (90, 1), (16, 1), (0, 1), (2000, 1)],
         "portions in a padded order": [(15, 1), (0, 130), (3000, 4), (31, 1), (7, 2)],
         "one of each": [(4000, 3), (4000, 1)]}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("what", list(STEPS))
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (12, 4, 128)])
def test_a_step_of_both_behind_its_append(heads, kv_heads, dim, what, dtype):
    """The append, the portions' attention and the single tokens' beside it, launched without a wait, eagerly and from a graph; every row against the
    formula over what the pages hold then."""
    page, sequences = 16, STEPS[what]
    positions, seq, table, starts, context, total = _batch(sequences, page, 1)
    plan, scale, tokens = _plan(sequences, starts), dim ** -0.5, positions.numel()
    inv_freq = (10000.0 ** (-torch.arange(0, dim, 2, device=DEVICE) / dim)).float()
    start = _pages(total, kv_heads, page, dim, 5)
    pages = _copy(start)
    given = torch.randn((tokens, (heads + 2 * kv_heads) * dim), generator=_generator(3), device=DEVICE).to(dtype)
    qkv, out = given.clone(), torch.empty((tokens, heads * dim), dtype=dtype, device=DEVICE)

    def step():
        ops.rope_kv_write_int8(qkv, positions, seq, table, pages, inv_freq, heads, kv_heads, dim, dim)
        ops.paged_attention_int8(qkv, qkv.stride(0), out, pages, table, starts, context, len(sequences), max(n for _, n in sequences), heads, kv_heads, dim,
                                 scale, plan=plan, after_append=True)

    def reset():
        qkv.copy_(given)
        out.fill_(math.nan)
        for name in ("k", "v", "k_scale", "v_scale"):
            getattr(pages, name).copy_(getattr(start, name))

    torch.cuda.synchronize()
    step()
    _hold(out, qkv, pages, table, starts, sequences, heads, kv_heads, dim, page, scale, dtype)
    eager = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(4):
        reset()
        torch.cuda.synchronize()
        graph.replay()
        assert torch.equal(out, eager)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_portion_alone_and_among_others(dtype):
    """How many blocks share a portion's keys, and how many of its tiles are a block's, goes by the step; what comes out stays within the bound."""
    heads, kv_heads, dim, page, scale = 16, 4, 128, 16, 0.09
    mine = (1500, 70)
    for sequences in ([mine], [mine, (0, 2)], [mine] + [(100 * i, 60) for i in range(9)], [mine] + [(40, 1500)] * 3 + [(70, 1), (3000, 1)]):
        positions, seq, table, starts, context, total = _batch(sequences, page, 1)
        pages = _pages(total, kv_heads, page, dim, 1)
        q = torch.randn((positions.numel(), heads * dim), generator=_generator(3), device=DEVICE).to(dtype)
        out = torch.full_like(q, math.nan)
        ops.paged_attention_int8(q, q.stride(0), out, pages, table, starts, context, len(sequences), max(n for _, n in sequences), heads, kv_heads, dim, scale,
                                 plan=_plan(sequences, starts))
        _hold(out, q, pages, table, starts, sequences, heads, kv_heads, dim, page, scale, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_two_layers_on_two_streams_at_once(dtype):
    """Nothing orders the streams, so each layer's work spaces have to be its own."""
    heads, kv_heads, dim, page = 8, 2, 64, 16
    sequences = [(2000, 1), (33, 300), (700, 1), (900, 40)]
    positions, seq, table, starts, context, total = _batch(sequences, page, 1)
    plan, tokens = _plan(sequences, starts), positions.numel()
    g = _generator(3)
    x = [torch.randn((tokens, 256), generator=g, device=DEVICE).to(dtype) for _ in range(2)]
    w_qkv = ops.quantise_weight(torch.randn(((heads + 2 * kv_heads) * dim, 256), generator=g, device=DEVICE))
    w_out = ops.quantise_weight(torch.randn((256, heads * dim), generator=g, device=DEVICE))
    start = _pages(total, kv_heads, page, dim, 5)

    def layer(x, pages):
        qkv = ops.linear_int8(x, w_qkv)
        ops.rope_kv_write_int8(qkv, positions, seq, table, pages, None, heads, kv_heads, dim, 0)
        mixed = torch.empty((tokens, heads * dim), dtype=dtype, device=DEVICE)
        ops.paged_attention_int8(qkv, qkv.stride(0), mixed, pages, table, starts, context, len(sequences), 300, heads, kv_heads, dim, 0.125, plan=plan,
                                 after_append=True)
        return ops.linear_int8(mixed, w_out)

    want = [layer(one, _copy(start)) for one in x]
    streams = [torch.cuda.Stream() for _ in range(2)]
    pages = [[_copy(start) for _ in range(2)] for _ in range(8)]
    torch.cuda.synchronize()
    got = []
    for turn in range(8):
        for stream, one, mine in zip(streams, x, pages[turn]):
            with torch.cuda.stream(stream):
                got.append(layer(one, mine))
    torch.cuda.synchronize()
    for i, result in enumerate(got):
        assert torch.equal(result, want[i % 2])
