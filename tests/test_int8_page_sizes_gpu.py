"""Appending to pages of 8 bits, of any number of tokens and at any number of tokens a call: what fits a page of the engine's default size is
asked of every other, to the bit."""

from __future__ import annotations

import pytest
import torch

from liteinfer_b200 import ops
from test_int8_gpu import DEVICE, _batch, _generator

pytestmark = pytest.mark.gpu


def _append(sequences, page, heads, kv_heads, dim, rotary, dtype, qkv):
    """(q rotated, the pages, where each token went: [tokens] pages and slots)."""
    positions, seq, table, _, _, total = _batch(sequences, page, 1)
    inv_freq = (10000.0 ** (-torch.arange(0, rotary, 2, device=DEVICE) / rotary)).float()
    pages = ops.Int8Pages.zeros(total, kv_heads, page, dim, DEVICE)
    q_out = torch.empty((positions.numel(), heads * dim), dtype=dtype, device=DEVICE)
    ops.rope_kv_write_int8(qkv, positions, seq, table, pages, inv_freq, heads, kv_heads, dim, rotary, q_out=q_out)
    return q_out, pages, table[seq.long(), positions.long() // page].long(), positions.long() % page


# Head size, rotated dimensions and tokens of a page: with 128 dimensions, 80 tokens are the most whose cosines take 40 KB.
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,rotary,page", [(128, 128, 72), (128, 128, 80), (128, 128, 96), (128, 128, 128), (128, 128, 400), (128, 128, 512),
                                             (64, 64, 256), (64, 64, 1024), (64, 64, 1040), (64, 32, 2048), (512, 512, 16), (512, 512, 32),
                                             (64, 20, 16), (64, 20, 1000)])
@pytest.mark.parametrize("tokens", [1, 300, 3300])
def test_append_to_pages_of_any_size(dim, rotary, page, tokens, dtype):
    """A prompt of `tokens` and a few single tokens: q is rotated as in pages of 16, every page's scale is that of its largest number, and what is
    held is each number divided by it and rounded (keys as they are rotated when they are queries)."""
    heads, kv_heads = 1, 1
    sequences = [(0, tokens), (0, 1), (page, 1), (0, 3)]
    rows = sum(new for _, new in sequences)
    qkv = torch.randn((rows, 3 * dim), generator=_generator(2), device=DEVICE).to(dtype)
    q_out, pages, at, slot = _append(sequences, page, heads, kv_heads, dim, rotary, dtype, qkv)
    # What small pages rotate is held to the formula elsewhere.  Here keys stand in the queries' place as well, in 32 bits, where nothing is
    # rounded behind the rotation.
    keys = torch.cat((qkv[:, dim:2 * dim], qkv[:, dim:]), dim=1).float()
    turned, _, _, _ = _append(sequences, 16 if dim < 512 else 5, heads, kv_heads, dim, rotary, torch.float32, keys)
    queries, _, _, _ = _append(sequences, 16 if dim < 512 else 5, heads, kv_heads, dim, rotary, torch.float32, qkv.float())
    assert torch.equal(q_out, queries.to(dtype))
    for pool, scale, new in ((pages.k, pages.k_scale, turned), (pages.v, pages.v_scale, qkv[:, 2 * dim:].float())):
        need = torch.zeros(scale.shape[0], device=DEVICE).index_reduce_(0, at, new.abs().amax(1) * torch.tensor(1 / 127, device=DEVICE), "amax")
        assert torch.equal(scale[:, 0], need)
        want = torch.zeros_like(pool)
        want[at, 0, slot] = torch.round(new / need[at][:, None]).clamp(-127, 127).to(torch.int8)
        assert torch.equal(pool, want)
