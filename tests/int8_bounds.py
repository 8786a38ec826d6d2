"""How far the attention over pages of 8 bits may be from its formula in 64 bits, element by element, from what its kernels round.

Both forms.  A score's terms are added up in 32 bits (2 dim roundings, or products with what is cut off, of 2^-24 of them); exponentials
are within 2^-22 and what goes into them is rounded, 2^-20 in all; with a cap the tangent is within 2^-19 of the cap.  An error e of a score
moves a weight by e and the denominator by as much.  Sums over keys have 32 bits.  The result is rounded once to its type.

Portions: weights have 11 bits for bfloat16, 22 for float32; what lies 2^30 below the largest goes to nothing.

Single tokens: for bfloat16 a query's numbers are whole ones of a 16,256th of its head's largest, half a step off at most, so a score is off by
half a step times the sum of a key's numbers; for float32 they keep 22 bits, and 2^-25 of the largest.  Weights as above; the base-2
logarithm of a page's scale of values is within 2^-22 of its size, or of one."""

from __future__ import annotations

import torch

import plain_int8 as plain


def attention(form, dtype, q, k, v, scale, heads, kv_heads, first, v_scales=None, **mask):
    """(the formula, the bound), both [new, heads, dim]; arguments as `plain_int8.attention`, `form` "portion" or "single", `v_scales`
    the scales of the pages that are seen."""
    want, terms = plain.attention(q, k, v, scale, heads, kv_heads, first, **mask)
    around, _ = plain.attention(q, k, v.abs(), scale, heads, kv_heads, first, **mask)
    most, _ = plain.attention(q, k, v.abs().amax(-1, keepdim=True).expand_as(v), scale, heads, kv_heads, first, **mask)
    dim, keys = q.shape[-1], k.shape[0]
    short = dtype is torch.bfloat16
    result, weight = (2.0 ** -8, 2.0 ** -11) if short else (2.0 ** -23, 2.0 ** -22)
    score = 2 * dim * 2.0 ** -24 * terms + 2.0 ** -20 + mask.get("softcap", 0.0) * 2.0 ** -19
    if form == "single":
        top = q.abs().amax(-1, keepdim=True)                                                       # [new, heads, 1]
        sums = k.abs().sum(-1).amax(0).repeat_interleave(heads // kv_heads)[None, :, None]
        score = score + abs(scale) * sums * top * (1 / 32512 if short else 2.0 ** -25)
        sizes = v_scales[v_scales > 0].double().log2().abs().max() if v_scales is not None and bool((v_scales > 0).any()) else 0.0
        weight = weight + (1 + float(sizes)) * 2.0 ** -22
    return want, want.abs() * result + around * (weight + 2 * score + keys * 2.0 ** -23) * 1.01 + most * 2.0 ** -24
