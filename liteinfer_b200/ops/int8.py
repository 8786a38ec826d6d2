"""Serving in 8 bits: a paged cache held in 8 bits and products with weights in 8 bits.  The operators' Python faces, in the
manner of `ops.kernels`: every function checks its tensors, launches on torch's current stream and raises when the launch is
refused.

What is held in 8 bits is a run of numbers with one scale, x ~ q * scale: scale = max |x| * (1 / 127), q = rint(x / scale).  The
runs are a page's tokens of one KV head (keys and values apart) in the cache, an output channel of a weight, a token of
a product's activations.  A run of zeros has the scale 0; one with an infinity or a NaN reads back as NaN.
"""

from __future__ import annotations

import struct
from dataclasses import dataclass, replace

import torch

from liteinfer_b200.ops import kernels as _k
from liteinfer_b200.ops.kernels import _check, _code, _fn, _here, _on_gpu, _rows2d

# The C entries take one structure of 8-byte fields (q: a whole number or an address, d: a number).
_k._SIGNATURES.update({
    "li_rope_kv_write_int8": ("int8_cache", [_k.ctypes.c_char_p]),
    "li_read_pages_int8": ("int8_cache", [_k.ctypes.c_char_p]),
    "li_attention_int8": ("attention_int8", [_k.ctypes.c_char_p]),
    "li_attention_int8_supports": ("attention_int8", [_k.c_int, _k.c_int, _k.c_int, _k.c_int]),
    "li_attention_int8_capacity": ("attention_int8", [_k.c_int, _k.c_int, _k.c_int]),
    "li_attention_int8_prompt": ("attention_int8_prompt", [_k.ctypes.c_char_p]),
    "li_attention_int8_prompt_supports": ("attention_int8_prompt", [_k.c_int, _k.c_int, _k.c_int, _k.c_int]),
    "li_quantise_rows": ("gemm_int8", [_k.ctypes.c_char_p]),
    "li_linear_int8": ("gemm_int8", [_k.ctypes.c_char_p]),
})
_ROPE_KV_WRITE = struct.Struct("=21qdq").pack
_READ_PAGES = struct.Struct("=22q").pack
_ATTENTION = struct.Struct("=20qdqd5q").pack
_ATTENTION_PROMPT = struct.Struct("=22qd2qd5q").pack
_QUANTISE_ROWS = struct.Struct("=9q").pack
_LINEAR = struct.Struct("=17q").pack
_NEEDS_PLACE = 100003          # li_linear_int8: this product wants a place for x in 8 bits


def _stream() -> int:
    """The current stream's handle (of `torch.cuda.current_stream()`, without the object around it, which takes the host 5 us)."""
    pinned = _here.stream
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device()) if pinned is None else pinned


def _refuse(condition: bool, why: str) -> None:
    if condition:
        raise ValueError(why)


def _ints(*tensors: torch.Tensor) -> None:
    """Contiguous int32 tensors on the GPU."""
    for t in tensors:
        if t.dtype is not torch.int32 or not t.is_cuda or not t.is_contiguous():
            _on_gpu(t)
            _k._int32(t, "positions, sequences, tables and lengths")


# ------------------------------------------------------------------ the cache
@dataclass
class Int8Pages:
    """One layer's pages of keys and values in 8 bits: `k` and `v` [pages, kv_heads, page_size, head_dim] int8, `k_scale` and
    `v_scale` [pages, kv_heads] float32."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    @classmethod
    def zeros(cls, pages: int, kv_heads: int, page_size: int, head_dim: int, device: torch.device | str) -> "Int8Pages":
        pool = lambda: torch.zeros((pages, kv_heads, page_size, head_dim), dtype=torch.int8, device=device)
        scale = lambda: torch.zeros((pages, kv_heads), dtype=torch.float32, device=device)
        return cls(pool(), pool(), scale(), scale())

    def check(self, kv_heads: int, head_dim: int) -> tuple[int, int]:
        """(pages, page_size) of pages that hold what they should; raises if they do not."""
        k, v, k_scale, v_scale = self.k, self.v, self.k_scale, self.v_scale
        shape, scales = k.shape, k_scale.shape
        if len(shape) != 4 or shape[1] != kv_heads or shape[3] != head_dim or v.shape != shape:
            raise ValueError(f"8-bit pages are [pages, {kv_heads}, page_size, {head_dim}], got {tuple(shape)} and {tuple(v.shape)}")
        if k.dtype is not torch.int8 or v.dtype is not torch.int8:
            raise ValueError("8-bit pages are int8")
        if len(scales) != 2 or scales[0] != shape[0] or scales[1] != kv_heads or v_scale.shape != scales:
            raise ValueError("8-bit pages have a scale for each page and head")
        if k_scale.dtype is not torch.float32 or v_scale.dtype is not torch.float32:
            raise ValueError("the pages' scales are float32")
        _on_gpu(k, v, k_scale, v_scale)
        return shape[0], shape[2]


def rope_kv_write_int8(qkv: torch.Tensor, positions: torch.Tensor, seq_of_token: torch.Tensor, block_table: torch.Tensor,
                       pages: Int8Pages, inv_freq: torch.Tensor | None, heads: int, kv_heads: int, head_dim: int,
                       rotary_dim: int, store: bool = True, cos_sin_scale: float = 1.0,
                       q_out: torch.Tensor | None = None) -> None:
    """`rope_kv_write` into pages of 8 bits: rotates q (into `q_out` [tokens, heads * head_dim], or in place) and k, and
    appends k and v of every token to its page (with `store` False only q is rotated).

    qkv: rows [q heads | k heads | v heads], which may lie in wider rows.  A sequence's tokens lie one behind the other in
    the batch, at consecutive positions; a token with `seq_of_token` -1 is padding and a page of -1 is skipped.  A page's
    scale grows where its new tokens need it (by a quarter at least, the tokens before them are then rounded again); a
    token in slot 0 starts its page anew, and what lay behind a call's last token in its page is forgotten.
    """
    _rows2d(qkv, "qkv")
    _ints(positions, seq_of_token, block_table)
    num_pages, page_size = pages.check(kv_heads, head_dim)
    tokens, width = qkv.shape
    _refuse(width < (heads + 2 * kv_heads) * head_dim, f"a row of qkv has {width} numbers, fewer than its heads need")
    _refuse(positions.numel() != tokens or seq_of_token.numel() != tokens, "every token has a position and a sequence")
    if inv_freq is not None:
        _on_gpu(inv_freq)
        _refuse(inv_freq.dtype is not torch.float32 or inv_freq.numel() * 2 != rotary_dim, "inv_freq holds rotary_dim / 2 numbers of float32")
    if q_out is None:
        q_out = qkv
    else:
        _rows2d(q_out, "q_out")
        _refuse(q_out.dtype is not qkv.dtype or q_out.shape != (tokens, heads * head_dim), "q_out is [tokens, heads * head_dim] of qkv's type")
    _check(_fn("li_rope_kv_write_int8")(_ROPE_KV_WRITE(
        _code(qkv), qkv.data_ptr(), qkv.stride(0), q_out.data_ptr(), q_out.stride(0), positions.data_ptr(),
        seq_of_token.data_ptr(), block_table.data_ptr(), block_table.stride(0), pages.k.data_ptr(), pages.v.data_ptr(),
        pages.k_scale.data_ptr(), pages.v_scale.data_ptr(), 0 if inv_freq is None else inv_freq.data_ptr(), tokens, heads, kv_heads,
        head_dim, rotary_dim, page_size, num_pages if store else 0, cos_sin_scale, _stream())), "rope_kv_write_int8")


def read_pages_int8(pages: Int8Pages, block_table: torch.Tensor, lens: torch.Tensor, k_out: torch.Tensor,
                    v_out: torch.Tensor) -> None:
    """The numbers that pages stand for, in k_out's type: k_out and v_out [rows, blocks, kv_heads, page_size, head_dim]
    receive the pages that block_table [rows, blocks] names.  Row r holds lens[r] tokens, page_size a block; the slots
    behind them, and all of a page of -1, read as zeros."""
    _refuse(pages.k.dim() != 4, "8-bit pages are [pages, kv_heads, page_size, head_dim]")
    _, kv_heads, _, head_dim = pages.k.shape
    num_pages, page_size = pages.check(kv_heads, head_dim)
    _ints(block_table, lens)
    _on_gpu(k_out, v_out)
    rows, blocks = block_table.shape
    _refuse(k_out.shape != (rows, blocks, kv_heads, page_size, head_dim) or v_out.shape != k_out.shape or k_out.dtype is not v_out.dtype,
            "what is read is [rows, blocks, kv_heads, page_size, head_dim], keys and values alike")
    _refuse(lens.numel() != rows, "every row has a length")
    _check(_fn("li_read_pages_int8")(_READ_PAGES(
        _code(k_out), pages.k.data_ptr(), pages.v.data_ptr(), pages.k_scale.data_ptr(), pages.v_scale.data_ptr(),
        block_table.data_ptr(), block_table.stride(0), lens.data_ptr(), k_out.data_ptr(), v_out.data_ptr(), rows, blocks,
        kv_heads, head_dim, page_size, num_pages, 0, 0, 0, 0, 0, _stream())), "read_pages_int8")


def paged_attention_int8(q: torch.Tensor, q_row_stride: int, out: torch.Tensor, pages: Int8Pages, block_table: torch.Tensor,
                         query_start_loc: torch.Tensor, context_lens: torch.Tensor, num_seqs: int, max_q_len: int, heads: int,
                         kv_heads: int, head_dim: int, scale: float, window: int = 0, plan=None,
                         decode_splits: int | None = None, keep_first: int = 0, softcap: float = 0.0,
                         sink: torch.Tensor | None = None, chunk: int = 0, after_append: bool = False) -> torch.Tensor:
    """`paged_attention` over pages of 8 bits; arguments as there (keys and values of one size).

    `after_append`: the caller says that the launch ahead of this one on the stream is a `rope_kv_write_int8`, and that it wrote one token
    at most of every sequence that is attended as a single token (a step of the engine).  Their older pages are then read while that
    launch still writes the newest ones.  After an append of several of a sequence's tokens it would be wrong.

    Single tokens (with a `plan`, or where no sequence brings more than one) of head size 64 or 128, groups of at most 16 heads and
    pages of a multiple of 16 tokens read the pages as they are; `decode_splits` blocks share a sequence's keys (rounded down to a
    power of two, 8 at most; None: chosen from the batch and the context).  Portions of prompts of these head and page sizes
    read whole numbers that are spread out to 16 bits first, exactly, and keep the scales apart.  For everything else the
    pages that can be seen are read back into q's type once, and `paged_attention` runs over those.  Either is made room for by the
    longest context of a launch; so many sequences go at a time as `WORK_BYTES` hold, one at least (`attention_int8_work`).
    """
    _rows2d(q, "q"); _rows2d(out, "out")
    _ints(block_table, query_start_loc, context_lens)
    num_pages, page_size = pages.check(kv_heads, head_dim)
    dtype = q.dtype
    code = _code(q)
    _refuse(dtype is not out.dtype or out.shape[1] != heads * head_dim, "out is [tokens, heads * head_dim] of q's type")
    _refuse(heads % kv_heads != 0, "the query heads are a multiple of the KV heads")
    _refuse(q.shape[1] < heads * head_dim, f"a row of q has {q.shape[1]} numbers, fewer than its heads need")
    _refuse(num_seqs > block_table.shape[0] or num_seqs > context_lens.numel() or num_seqs >= query_start_loc.numel(),
            "every sequence has a row of the block table, a length and a start, the last one an end")
    if sink is not None:
        _on_gpu(sink)
        _refuse(sink.dtype is not torch.float32 or sink.numel() != heads, "a sink is float32, one number a head")
    _refuse(chunk > 0 and window > 0, "an attention has a window or chunks")
    span = -chunk if chunk > 0 else window if window > 0 else 0
    kept = keep_first if window > 0 and keep_first > 0 else 0
    direct = not kept and _supports("li_attention_int8_supports", heads, kv_heads, head_dim, page_size)
    portions = _supports("li_attention_int8_prompt_supports", heads, kv_heads, head_dim, page_size)
    if plan is None:
        prompts, singles = (0, num_seqs) if direct and max_q_len == 1 else (num_seqs, 0)
    else:
        prompts, singles = plan.num_prefill, plan.num_decode
    table, stream = block_table.data_ptr(), _stream()
    k, v, k_scale, v_scale = pages.k.data_ptr(), pages.v.data_ptr(), pages.k_scale.data_ptr(), pages.v_scale.data_ptr()
    stride, starts, contexts = block_table.stride(0), query_start_loc.data_ptr(), context_lens.data_ptr()

    most = block_table.shape[1]
    beside = False
    if prompts and portions:
        if plan is None:
            sequences, longest, most_queries = 0, 0, max_q_len
        else:
            sequences, longest, most_queries = plan.prefill_seqs.data_ptr(), plan.max_prefill_context_len, plan.max_prefill_query_len
        blocks = min(-(-longest // page_size), most) if longest else most
        each, rest = _spread_bytes(blocks * page_size, q.shape[0], heads, kv_heads, head_dim, dtype)
        at_once = _at_once(prompts, each)
        work = torch.empty((at_once * each + rest,), dtype=torch.int8, device=q.device)
        for first in range(0, prompts, at_once):        # (in a list of sequences, or in the batch itself)
            here = (table, starts, contexts, sequences + 4 * first) if sequences else (table + 4 * first * stride, starts + 4 * first, contexts + 4 * first, 0)
            _check(_fn("li_attention_int8_prompt")(_ATTENTION_PROMPT(
                code, q.data_ptr(), q.shape[0], q_row_stride, out.data_ptr(), out.stride(0), k, v, k_scale, v_scale, here[0], stride, here[1], here[2],
                here[3], min(at_once, prompts - first), most_queries, heads, kv_heads, head_dim, page_size, num_pages, scale, span, kept, softcap,
                0 if sink is None else sink.data_ptr(), work.data_ptr(), blocks, _k.scratch_for(q.device).gemm_error.data_ptr(), stream)),
                "paged_attention_int8")
        del work                        # (what follows on the stream may have its place)
        prompts, beside = 0, most_queries > 0 and blocks > 0       # (the single tokens' kernel need not wait for this one, if there is one)
    # (Where `paged_attention` takes all sequences in one launch, it takes the single tokens next to portions too.)
    every = plan is None or not _k.mma_attention_supports(dtype, heads, kv_heads, head_dim)
    if singles and direct and (plan is None or not prompts or not every):
        if plan is None:
            sequences, longest = 0, block_table.shape[1] * page_size
        else:
            rows = plan.decode_seqs if plan.decode_longest_first is None else plan.decode_longest_first
            sequences, longest = rows.data_ptr(), plan.max_decode_context_len
        splits = decode_splits_int8(code, singles, heads, kv_heads, head_dim, min(longest, abs(span)) if span else longest, decode_splits)
        _check(_fn("li_attention_int8")(_ATTENTION(
            code, q.data_ptr(), q_row_stride, out.data_ptr(), out.stride(0), k, v, k_scale, v_scale, table, stride, starts, contexts,
            sequences, singles, heads, kv_heads, head_dim, page_size, num_pages, scale, span, softcap,
            0 if sink is None else sink.data_ptr(), splits, beside, after_append, stream)), "paged_attention_int8")
        singles = 0
    if not prompts and not singles:
        return out

    # The pages that the rest can see, in q's type, and a table of them, in one piece of memory.
    part = plan
    if part is not None and prompts != part.num_prefill:
        part = replace(part, num_prefill=0, prefill_seqs=None, max_prefill_query_len=0)
    if part is not None and singles != part.num_decode:
        part = replace(part, num_decode=0, decode_seqs=None, decode_tokens=None, decode_longest_first=None)
    options = dict(decode_splits=decode_splits, keep_first=keep_first, softcap=softcap, sink=sink, chunk=chunk)

    def over_read_back(count, longest, part, sequences=None, first=0):
        """Attention of `count` sequences of up to `longest` tokens (0: not known), the rows of the batch that `sequences` names or those from
        `first` on."""
        blocks = min(-(-longest // page_size), most) if longest else most
        size = _read_back_bytes(count * blocks * page_size, kv_heads, head_dim, dtype)
        rows = block_table.shape[0] - first
        work = torch.empty((2 * size + 4 * rows * blocks,), dtype=torch.int8, device=q.device)
        keys = work.data_ptr()
        _check(_fn("li_read_pages_int8")(_READ_PAGES(
            code, k, v, k_scale, v_scale, table + 4 * first * stride, stride, contexts + 4 * first, keys, keys + size, count, blocks, kv_heads, head_dim,
            page_size, num_pages, 0 if sequences is None else sequences.data_ptr(), starts + 4 * first, span, kept, keys + 2 * size, stream)),
            "read_pages_int8")
        pools = work[:2 * size].view(dtype).view(2, count * blocks, kv_heads, page_size, head_dim)
        _k.paged_attention(q, q_row_stride, out, pools[0], pools[1], work[2 * size:].view(torch.int32).view(-1, blocks), query_start_loc[first:],
                           context_lens[first:], count if sequences is None else num_seqs, max_q_len, heads, kv_heads, head_dim, scale, window, plan=part,
                           **options)

    def room_for(count, longest):
        return _at_once(count, 2 * _read_back_bytes(min(longest, most * page_size) if longest else most * page_size, kv_heads, head_dim, dtype))

    known = [0] if plan is None else [plan.max_prefill_context_len] * (plan.num_prefill > 0) + [plan.max_decode_context_len] * (plan.num_decode > 0)
    whole = max(known) if min(known) > 0 else 0
    if every or (prompts and singles and room_for(num_seqs, whole) >= num_seqs):
        # (A plan that deals the sequences to launches of their own goes with all of them.)
        at_once = room_for(num_seqs, whole)
        for first in range(0, num_seqs, at_once):
            over_read_back(min(at_once, num_seqs - first), whole, part, first=first)
        return out
    no_portions = dict(num_prefill=0, prefill_seqs=None, max_prefill_query_len=0)
    no_singles = dict(num_decode=0, decode_seqs=None, decode_tokens=None, decode_longest_first=None)
    if prompts:
        at_once = room_for(prompts, plan.max_prefill_context_len)
        for first in range(0, prompts, at_once):
            rows, count = plan.prefill_seqs[first:first + at_once], min(at_once, prompts - first)
            over_read_back(count, plan.max_prefill_context_len, replace(plan, num_prefill=count, prefill_seqs=rows, **no_singles), rows)
    if singles:
        at_once = room_for(singles, plan.max_decode_context_len)
        for first in range(0, singles, at_once):
            some = slice(first, first + at_once)
            mine = replace(plan, **no_portions)
            if at_once < singles:
                mine = replace(mine, num_decode=min(at_once, singles - first), decode_seqs=plan.decode_seqs[some], decode_tokens=plan.decode_tokens[some],
                               decode_longest_first=None)
            over_read_back(mine.num_decode, plan.max_decode_context_len, mine, mine.decode_seqs)
    return out


# The most memory that a call of `paged_attention_int8` takes to spread pages out or to read them back, but for a single sequence of a launch,
# which it takes whole.
WORK_BYTES = 1 << 30


def _spread_bytes(context: int, tokens: int, heads: int, kv_heads: int, head_dim: int, dtype: torch.dtype) -> tuple[int, int]:
    """What a portion of a context takes spread out to 16 bits, and what its launch takes besides (li_attention_int8_prompt)."""
    return context * kv_heads * (4 * head_dim + 1), 128 + (tokens * heads * (4 * head_dim + 4) if dtype is torch.float32 else 0)


def _read_back_bytes(tokens: int, kv_heads: int, head_dim: int, dtype: torch.dtype) -> int:
    """What keys (or values) of this many tokens take in q's type."""
    return tokens * kv_heads * head_dim * dtype.itemsize


def _at_once(count: int, each: int) -> int:
    """How many of `count` sequences go at a time."""
    return max(1, min(count, WORK_BYTES // max(1, each)))


def attention_int8_work(sequences: int, context: int, tokens: int, heads: int, kv_heads: int, head_dim: int, page_size: int, dtype: torch.dtype) -> int:
    """The most bytes that a call of `paged_attention_int8` takes beside its arguments, over `sequences` of up to `context` tokens that bring
    `tokens` in all."""
    context = -(-context // page_size) * page_size
    spread, rest = _spread_bytes(context, tokens, heads, kv_heads, head_dim, dtype)
    read_back = 2 * _read_back_bytes(context, kv_heads, head_dim, dtype)
    return max(_at_once(sequences, spread) * spread + rest, _at_once(sequences, read_back) * read_back + 4 * sequences * context // page_size)


_supported: dict[tuple[str, int, int, int, int], bool] = {}
_capacity: dict[tuple[int, int, bool], int] = {}


def _supports(entry: str, *sizes: int) -> bool:
    """Whether an attention's C entry says that it takes these sizes: heads, kv_heads, head_dim, page_size."""
    key = (entry, *sizes)
    found = _supported.get(key)
    if found is None:
        found = _supported[key] = bool(_fn(entry)(*sizes))
    return found


def decode_splits_int8(dtype_code: int, count: int, heads: int, kv_heads: int, head_dim: int, longest: int,
                       wanted: int | None = None) -> int:
    """Blocks (1, 2, 4 or 8) that share a sequence's keys in a launch over `count` single tokens of contexts up to `longest`."""
    if wanted is None:
        groups = heads // kv_heads
        key = (dtype_code, head_dim, groups <= 8)
        if key not in _capacity:
            _capacity[key] = int(_fn("li_attention_int8_capacity")(dtype_code, head_dim, groups)) or 2 * _k.NUM_SMS
        # As many as run at once, 128 keys each at least, and 512 where most SMs have a block without splitting: a merge costs some 2 us,
        # and a cluster starts when all of it has a place (16 sequences of 600 keys, 8 KV heads of 64: 8.2 us unsplit, 9.8 with two).  A
        # batch that fills the device is split in two where contexts are long: of many lengths, the longest ones end sooner (64 of 400
        # to 8,191 of 128: 138 and 128 us), and of one length it costs nothing.
        pairs = max(1, count * kv_heads)
        wanted = min(_capacity[key] // pairs, max(1, longest // (128 if pairs <= 96 else 512)))
        if wanted <= 1 and longest >= 3000 and pairs <= 2 * _capacity[key]:
            wanted = 2
    return 8 if wanted >= 8 else 4 if wanted >= 4 else 2 if wanted >= 2 else 1


# ------------------------------------------------------------------ products
@dataclass
class Int8Weight:
    """A weight [N, K] in 8 bits: `q` [N, padded K] int8, its rows filled up with zeros to a multiple of 16, and `scale` [N]
    float32."""

    q: torch.Tensor
    scale: torch.Tensor
    inner: int                  # K
    at_rest: bool = False       # no kernel writes it from here on (a model's parameter): it may be read before the kernels ahead are done

    @property
    def shape(self) -> tuple[int, int]:
        return self.q.shape[0], self.inner

    @property
    def device(self) -> torch.device:
        return self.q.device


def quantise_rows(x: torch.Tensor, q: torch.Tensor, scale: torch.Tensor) -> None:
    """x [M, K] (float32 or bfloat16; its rows may lie in wider ones) -> q [M, padded K] int8, zeros from K on, and scale [M]."""
    _rows2d(x, "x")
    _on_gpu(q, scale)
    M, K = x.shape
    _refuse(q.dtype is not torch.int8 or q.dim() != 2 or q.shape[0] != M or q.shape[1] != -(-K // 16) * 16,
            "rows in 8 bits are int8, as many numbers as x's filled up to a multiple of 16")
    _refuse(scale.dtype is not torch.float32 or scale.numel() != M, "every row has a scale of float32")
    _check(_fn("li_quantise_rows")(_QUANTISE_ROWS(_code(x), x.data_ptr(), x.stride(0), q.data_ptr(), q.shape[1], scale.data_ptr(), M, K,
                                                  _stream())), "quantise_rows")


def quantise_weight(weight: torch.Tensor) -> Int8Weight:
    """A weight [N, K] (float32 or bfloat16) as `linear_int8` takes it."""
    N, K = weight.shape
    made = Int8Weight(torch.empty((N, -(-K // 16) * 16), dtype=torch.int8, device=weight.device),
                      torch.empty((N,), dtype=torch.float32, device=weight.device), K)
    quantise_rows(weight, made.q, made.scale)
    return made


def linear_int8(x: torch.Tensor, weight: Int8Weight, out: torch.Tensor | None = None,
                bias: torch.Tensor | None = None) -> torch.Tensor:
    """out[M, N] = x[M, K] @ weight^T (+ bias), x quantised row by row on the way; float32 or bfloat16 in and out.  x's rows
    may lie in wider ones."""
    _rows2d(x, "x")
    w, w_scale = weight.q, weight.scale
    M, K = x.shape
    N, padded = w.shape
    dtype = x.dtype
    _refuse(weight.inner != K, "a row of x has as many numbers as one of the weight")
    _refuse(padded % 16 != 0 or padded < K, "the rows of a weight in 8 bits are filled up to a multiple of 16")
    _refuse(w.dtype is not torch.int8 or w_scale.dtype is not torch.float32 or w_scale.numel() != N,
            "a weight in 8 bits is int8 with a scale of float32 for each row")
    if out is None:
        out = torch.empty((M, N), dtype=dtype, device=x.device)
    else:
        _refuse(out.shape != (M, N) or out.dtype is not dtype, "out is [M, N] of x's type")
    _on_gpu(w, w_scale, out, bias)
    _refuse(bias is not None and (bias.dtype is not dtype or bias.numel() != N), "a bias has x's type and a number for each output")
    error_flag = _k.scratch_for(x.device).gemm_error.data_ptr()
    common = (w.data_ptr(), padded, w_scale.data_ptr(), 0 if bias is None else bias.data_ptr(), out.data_ptr(), N, error_flag, weight.at_rest)
    code, start, stride, stream, run = _code(x), x.data_ptr(), x.stride(0), _stream(), _fn("li_linear_int8")
    # A few rows may go as one kernel, in which every block quantises them: that takes the host 7 us instead of 13.  (In a captured graph the
    # host's time is nobody's, and the device wants two kernels from the second row on: 2,048 x 2,048 with one row 3.5 us and 4.2, with
    # eight 6.4 and 4.3.)
    if M <= 16 and M * padded <= 16384 and (M == 1 or not torch.cuda.is_current_stream_capturing()):
        done = run(_LINEAR(code, start, stride, 0, padded, 0, M, K, stream, *common))
        if done != _NEEDS_PLACE:
            _check(done, "linear_int8")
            return out
    # x in 8 bits and its scales: one piece of memory, of this call alone.  Its rows begin at 128 bytes, or a tile's piece of each costs a
    # memory sector more (5,889 x 6,320 x 6,800: 245 us without, 203 with).
    row = -(-padded // 128) * 128
    work = torch.empty((M * row + 4 * M,), dtype=torch.int8, device=x.device)
    place = work.data_ptr()
    _check(run(_LINEAR(code, start, stride, place, row, place + M * row, M, K, stream, *common)), "linear_int8")
    return out
