"""A quantised paged K/V cache and attention over it, on gfx950.

The cache holds K and V with one E8M0 scale per 32 columns of a row, in 8 bits
(MXFP8, E4M3 codes: ``quant.mxfp8_qk_quant`` bit for bit below 3e38) or in 4 (MXFP4,
E2M1 codes), in pages that sequences take as they grow.  ``write_kv_cache`` quantises
new rows into it, ``append_kv_cache`` rotates Q and K by their positions on the way,
``paged_attention`` attends over it (one token of each sequence, or a chunk),
``read_kv_cache`` gives the values back, e.g. for ``fake_quant_attention``.

These are for inference: they have no derivative, backward or forward, and refuse inputs that
ask for one.  No call synchronises; all of them can be captured in a HIP graph.
Arguments are checked in ``csrc/lbfq_torch.cpp``.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib

BLOCK = 32  # columns of a scale
PAGE_SIZES = (16, 32, 64, 128, 256, 512, 1024)


class PagedKVCache(NamedTuple):
    """The tensors of a cache, contiguous, on one device.

    Row ``r`` of page ``p`` of head ``h`` is ``k_codes[p, h, r]``; its value is code *
    2^(scale - 127), ``k_scale[p, h, r, c]`` for columns 32 c ... 32 c + 31.  A cache
    that is not filled by ``write_kv_cache`` holds no NaN code and no scale of 255 where
    a query looks.  In 4 bits an element of the codes holds two: the even column in its
    low half, the odd one in its high half, 0, 1/2, 1, 3/2, 2, 3, 4, 6 as 0 ... 7 and plus
    8 for the negative ones.  (Torch can do little with that dtype: copy pages as
    ``k_codes.view(torch.uint8)``.)
    """

    k_codes: torch.Tensor  # (pages, H, page size, D) float8_e4m3fn, or (..., D / 2) float4_e2m1fn_x2
    k_scale: torch.Tensor  # (pages, H, page size, D / 32) uint8, E8M0
    v_codes: torch.Tensor
    v_scale: torch.Tensor


def empty_kv_cache(num_pages: int, page_size: int, heads: int, head_dim: int, *, device="cuda",
                   bits: int = 8) -> PagedKVCache:
    """A cache of zeros.  page_size: 16 to 1024 tokens, a power of two; bits of a code: 8 or 4."""
    if head_dim not in (64, 128):
        raise ValueError(f"D must be 64 or 128; got {head_dim}")
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES}; got {page_size}")
    if num_pages <= 0 or heads <= 0:
        raise ValueError(f"num_pages and heads must be positive; got {num_pages} and {heads}")
    if bits not in (4, 8):
        raise ValueError(f"bits must be 4 or 8; got {bits}")
    rows = (int(num_pages), int(heads), int(page_size))
    width, code = (head_dim, torch.float8_e4m3fn) if bits == 8 else (head_dim // 2, torch.float4_e2m1fn_x2)
    k, v = (torch.zeros((*rows, width), dtype=torch.uint8, device=device).view(code) for _ in range(2))
    ks, vs = (torch.full((*rows, head_dim // BLOCK), 127, dtype=torch.uint8, device=device) for _ in range(2))
    return PagedKVCache(k, ks, v, vs)


def write_kv_cache(k: torch.Tensor, v: torch.Tensor, cache: PagedKVCache, slots: torch.Tensor) -> None:
    """Quantise rows of K and V into their slots of the cache.

    ``k`` and ``v`` are (T, H, D) in fp32, fp16 or bf16 (views are read where they
    are); ``slots`` (T,) int64 holds page * page_size + row of each token.  A slot
    outside the cache (-1 for padding) is skipped.  The slots of one call must
    differ: what one that is named twice holds afterwards is not defined.

    Per 32 columns the scale is 2^ceil(log2(max(amax, 1e-4) / 448)), at most 2^119,
    and the codes round to nearest, ties to even.  As with the package's other
    quantisers, a NaN leaves its block's scale alone and becomes -448 * scale.  An
    infinity, or anything past 448 * 2^119 = 3e38, is held as that: the cache's
    values are finite, and what a query does not see cannot reach its result.  In 4 bits
    the same with 6 in the place of 448, and 6 * 2^125 = 2.6e38 as the largest.
    """
    _lib.torch_ops().write_kv_cache(k, v, *cache, slots)


def append_kv_cache(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, cache: PagedKVCache, slots: torch.Tensor,
                    cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, *,
                    pairs: str = "adjacent") -> torch.Tensor | None:
    """Rotate new rows of Q and K by their positions, write K and V into the cache, return Q.

    ``k`` and ``v`` are (T, H, D) and ``q`` (T, Hq, D) (or None: only the cache is
    written, and None returned) in one of fp32, fp16 and bf16; views are read where
    they are.  The first R columns are rotated in pairs as by ``qk_norm_rope``, with
    ``cos`` and ``sin`` (P, R/2) fp32 (``rotary_table``) and ``positions`` (T,) int32
    or int64; a negative position is not rotated.  A model that normalises Q and K
    calls ``qk_norm_rope`` and ``write_kv_cache`` instead.  ``slots`` as in
    ``write_kv_cache``.

    The rotated values are fp32, each product and the sum rounded.  Q is rounded once
    more, to its dtype; K goes from there into the cache, without a rounding to 16
    bits on the way.  A token whose position lies past the tables comes out as NaN in
    Q's rotated columns, and nothing of it is written.  Returns a new contiguous tensor.
    """
    return _lib.torch_ops().append_kv_cache(q, k, v, *cache, slots, cos, sin, positions, pairs)


def read_kv_cache(cache: PagedKVCache, block_table: torch.Tensor, seq_lens: torch.Tensor, max_len: int, *,
                  dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V of the first ``max_len`` tokens of each sequence, (B, max_len, H, D).

    ``block_table`` (B, pages) int32 lists each sequence's pages in order and
    ``seq_lens`` (B,) int32 its tokens.  Rows behind a sequence's end, and rows whose
    page id lies outside the cache, are zero.  Values are code * 2^(scale - 127),
    rounded once to ``dtype`` (fp32 and, but for the largest and smallest scales,
    bf16 hold them exactly).
    """
    return _lib.torch_ops().read_kv_cache(*cache, block_table, seq_lens, max_len, dtype)


def paged_attention(q: torch.Tensor, cache: PagedKVCache, block_table: torch.Tensor, seq_lens: torch.Tensor,
                    query_starts: torch.Tensor, *, max_query_len: int | None = None, sm_scale: float | None = None,
                    causal: bool = True, window: int | None = None, out: torch.Tensor | None = None,
                    return_lse: bool = False):
    """Attention of each sequence's new tokens over its cached keys and values.

    ``q`` (T, Hq, D) bf16 or fp16 holds the new tokens of all sequences, those of
    sequence b in rows ``query_starts[b]`` ... ``query_starts[b + 1]`` (int32 (B + 1,),
    ascending); they are the last of its ``seq_lens[b]`` tokens, whose keys and
    values are in the cache already (``write_kv_cache`` first).  ``block_table`` as in
    ``read_kv_cache``; lengths are cut to what it holds.  Hq is a multiple of the
    cache's heads, which neighbouring query heads share.

    ``causal``: a query sees the keys up to its own position, otherwise all of the
    sequence's (a chunk of frames that attends within itself).  ``window``: only the
    last ``window`` keys up to its position (and, not causal, those behind it).  Keys
    on pages whose id lies outside the cache are not seen.  A query that sees
    nothing gives zeros.

    ``max_query_len``: the most new tokens of a sequence, if known.  It picks the kernel
    (one token, or a chunk) and, with the table's width, the parts that the keys are
    cut into, and so the workspace (at most 1 GiB); a sequence may hold more, and
    results do not depend on it beyond rounding.  ``sm_scale``: 1/sqrt(D) by default, in 2^-64 ... 2^15.
    ``out``: takes the result, rows of no sequence left as they are (in a new tensor
    they are zero).  It may be ``q`` itself, or lie over parts of it (then q is copied
    first); with the other inputs it shares no memory, nor do its rows overlap.  ``return_lse``: also the natural
    log of each row's sum of exponentials, fp32 (T, Hq), -inf for a row that sees
    nothing.

    Scores, softmax and sums are fp32 on exact products of cached values and
    queries; P is rounded for the second product, to 11 bits or more down to 2^-21
    of the row's largest (single tokens: 16 bits), and the result once.  Over a cache in
    4 bits each query column is first taken to 2^-19 of the largest of its 32, or to
    2^-129 (bf16 holds columns down to 2^-11 of that exactly, fp16 to 2^-8); where eight
    or more of the 32 are below 2^-10 of the largest, to 2^-39 of it, or 2^-130, at a
    fifth (single tokens) to a half more time.  A NaN in a query makes its row NaN, in 4
    bits an infinity too.
    Values are right down to the smallest scales, 2^-127.  Averages stay finite up to the cache's largest values, 448 * 2^119 or 6 * 2^125.
    """
    out, lse = _lib.torch_ops().paged_attention(q, *cache, block_table, seq_lens, query_starts, max_query_len, sm_scale,
                                                causal, window, out, return_lse)
    return (out, lse) if return_lse else out


__all__ = ["PagedKVCache", "append_kv_cache", "empty_kv_cache", "paged_attention", "read_kv_cache", "write_kv_cache"]
