"""A quantised paged K/V cache and attention over it, on gfx950.

The cache holds K and V in the package's MXFP8 format (E4M3 codes, one E8M0
scale per 32 columns of a row: ``quant.mxfp8_qk_quant`` bit for bit below 3e38),
in pages that sequences take as they grow.  ``write_kv_cache`` quantises new rows into
it, ``paged_attention`` attends over it (one token of each sequence, or a chunk),
``read_kv_cache`` gives the values back, e.g. for ``fake_quant_attention``.

These are for inference: they have no backward pass and refuse inputs that ask
for one.  No call synchronises; all of them can be captured in a HIP graph.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import _lib
from ._ops import _dt
from .qk_norm import on_device, row_strides, rows_16b

BLOCK = 32  # columns of a scale
PAGE_SIZES = (16, 32, 64, 128, 256, 512, 1024)


class PagedKVCache(NamedTuple):
    """The tensors of a cache, contiguous, on one device.

    Row ``r`` of page ``p`` of head ``h`` is ``k_codes[p, h, r]``; its value is code *
    2^(scale - 127), ``k_scale[p, h, r, c]`` for columns 32 c ... 32 c + 31.
    """

    k_codes: torch.Tensor  # (pages, H, page size, D) float8_e4m3fn
    k_scale: torch.Tensor  # (pages, H, page size, D / 32) uint8, E8M0
    v_codes: torch.Tensor
    v_scale: torch.Tensor


def empty_kv_cache(num_pages: int, page_size: int, heads: int, head_dim: int, *, device="cuda") -> PagedKVCache:
    """A cache of zeros.  page_size: 16 to 1024 tokens, a power of two."""
    if head_dim not in (64, 128):
        raise ValueError(f"D must be 64 or 128; got {head_dim}")
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES}; got {page_size}")
    if num_pages <= 0 or heads <= 0:
        raise ValueError(f"num_pages and heads must be positive; got {num_pages} and {heads}")
    rows = (int(num_pages), int(heads), int(page_size))
    k, v = (torch.zeros((*rows, head_dim), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
            for _ in range(2))
    ks, vs = (torch.full((*rows, head_dim // BLOCK), 127, dtype=torch.uint8, device=device) for _ in range(2))
    return PagedKVCache(k, ks, v, vs)


def _check_cache(cache: PagedKVCache):
    """-> (pages, heads, page size, D, device index) of a cache that the kernels can take."""
    kc, ks, vc, vs = cache
    shape = kc.shape
    if len(shape) != 4:
        raise ValueError(f"cache codes must be (pages, H, page size, D); got {tuple(shape)}")
    n, h, page, d = shape
    if d not in (64, 128):
        raise ValueError(f"cache D must be 64 or 128; got {d}")
    if page not in PAGE_SIZES:
        raise ValueError(f"cache page size must be one of {PAGE_SIZES}; got {page}")
    sshape = (n, h, page, d // BLOCK)
    if vc.shape != shape or ks.shape != sshape or vs.shape != sshape:
        raise ValueError(f"cache tensors must be codes {tuple(shape)} and scales {sshape}; got "
                         f"{tuple(vc.shape)}, {tuple(ks.shape)} and {tuple(vs.shape)}")
    f8, u8 = torch.float8_e4m3fn, torch.uint8
    if kc.dtype != f8 or vc.dtype != f8 or ks.dtype != u8 or vs.dtype != u8:
        raise TypeError("cache codes must be float8_e4m3fn and scales uint8; got "
                        f"{kc.dtype}, {vc.dtype}, {ks.dtype} and {vs.dtype}")
    index = kc.get_device()
    if not kc.is_cuda or ks.get_device() != index or vc.get_device() != index or vs.get_device() != index:
        raise ValueError("cache tensors must live on one CUDA device")
    if not (kc.is_contiguous() and ks.is_contiguous() and vc.is_contiguous() and vs.is_contiguous()):
        raise ValueError("cache tensors must be contiguous")
    if n == 0 or h == 0:
        raise ValueError(f"the cache is empty: {tuple(shape)}")
    return n, h, page, d, index


def _set_cache(p, cache: PagedKVCache, num_pages: int, page: int) -> None:
    kc, ks, vc, vs = cache
    p.k_codes = kc.data_ptr(); p.k_scale = ks.data_ptr(); p.v_codes = vc.data_ptr(); p.v_scale = vs.data_ptr()
    p.num_pages = num_pages
    p.page_shift = page.bit_length() - 1


def _refuse_grad(who: str):
    raise ValueError(f"{who} has no backward pass; detach its inputs or call it under torch.no_grad()")


def _check_index(t: torch.Tensor, name: str, n: int, index: int, dtype) -> None:
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}; got {t.dtype}")
    if t.shape != (n,):
        raise ValueError(f"{name} must have shape {(n,)}; got {tuple(t.shape)}")
    if t.get_device() != index:
        raise ValueError(f"{name} must live on cuda:{index}; got {t.device}")


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
    values are finite, and what a query does not see cannot reach its result.
    """
    n, h, page, d, index = _check_cache(cache)
    shape = k.shape
    if len(shape) != 3 or shape[1] != h or shape[2] != d or v.shape != shape:
        raise ValueError(f"k and v must be (T, {h}, {d}); got {tuple(shape)} and {tuple(v.shape)}")
    if k.get_device() != index or v.get_device() != index:
        raise ValueError(f"k and v must live on the cache's cuda:{index}; got {k.device} and {v.device}")
    if v.dtype != k.dtype:
        raise TypeError(f"k and v must have one dtype; got {k.dtype} and {v.dtype}")
    dt = _dt(k)
    t = shape[0]
    _check_index(slots, "slots", t, index, torch.int64)
    if (k.requires_grad or v.requires_grad) and torch.is_grad_enabled():
        _refuse_grad("write_kv_cache")
    if t == 0:
        return
    k, v, slots = rows_16b(k), rows_16b(v), slots.contiguous()
    p = _lib.KvWriteParams()
    p.k = k.data_ptr(); p.v = v.data_ptr(); p.dtype = dt
    p.T = t; p.H = h; p.D = d
    p.k_t, p.k_h = row_strides(k)
    p.v_t, p.v_h = row_strides(v)
    p.slots = slots.data_ptr()
    _set_cache(p, cache, n, page)
    with on_device(index):
        _lib.check(_lib.load().lbfq_kv_write(p, _lib.stream_handle(k.device)), "lbfq_kv_write")


def _check_table(block_table: torch.Tensor, index: int) -> torch.Tensor:
    if block_table.ndim != 2 or block_table.dtype != torch.int32:
        raise TypeError(f"block_table must be (B, pages) int32; got {tuple(block_table.shape)} {block_table.dtype}")
    if block_table.get_device() != index:
        raise ValueError(f"block_table must live on the cache's cuda:{index}; got {block_table.device}")
    return block_table if block_table.stride(1) == 1 else block_table.contiguous()


def read_kv_cache(cache: PagedKVCache, block_table: torch.Tensor, seq_lens: torch.Tensor, max_len: int, *,
                  dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V of the first ``max_len`` tokens of each sequence, (B, max_len, H, D).

    ``block_table`` (B, pages) int32 lists each sequence's pages in order and
    ``seq_lens`` (B,) int32 its tokens.  Rows behind a sequence's end, and rows whose
    page id lies outside the cache, are zero.  Values are code * 2^(scale - 127),
    rounded once to ``dtype`` (fp32 and, but for the largest and smallest scales,
    bf16 hold them exactly).
    """
    n, h, page, d, index = _check_cache(cache)
    block_table = _check_table(block_table, index)
    b, cols = block_table.shape
    _check_index(seq_lens, "seq_lens", b, index, torch.int32)
    if dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"unsupported dtype {dtype}; expected float32, float16 or bfloat16")
    max_len = int(max_len)
    if max_len < 0:
        raise ValueError(f"max_len must not be negative; got {max_len}")
    k = torch.empty((b, max_len, h, d), dtype=dtype, device=block_table.device)
    v = torch.empty_like(k)
    if b == 0 or max_len == 0:
        return k, v
    seq_lens = seq_lens.contiguous()
    p = _lib.KvReadParams()
    _set_cache(p, cache, n, page)
    p.B = b; p.H = h; p.D = d; p.max_len = max_len
    p.block_table = block_table.data_ptr(); p.table_stride = block_table.stride(0)
    p.table_cols = cols
    p.seq_lens = seq_lens.data_ptr()
    p.k_out = k.data_ptr(); p.v_out = v.data_ptr(); p.dtype = _lib.DTYPE_CODE[dtype]
    with on_device(index):
        _lib.check(_lib.load().lbfq_kv_read(p, _lib.stream_handle(k.device)), "lbfq_kv_read")
    return k, v


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

    ``max_query_len``: the most new tokens of a sequence, if known; it sizes the
    launch, and results do not depend on it.  ``sm_scale``: 1/sqrt(D) by default, in 2^-64 ... 2^15.
    ``out``: takes the result, rows of no sequence left as they are (in a new tensor
    they are zero); it may not overlap the inputs.  ``return_lse``: also the natural
    log of each row's sum of exponentials, fp32 (T, Hq), -inf for a row that sees
    nothing.

    Scores, softmax and sums are fp32 on exact products of cached values and
    queries; P is rounded for the second product, to 11 bits or more down to 2^-21
    of the row's largest, and the result once.  A NaN in a query makes its row NaN.
    """
    n, hk, page, d, index = _check_cache(cache)
    shape = q.shape
    if len(shape) != 3 or shape[2] != d:
        raise ValueError(f"q must be (T, Hq, {d}); got {tuple(shape)}")
    if q.get_device() != index:
        raise ValueError(f"q must live on the cache's cuda:{index}; got {q.device}")
    if q.dtype != torch.bfloat16 and q.dtype != torch.float16:
        raise TypeError(f"q must be bfloat16 or float16; got {q.dtype}")
    t, hq, _ = shape
    if hq == 0 or hq % hk:
        raise ValueError(f"the query heads ({hq}) must be a multiple of the cache's ({hk})")
    block_table = _check_table(block_table, index)
    b, cols = block_table.shape
    if cols == 0:
        raise ValueError("block_table has no columns")
    _check_index(seq_lens, "seq_lens", b, index, torch.int32)
    _check_index(query_starts, "query_starts", b + 1, index, torch.int32)
    sm_scale = 1.0 / math.sqrt(d) if sm_scale is None else float(sm_scale)
    if not 2.0 ** -64 <= sm_scale <= 2.0 ** 15:
        raise ValueError(f"sm_scale must lie in 2^-64 ... 2^15; got {sm_scale}")
    if window is not None and window <= 0:
        raise ValueError(f"window must be positive; got {window}")
    if max_query_len is not None and max_query_len < 0:
        raise ValueError(f"max_query_len must not be negative; got {max_query_len}")
    if q.requires_grad and torch.is_grad_enabled():
        _refuse_grad("paged_attention")
    given = out is not None
    if given:
        if out.shape != shape or out.dtype != q.dtype or out.get_device() != index:
            raise ValueError(f"out must be {tuple(shape)} {q.dtype} on {q.device}; got {tuple(out.shape)} {out.dtype} "
                             f"on {out.device}")
        if rows_16b(out) is not out or any(st == 0 and m > 1 for st, m in zip(out.stride(), shape)):
            raise ValueError("out must have contiguous, distinct rows that start on 16-byte boundaries")
    else:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = q.new_empty((t, hq), dtype=torch.float32) if return_lse else None
    if b == 0 or t == 0:
        if not given:
            out.zero_()
        if return_lse:
            lse.fill_(-math.inf)
        return (out, lse) if return_lse else out
    q, seq_lens, query_starts = rows_16b(q), seq_lens.contiguous(), query_starts.contiguous()
    p = _lib.PagedParams()
    p.q = q.data_ptr(); p.dtype = _lib.DTYPE_CODE[q.dtype]
    p.T = t; p.Hq = hq; p.Hk = hk; p.D = d; p.B = b
    p.q_t, p.q_h = row_strides(q)
    _set_cache(p, cache, n, page)
    p.block_table = block_table.data_ptr(); p.table_stride = block_table.stride(0)
    p.table_cols = cols
    p.seq_lens = seq_lens.data_ptr(); p.query_starts = query_starts.data_ptr()
    p.max_query_len = max_query_len or 0
    p.sm_scale = sm_scale; p.causal = 1 if causal else 0
    p.window = min(int(window), 1 << 30) if window else 0
    p.out = out.data_ptr()
    p.out_t, p.out_h = row_strides(out)
    if return_lse:
        p.lse = lse.data_ptr()
    p.fill_rest = 0 if given else 1
    lib = _lib.load()
    with on_device(index):
        need = lib.lbfq_paged_attention_workspace_bytes(p)
        if need:
            ws = q.new_empty(need, dtype=torch.uint8)
            p.workspace = ws.data_ptr(); p.workspace_bytes = need
        _lib.check(lib.lbfq_paged_attention(p, _lib.stream_handle(q.device)), "lbfq_paged_attention")
    return (out, lse) if return_lse else out


__all__ = ["PagedKVCache", "empty_kv_cache", "paged_attention", "read_kv_cache", "write_kv_cache"]
