"""Paged attention where the values that queries see are as small as the cache's scales go, 2^-127: in all
columns, in some blocks of 32 beside larger ones, and with larger ones in front of them.  Over both widths
of the cache, one token and a chunk, the keys in one part and in several.  Bounds: kv_reference.attend."""

import pytest
import torch

import kv_reference as ref
import test_gpu_paged_attention as eight
import test_gpu_paged_attention_4bit as four
import test_gpu_paged_large_values as large_values

pytestmark = pytest.mark.gpu


def run_and_check(bits, args, what, n):
    from low_bit_fake_quant import paged_attention
    out, lse = paged_attention(*args, max_query_len=n, return_lse=True)
    want, wlse, tol, ltol = (ref if bits == 8 else four).attend(*args)
    large_values.check(out, want, tol, what)
    ref.check(lse, wlse, ltol, what + " lse")


def problem(gpu, bits, n, L, d, dtype=torch.bfloat16):
    lens = [L, L - L // 3]
    return (eight if bits == 8 else four).problem(gpu, lens=lens, counts=[n, n], d=d, dtype=dtype, page=64, garbage=False,
                                                  qscale=0.3)


SIZES = [(1, 90), (1, 5000), (40, 100), (40, 3000)]


@pytest.mark.parametrize("n,L", SIZES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("low,high", [(0, 2), (1, 20), (0, 31), (31, 33), (40, 44), (0, 90), (150, 170)])
def test_small_scales(gpu, low, high, bits, d, n, L):
    args = problem(gpu, bits, n, L, d)
    scale = args[1][3]
    pick = torch.randint(low, high + 1, scale.shape, generator=torch.Generator().manual_seed(low + high), dtype=torch.uint8)
    scale.copy_(pick.to(gpu))
    run_and_check(bits, args, f"scales {low} ... {high}", n)


@pytest.mark.parametrize("n,L", SIZES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("small,large", [((0, 6), (24, 31)), ((0, 31), (110, 130)), ((3, 20), (200, 246))])
def test_blocks_of_columns_far_apart(gpu, small, large, dtype, bits, d, n, L):
    """The first block's scales are small for all keys, the last's large."""
    args = problem(gpu, bits, n, L, d, dtype)
    scale = args[1][3]
    g = torch.Generator().manual_seed(7)
    for block, (low, high) in ((0, small), (-1, large)):
        scale[..., block] = torch.randint(low, high + 1, scale.shape[:-1], generator=g, dtype=torch.uint8).to(gpu)
    run_and_check(bits, args, f"{small} beside {large}", n)


@pytest.mark.parametrize("n,L", SIZES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("order", ["up", "down", "one"])
def test_scales_that_grow_or_fall_along_the_keys(gpu, order, bits, d, n, L):
    """From 20 to 240 over the sequence's keys, back, or at one key alone; each block's a little different."""
    args = problem(gpu, bits, n, L, d)
    _, cache, table, lens, _ = args
    scale = cache[3]
    for b in range(2):
        length = int(lens[b])
        at = torch.arange(length)
        x = at * 220 // length + 20
        x = {"up": x, "down": 260 - x, "one": torch.where(at == length // 2, 230, 25)}[order]
        x = (x[:, None, None] + torch.arange(d // 32)).to(torch.uint8).expand(length, 2, d // 32).to(gpu)
        page = table[b].long()[at.to(gpu) // 64]
        scale[page, :, at.to(gpu) % 64] = x
    run_and_check(bits, args, order, n)


@pytest.mark.parametrize("n,L", [(1, 300), (40, 300), (200, 2500)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("causal,window", [(True, None), (True, 70), (False, 33), (False, None)])
def test_masks_over_scales_far_apart(gpu, causal, window, bits, d, n, L):
    """Windows, pages that are not there, shared heads, more new tokens than a sequence has, rows behind the last one; what no
    query sees has any bytes, scales of 255 among them."""
    from low_bit_fake_quant import paged_attention
    lens, counts = [L, 0, 17, L // 2], [n, n, n, min(n, 5)]
    args = (eight if bits == 8 else four).problem(gpu, lens=lens, counts=counts, hq=6, d=d, page=16, tail=3, qscale=0.3)
    q, cache, table, sl, starts = args
    g = torch.Generator().manual_seed(d + n)
    table[0, 1] = -1
    table[3, 2] = cache[0].shape[0] + 5
    for b, length in enumerate(lens):
        at = torch.arange(length, device=gpu)
        page = table[b].long()[at // 16]
        there = (page >= 0) & (page < cache[0].shape[0])
        low = torch.tensor([0, 60, 20, 30])[:d // 32]  # a stretch of 100 scales, another for each block
        x = (torch.randint(0, 100, (length, 2, d // 32), generator=g) + low).to(torch.uint8).to(gpu)
        cache[3][page[there], :, at[there] % 16] = x[there]
    out, lse = paged_attention(*args, max_query_len=n, causal=causal, window=window, return_lse=True)
    want, wlse, tol, ltol = (ref if bits == 8 else four).attend(*args, causal=causal, window=window)
    large_values.check(out, want, tol, "out")
    ref.check(lse, wlse, ltol, "lse")
