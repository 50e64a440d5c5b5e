"""Paged attention over 4 bits of one sequence whose row tiles fill more than half of the chip, but not all of it: a long
and a short part of the keys (which each test makes sure of).  Bounds: test_gpu_paged_attention_4bit.attend."""

import pytest
import torch

import kv_reference as ref
import test_gpu_paged_attention_4bit as four
import test_paged_plan_unequal_cpu as plans

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


@pytest.mark.parametrize("n,L,cols,hq,hk,d,dtype,causal,window,before,behind", [
    (2700, 8150, 128, 16, 16, 128, BF, False, None, 0, 0),
    (2700, 8192, 128, 16, 16, 128, BF, False, None, 5, 0),  # rows of no sequence in front
    (2690, 8129, 128, 16, 16, 128, FP, False, None, 0, 9),  # and behind
    (2900, 8192, 128, 16, 16, 128, FP, True, None, 0, 0),
    (2700, 8150, 128, 16, 16, 128, BF, True, 7000, 0, 0),
    (1400, 8177, 128, 32, 8, 128, BF, False, None, 0, 0),  # shared heads
    (2700, 6100, 96, 24, 24, 64, FP, False, None, 0, 0),
    (2700, 6144, 96, 24, 24, 64, BF, True, None, 3, 0),
    (2700, 3000, 128, 16, 16, 128, BF, False, None, 0, 0),  # much shorter than its table
    (2700, 2800, 128, 16, 16, 128, BF, True, None, 0, 0),
    (2700, 130, 128, 16, 16, 128, BF, False, None, 0, 0),  # less than a part's least
    (2700, 30, 128, 16, 16, 128, BF, True, None, 0, 0),  # and most queries see nothing
    (2700, 0, 128, 16, 16, 128, BF, False, None, 0, 0)])
def test_two_unequal_parts(gpu, n, L, cols, hq, hk, d, dtype, causal, window, before, behind):
    from low_bit_fake_quant import _lib, paged_attention
    parts, share = plans.plan(_lib.load(), n + before + behind, 64 * cols, hq=hq, hk=hk, d=d, causal=causal, window=window,
                              dtype=1 if dtype == FP else 2)
    assert parts == 2 and share > 0
    q, cache, table, lens, starts = four.problem(gpu, lens=[L], counts=[n], hq=hq, hk=hk, d=d, dtype=dtype, page=64, cols=cols,
                                                 tail=before + behind, garbage=L != 8150)
    q, starts = torch.roll(q, before, 0), starts + before
    out, lse = paged_attention(q, cache, table, lens, starts, causal=causal, window=window, return_lse=True)
    g, step = hq // hk, 4
    for h in range(0, hk, step):
        part = type(cache)(*(t.view(torch.uint8)[:, h:h + step].contiguous().view(t.dtype) for t in cache))
        rows = slice(g * h, g * (h + step))
        want, wlse, tol, ltol = four.attend(q[:, rows].contiguous(), part, table, lens, starts, causal=causal, window=window)
        ref.check(out[:, rows], want, tol, "out")
        ref.check(lse[:, rows], wlse, ltol, "lse")
