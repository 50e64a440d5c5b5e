"""Paged attention over 4 bits for queries whose columns lie far apart: where much of a block of 32 is below 2^-10 of its
largest, each column is kept to 2^-39 of that, whatever K has there.

Bounds: kv_reference.attend, to which is added what the query's terms leave (dq: 2^-39, or, where nothing lies so far apart,
2^-19 of the largest of 32 columns times sum |k_j| sm_scale: a score's error), and, as in
test_gpu_paged_attention_4bit.attend, 2^-32 sum |V_j| for weights that are fp16's smallest numbers."""

import math

import pytest
import torch

import kv4_reference as ref4
import kv_reference as ref
import test_gpu_paged_attention_4bit as four

pytestmark = pytest.mark.gpu


def far_apart(q):
    """Whether a row takes four more terms for some block of columns."""
    x = q.double().abs().unflatten(-1, (-1, 32))
    top = x.amax(-1, keepdim=True)
    return (((x > 0) & (x < top * 2.0 ** -10)).sum(-1) >= 8).any(-1)


def attend(q, cache, table, lens, starts, sm_scale=None, everywhere=False):
    cache = ref4.widen(cache)
    out, lse, tol, ltol = ref.attend(q, cache, table, lens, starts, sm_scale=sm_scale)
    bits = torch.where(far_apart(q) | everywhere, 2.0 ** -39, 2.0 ** -19)[..., None]
    for b in range(table.shape[0]):
        r = slice(int(starts[b]), int(starts[b + 1]))
        n = r.stop - r.start
        k, v = (torch.nan_to_num(ref.rows_of(cache[i], cache[i + 1], table[b], int(lens[b]))).abs() for i in (0, 2))
        g = q.shape[1] // v.shape[1]
        seen = ref.visible(n, v.shape[0], True, None, q.device).any(0)
        top = (bits[r] * q[r].double().abs().unflatten(-1, (-1, 32)).amax(-1)).repeat_interleave(32, -1)
        kt = k[seen].permute(1, 2, 0).repeat_interleave(g, 0).contiguous()
        dq = torch.bmm(top.transpose(0, 1).contiguous(), kt).amax(-1).t() * (sm_scale or 1.0 / math.sqrt(q.shape[2]))
        tol[r] += 2 * dq[..., None] * v[seen].amax(0).repeat_interleave(g, 0) + 2.0 ** -32 * v[seen].sum(0).repeat_interleave(g, 0)
        ltol[r] += dq
    return out, lse, tol, ltol


def run_and_check(args, what, hint, rows=slice(None), **kw):
    from low_bit_fake_quant import paged_attention
    sm = kw.get("sm_scale")
    out, lse = paged_attention(*args, max_query_len=hint, return_lse=True, sm_scale=sm)
    want, wlse, tol, ltol = attend(*args, **kw)
    ref.check(out[rows], want[rows], tol[rows], what)
    ref.check(lse[rows], wlse[rows], ltol[rows], what + " lse")


def widened(q, kind, rows=slice(None)):
    """q with columns far apart; the largest of each block of 32 are of one size."""
    big = 4000.0 if q.dtype == torch.bfloat16 else 1000.0
    sign = torch.where(q >= 0, 1.0, -1.0)
    x = q.clone()
    if kind in ("first", "hidden"):  # one column of each block
        x[rows, :, ::32] = (big * sign[rows, :, ::32]).to(q.dtype)
    elif kind == "several":
        x[rows, :, 3::7] = (big * sign[rows, :, 3::7]).to(q.dtype)
    elif kind == "block":  # the second block only
        x[rows, :, 33] = big
    elif kind == "steps":  # each column half as large as the one before, down to fp16's smallest
        i = torch.arange(q.shape[-1], device=q.device) % 32
        x[rows] = (sign[rows] * torch.exp2(8.0 - i.clamp(max=31 if q.dtype == torch.bfloat16 else 22))).to(q.dtype)
    return x


def problem(gpu, kind, dtype, d, lens, counts, **kw):
    args = four.problem(gpu, lens=lens, counts=counts, d=d, dtype=dtype, garbage=False, qscale=1.0, **kw)
    if kind in ("hidden", "steps"):  # K is 0 in the largest column
        args[1][0].view(torch.uint8)[..., ::16] &= 0xF0
    return args


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,L", [(1, 150), (1, 5000), (40, 150), (40, 3000)])
@pytest.mark.parametrize("kind", ["first", "hidden", "several", "block", "steps"])
def test_columns_far_apart(gpu, kind, n, L, d, dtype):
    q, cache, table, lens, starts = problem(gpu, kind, dtype, d, [L, L - 60], [n, n])
    q = widened(q, kind)
    assert far_apart(q).all()
    run_and_check((q, cache, table, lens, starts), kind, n, sm_scale=0.001 if kind in ("first", "several", "block") else 0.1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,hint", [(1, 1), (12, 1), (200, 200)])
def test_one_row_among_ordinary_ones(gpu, n, hint, d, dtype):
    """(12 tokens of two heads for the kernel of single tokens: two rounds of 16 rows)"""
    q, cache, table, lens, starts = problem(gpu, "hidden", dtype, d, [400, 300, 350], [n, n, n])
    for row in (0, 2 * n - 1, 3 * n - 1):
        x = widened(q, "hidden", slice(row, row + 1))
        assert int(far_apart(x).any(-1).sum()) == 1
        run_and_check((x, cache, table, lens, starts), f"row {row}", hint, sm_scale=0.1)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_rows_that_are_not_numbers_stay_alone(gpu, value, n, d):
    from low_bit_fake_quant import paged_attention
    q, cache, table, lens, starts = problem(gpu, "hidden", torch.bfloat16, d, [150, 140], [n, n])
    x = widened(q, "hidden")
    x[0, 1, 5] = value
    out = paged_attention(x, cache, table, lens, starts, max_query_len=n, sm_scale=0.1)
    assert torch.isnan(out[0, 1]).all() and int(torch.isnan(out).sum()) == d
    x[0] = widened(q, "hidden")[0]
    want = paged_attention(x, cache, table, lens, starts, max_query_len=n, sm_scale=0.1)
    assert torch.equal(out[1:], want[1:]) and torch.equal(out[0, ::3], want[0, ::3])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("n", [1, 40])
def test_the_smallest_queries(gpu, n, dtype):
    """Columns far apart next to the dtype's smallest numbers (scores of nothing: an average of V)."""
    q, cache, table, lens, starts = problem(gpu, "steps", dtype, 128, [150, 90], [n, n])
    q = widened(q, "steps") * 2.0 ** (-10 if dtype == torch.float16 else -115)
    run_and_check((q, cache, table, lens, starts), "small", n, sm_scale=2.0 ** 15, everywhere=True)


@pytest.mark.parametrize("n", [1, 40])
def test_with_scales_of_v_far_apart(gpu, n):
    q, cache, table, lens, starts = problem(gpu, "hidden", torch.bfloat16, 128, [700, 90], [n, n])
    g = torch.Generator().manual_seed(4)
    cache[3].copy_(torch.randint(60, 160, cache[3].shape, generator=g, dtype=torch.uint8).to(gpu))
    run_and_check((widened(q, "hidden"), cache, table, lens, starts), "both", n, sm_scale=0.1)
