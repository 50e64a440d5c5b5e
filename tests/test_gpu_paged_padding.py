"""Paged attention in token buffers much longer than their sequences."""

import pytest
import torch

import kv_reference as ref
from test_gpu_paged_attention import problem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 100])
def test_a_buffer_of_2_26_rows(gpu, n):
    """Over 2^32 elements; the rows of the sequences are within their bounds, the others empty."""
    from low_bit_fake_quant import paged_attention
    q, cache, table, lens, starts = problem(gpu, lens=[4000, 900], counts=[n, n], hq=32, hk=8, d=64, page=64, garbage=False)
    T, at = (1 << 21) + 3, (1 << 21) - 2 * n
    big = torch.empty(T, 32, 64, dtype=q.dtype, device=gpu)
    big[at:at + 2 * n] = q
    out, lse = paged_attention(big, cache, table, lens, starts + at, max_query_len=n, return_lse=True)
    want, wlse, tol, ltol = ref.attend(q, cache, table, lens, starts)
    ref.check(out[at:at + 2 * n], want, tol, "rows")
    ref.check(lse[at:at + 2 * n], wlse, ltol, "lse")
    assert torch.isneginf(lse[:at]).all() and torch.isneginf(lse[at + 2 * n:]).all()
    for i in range(0, at, 1 << 18):
        assert not out[i:min(at, i + (1 << 18))].any()
    assert not out[at + 2 * n:].any()


@pytest.mark.parametrize("n,hq,hk,d,dtype", [(1, 5, 5, 64, torch.bfloat16), (1, 32, 8, 128, torch.float16), (40, 3, 1, 64, torch.float16),
                                             (200, 12, 12, 128, torch.bfloat16)])
@pytest.mark.parametrize("before,behind", [(0, 1), (0, 3000), (1, 0), (2500, 0), (700, 1501), (9000, 9000)])
def test_every_row_of_no_sequence_is_empty(gpu, before, behind, n, hq, hk, d, dtype):
    from low_bit_fake_quant import paged_attention
    q, cache, table, lens, starts = problem(gpu, lens=[90, 60], counts=[n, n], hq=hq, hk=hk, d=d, dtype=dtype, garbage=False)
    big = torch.cat([q.new_zeros(before, hq, d), q, q.new_zeros(behind, hq, d)])
    junk = [torch.full_like(big, float("nan")), torch.full(big.shape[:2], 7.0, device=gpu)]  # what new memory may hold
    del junk
    out, lse = paged_attention(big, cache, table, lens, starts + before, max_query_len=n, return_lse=True)
    want, wlse, tol, ltol = ref.attend(q, cache, table, lens, starts)
    rows = slice(before, before + 2 * n)
    ref.check(out[rows], want, tol, "rows")
    ref.check(lse[rows], wlse, ltol, "lse")
    rest = torch.ones(big.shape[0], dtype=torch.bool, device=gpu)
    rest[rows] = False
    assert torch.equal(out[rest], torch.zeros_like(out[rest])) and torch.isneginf(lse[rest]).all()
    kept = torch.full_like(big, 3.0)
    got, l2 = paged_attention(big, cache, table, lens, starts + before, max_query_len=n, return_lse=True, out=kept)
    assert torch.equal(got[rows], out[rows]) and (got[rest] == 3).all() and torch.equal(l2, lse)


def test_filling_a_padded_buffer_takes_no_longer_than_memory_does(gpu):
    """A call in a buffer of 30000 more tokens, beside the call without them and zeroing such a buffer: a tenth of the
    chip's workgroups on the job would show."""
    from low_bit_fake_quant import paged_attention
    q, cache, table, lens, starts = problem(gpu, lens=[100], counts=[64], hq=32, hk=8, page=64, garbage=False)
    big = torch.cat([q, q.new_zeros(30000, 32, 128)])

    def least(call):
        times = []
        for _ in range(12):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            call()
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    alone = least(lambda: paged_attention(q, cache, table, lens, starts)) + least(lambda: torch.zeros_like(big))
    assert least(lambda: paged_attention(big, cache, table, lens, starts)) < 10 * alone
