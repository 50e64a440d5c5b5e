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
