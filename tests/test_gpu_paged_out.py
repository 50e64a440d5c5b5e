"""Where paged attention's `out` may lie: rows of its own, in any order, not over each other."""

import pytest
import torch

from test_gpu_paged_attention import problem

pytestmark = pytest.mark.gpu


def inputs(dev, n, L):
    return problem(dev, lens=[L, L // 2], counts=[n, n], page=32, tail=3, garbage=False)


def test_rows_that_are_apart_in_any_order_are_taken(gpu):
    from low_bit_fake_quant import paged_attention
    q, cache, table, lens, starts = inputs(gpu, 2, 40)
    q, d = q[:4].clone(), 128
    want = paged_attention(q, cache, table, lens, starts, max_query_len=2)
    for strides in ((4 * d, d), (d, 4 * d), (5 * d, 3 * d + 8), (3 * d, 4 * d), (4 * d + 8, 3 * d), (7 * d, 2 * d)):
        flat = torch.zeros(40 * d, dtype=q.dtype, device=gpu)
        out = flat.as_strided((4, 4, d), (*strides, 1))
        starts_of = sorted(i * strides[0] + j * strides[1] for i in range(4) for j in range(4))
        apart = all(b - a >= d for a, b in zip(starts_of, starts_of[1:]))
        if apart:
            assert torch.equal(paged_attention(q, cache, table, lens, starts, max_query_len=2, out=out), want), strides
        else:
            with pytest.raises(ValueError, match="distinct rows"):
                paged_attention(q, cache, table, lens, starts, max_query_len=2, out=out)


@pytest.mark.parametrize("strides", [(128, 128), (256, 128), (512, 64), (512, 120), (64, 512), (384, 128), (0, 128), (512, 0),
                                     (136, 264)])
def test_rows_that_overlap_are_refused(gpu, strides):
    from low_bit_fake_quant import paged_attention
    q, cache, table, lens, starts = inputs(gpu, 2, 40)
    out = torch.zeros(8000, dtype=q.dtype, device=gpu).as_strided((q.shape[0], 4, 128), (*strides, 1))
    with pytest.raises(ValueError, match="distinct rows"):
        paged_attention(q, cache, table, lens, starts, out=out)
    assert not out.any()
