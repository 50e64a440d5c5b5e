"""Where paged attention's `out` may lie: rows of its own, anywhere; q's rows; not over itself or other inputs."""

import pytest
import torch

import kv_reference as ref
from test_gpu_paged_attention import problem

pytestmark = pytest.mark.gpu

CASES = [(1, 300), (1, 5000), (70, 200), (70, 5000)]  # one token and a chunk, keys in one part and in several


def inputs(dev, n, L):
    return problem(dev, lens=[L, L // 2], counts=[n, n], page=32, tail=3, garbage=False)


@pytest.mark.parametrize("n,L", CASES)
def test_out_over_the_queries(gpu, n, L):
    """q itself; q's memory from the next token or head on; other columns of one buffer; q's memory in another order.
    The result is that of a tensor of its own."""
    from low_bit_fake_quant import paged_attention
    q, cache, table, lens, starts = inputs(gpu, n, L)
    T, hq, d = q.shape
    used = int(starts[-1])
    call = lambda q, out: paged_attention(q, cache, table, lens, starts, max_query_len=n, out=out)  # noqa: E731
    want = call(q, torch.zeros_like(q))

    def places():
        flat = torch.zeros((T + 1) * (2 * hq + 1) * d, dtype=q.dtype, device=gpu)
        part = lambda off, st: flat.as_strided((T, hq, d), (*st, 1), off)  # noqa: E731
        whole = (hq * d, d)
        yield "itself", part(0, whole), part(0, whole)
        yield "a token on", part(0, whole), part(hq * d, whole)
        yield "a token back", part(hq * d, whole), part(0, whole)
        yield "a head on", part(0, whole), part(d, whole)
        yield "half a row on", part(0, whole), part(d // 2, whole)
        yield "other columns", part(0, (2 * hq * d, d)), part(hq * d, (2 * hq * d, d))
        yield "columns that meet", part(0, (2 * hq * d, d)), part((hq - 1) * d, (2 * hq * d, d))
        yield "another order", part(0, whole), part(0, (d, T * d))

    for what, x, out in places():
        x.copy_(q)
        keep = out.clone()
        got = call(x, out)
        assert got.data_ptr() == out.data_ptr()
        assert torch.equal(out[:used], want[:used]), what
        assert torch.equal(out[used:], keep[used:]), what
    ref.check(want[:used], *[x[:used] for i, x in enumerate(ref.attend(q, cache, table, lens, starts)) if i in (0, 2)], "own")


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


def test_out_in_other_inputs_memory_is_refused(gpu):
    from low_bit_fake_quant import paged_attention
    q, cache, table, lens, starts = inputs(gpu, 2, 40)
    T, hq, d = q.shape
    whole = torch.zeros(4 * T * hq * d, dtype=torch.uint8, device=gpu)
    out = whole[:2 * T * hq * d].view(q.dtype).view(T, hq, d)
    # what lies right behind it is not shared
    behind = whole[2 * T * hq * d:][:8 * lens.numel()].view(torch.int32)[:lens.numel()]
    behind.copy_(lens)
    want = paged_attention(q, cache, table, lens, starts)
    assert torch.equal(paged_attention(q, cache, table, behind, starts, out=out)[:4], want[:4])
    i32 = out.flatten().view(torch.int32)
    for kw in (dict(table=i32[-table.numel():].view_as(table).copy_(table)), dict(lens=i32[4:4 + lens.numel()].copy_(lens)),
               dict(starts=i32[-starts.numel():].copy_(starts))):
        a = dict(table=table, lens=lens, starts=starts)
        a.update(kw)
        with pytest.raises(ValueError, match="share memory"):
            paged_attention(q, cache, a["table"], a["lens"], a["starts"], out=out)
    for t in cache:
        own = t.view(torch.uint8).flatten()
        room = torch.zeros(2 * T * hq * d, dtype=torch.uint8, device=gpu)
        if own.numel() >= room.numel():
            o = own[:room.numel()].view(q.dtype).view(T, hq, d)
            with pytest.raises(ValueError, match="share memory"):
                paged_attention(q, cache, table, lens, starts, out=o)


def test_out_over_the_queries_of_workgroups_that_start_later(gpu):
    """More workgroups than run at a time: the first results are there before the last queries are read."""
    from low_bit_fake_quant import paged_attention
    n = 3000
    q, cache, table, lens, starts = problem(gpu, lens=[n], counts=[n], hq=64, hk=64, page=64, garbage=False)
    want = paged_attention(q, cache, table, lens, starts)
    flat = torch.zeros(n + 1, 64, 128, dtype=q.dtype, device=gpu)
    for x, out in ((flat[1:], flat[:-1]), (flat[:-1], flat[1:]), (flat[:-1], flat[:-1])):
        x.copy_(q)
        paged_attention(x, cache, table, lens, starts, out=out)
        assert torch.equal(out, want)
