"""Paged attention against its definition in 64 bits, at the lengths, masks, head
layouts and page sizes where it can go wrong; the bounds are those of its roundings
(kv_reference.attend)."""

import math

import pytest
import torch

import kv_reference as ref
from conftest import cpu_randn

pytestmark = pytest.mark.gpu


def problem(dev, *, lens, counts, hq=4, hk=2, d=128, page=16, dtype=torch.bfloat16, tail=0, seed=0, qscale=2.0,
            vscale=None, cols=None, garbage=True):
    """A cache whose unwritten rows and pages hold arbitrary bytes (NaN codes and
    scales among them), a shuffled table, queries; written rows are random with
    per-channel bias."""
    from low_bit_fake_quant import PagedKVCache, write_kv_cache
    B = len(lens)
    cols = cols or max(1, -(-max(lens) // page))
    pages = B * cols + 2
    g = torch.Generator().manual_seed(seed)
    by = lambda *s: (torch.randint(0, 256, s, generator=g, dtype=torch.uint8) if garbage else  # noqa: E731
                     torch.zeros(s, dtype=torch.uint8)).to(dev)
    f8 = torch.float8_e4m3fn
    cache = PagedKVCache(by(pages, hk, page, d).view(f8), by(pages, hk, page, d // 32),
                         by(pages, hk, page, d).view(f8), by(pages, hk, page, d // 32))
    if garbage:
        for t in (cache[0], cache[2]):
            t.view(torch.uint8)[:, :, ::3] = 0x7F
        for t in (cache[1], cache[3]):
            t[:, :, ::2] = 0xFF
    table = torch.randperm(pages, generator=g)[:B * cols].view(B, cols).int()
    slots = torch.tensor([int(table[b, j // page]) * page + j % page for b, n in enumerate(lens) for j in range(n)],
                         dtype=torch.int64)
    T = slots.numel()
    if T:
        k = torch.randn(T, hk, d, generator=g) + 2 * torch.randn(1, hk, d, generator=g)
        v = torch.randn(T, hk, d, generator=g) + torch.randn(1, hk, d, generator=g)
        if vscale is not None:
            v = v * vscale(T, g).view(T, 1, 1)
        write_kv_cache(k.to(dev), v.to(dev), cache, slots.to(dev))
    starts = torch.tensor([0] + counts).cumsum(0).int()
    q = (torch.randn(int(starts[-1]) + tail, hq, d, generator=g) * qscale).to(dtype)
    i32 = lambda t: torch.as_tensor(t, dtype=torch.int32).to(dev)  # noqa: E731
    return q.to(dev), cache, i32(table), i32(lens), i32(starts)


def run_and_check(args, what, hint=None, **kw):
    from low_bit_fake_quant import paged_attention
    out, lse = paged_attention(*args, max_query_len=hint, return_lse=True, **kw)
    want, wlse, tol, ltol = ref.attend(*args, **kw)
    ref.check(out, want, tol, what)
    ref.check(lse, wlse, ltol, what + " lse")
    return out, lse


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [1, 2, 5, 33])
def test_lengths_around_every_edge(gpu, n, d, dtype):
    """Up to n new tokens (more than the sequence holds for the short ones: rows
    that see nothing) over lengths around the pages' and tiles' ends."""
    args = problem(gpu, lens=EDGES, counts=[n] * len(EDGES), d=d, dtype=dtype, tail=3, seed=n)
    run_and_check(args, f"n={n}", hint=n)


@pytest.mark.parametrize("hq,hk", [(1, 1), (5, 5), (6, 2), (14, 2), (16, 1), (40, 2), (12, 12)])
@pytest.mark.parametrize("n", [1, 3, 70])
def test_shared_heads(gpu, n, hq, hk):
    args = problem(gpu, lens=[200, 77], counts=[n, max(1, n // 2)], hq=hq, hk=hk, d=64, page=32, seed=hq)
    run_and_check(args, f"{hq}/{hk}", hint=n)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 512, 1024])
@pytest.mark.parametrize("n", [1, 20])
def test_page_sizes(gpu, page, n):
    args = problem(gpu, lens=[1300, 1024, 3], counts=[n, n, n], page=page, seed=page, hq=3, hk=3)
    run_and_check(args, f"page {page}", hint=n)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [None, 1, 7, 64, 100, 5000])
@pytest.mark.parametrize("n", [1, 4, 150])
def test_masks(gpu, n, window, causal):
    args = problem(gpu, lens=[700, 65, 150, 9], counts=[n, n, min(n, 150), n], seed=n, page=32,
                   dtype=torch.float16 if n == 4 else torch.bfloat16)
    run_and_check(args, f"window {window} causal {causal}", hint=n, causal=causal, window=window)


@pytest.mark.parametrize("n", [1, 40])
def test_long_sequences_split_over_workgroups(gpu, n):
    args = problem(gpu, lens=[9000, 1, 5000], counts=[n, 1, n], page=64, tail=2, garbage=False)
    run_and_check(args, "long", hint=n)
    run_and_check(args, "long, no hint")
    run_and_check(args, "long, hint too small", hint=1)


def test_a_wide_table_and_short_sequences(gpu):
    """Most parts of the keys are empty: their sums are never written nor read."""
    args = problem(gpu, lens=[70, 3, 0], counts=[1, 1, 1], cols=3000)
    for _ in range(2):
        junk = torch.full((1 << 22,), math.nan, device=gpu)  # what a workspace may hold
        del junk
        run_and_check(args, "wide", hint=1)


@pytest.mark.parametrize("B,most,hq,hk,d", [(70, 40, 8, 2, 128), (150, 1, 4, 2, 64), (300, 19, 3, 3, 64),
                                            (4200, 18, 2, 1, 64)])
def test_many_ragged_sequences(gpu, B, most, hq, hk, d):
    """More sequences than a wave has lanes, and than 64 waves have: where each row
    tile belongs is found in two and in three looks.  Most have one new token, some none."""
    g = torch.Generator().manual_seed(B)
    counts = [[0, 1, 1, most][int(i)] for i in torch.randint(0, 4, (B,), generator=g)]
    counts[-1] = most
    lens = [int(n) for n in torch.randint(0, 40, (B,), generator=g)]
    args = problem(gpu, lens=lens, counts=counts, hq=hq, hk=hk, d=d, tail=2, garbage=False)
    run_and_check(args, f"{B} sequences", hint=most)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
def test_many_rows_of_few_parts(gpu, d, dtype):
    """Thousands of rows whose keys are split: several rows to a wave of the kernel that joins the parts."""
    args = problem(gpu, lens=[5000, 3100, 40], counts=[601, 300, 50], hq=6, hk=2, d=d, dtype=dtype, page=64, tail=2,
                   garbage=False)
    run_and_check(args, "joined", hint=601)
    run_and_check(args, "joined, no hint, window", window=900)


@pytest.mark.parametrize("n", [3, 200])
def test_rows_before_the_first_sequence(gpu, n):
    from low_bit_fake_quant import paged_attention
    q, cache, table, lens, starts = problem(gpu, lens=[400, 300, 7], counts=[n, n // 2, 1], tail=9)
    want, wl = paged_attention(q, cache, table, lens, starts, max_query_len=n, return_lse=True)
    q2 = torch.cat([q[-5:], q[:-5]])
    out, lse = paged_attention(q2, cache, table, lens, starts + 5, max_query_len=n, return_lse=True)
    assert torch.equal(out[5:], want[:-5]) and torch.equal(lse[5:], wl[:-5])
    assert not out[:5].any() and torch.isneginf(lse[:5]).all()
    one, l1 = paged_attention(q2[:5 + n], cache, table[:1], lens[:1], starts[:2] + 5, return_lse=True)
    ref.check(one[5:], *[x for i, x in enumerate(ref.attend(q[:n], cache, table[:1], lens[:1], starts[:2])) if i in (0, 2)],
              "one sequence")
    assert not one[:5].any() and torch.isneginf(l1[:5]).all()


@pytest.mark.parametrize("n", [1, 33])
def test_missing_pages_are_not_seen(gpu, n):
    q, cache, table, lens, starts = problem(gpu, lens=[200, 64, 40], counts=[n, n, n])
    table[0, 3], table[0, 7], table[1, 0] = -1, 1 << 30, table.shape[1] * 3 + 2
    table[2, :] = -1
    run_and_check((q, cache, table, lens, starts), "missing pages", hint=n)


@pytest.mark.parametrize("n", [1, 33])
def test_lengths_beyond_the_table_are_cut(gpu, n):
    q, cache, table, lens, starts = problem(gpu, lens=[64, 32], counts=[n, n])
    from low_bit_fake_quant import paged_attention
    cut = table[:, :2].contiguous()
    want = paged_attention(q, cache, cut, lens.clamp(max=32), starts, max_query_len=n)
    assert torch.equal(paged_attention(q, cache, cut, lens, starts, max_query_len=n), want)
    assert torch.equal(paged_attention(q, cache, table[:, :2], lens + 5000, starts, max_query_len=n), want)
    neg = paged_attention(q, cache, table, -lens, starts, max_query_len=n)
    assert not neg.any()


@pytest.mark.parametrize("n", [1, 50])
def test_nan_codes_that_no_row_sees(gpu, n):
    """Rows that a window excludes for every query, and rows behind the end, may
    hold anything: the result's bits do not change."""
    from low_bit_fake_quant import paged_attention
    q, cache, table, lens, starts = problem(gpu, lens=[300], counts=[n], garbage=False, cols=20)
    run = lambda: paged_attention(q, cache, table, lens, starts, window=40, max_query_len=n)  # noqa: E731
    want = run()
    page = 16
    for j in list(range(0, 300 - n - 40 + 1)) + list(range(300, 320)):
        p, r = int(table[0, j // page]), j % page
        for t in cache:
            t.view(torch.uint8)[p, :, r] = 0x7F if t.dtype != torch.uint8 else 0xFF
    got = run()
    assert torch.equal(got, want)
    ref.check(got, *[x for i, x in enumerate(ref.attend(q, type(cache)(*(t.clone() for t in cache)), table, lens, starts,
                                                       window=40)) if i in (0, 2)], "window")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("n", [2, 4, 40])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan"), 3e38, 1e20])
def test_huge_and_not_finite_keys_and_values_in_masked_places(gpu, bad, n, dtype):
    """The last token's K and V hold infinities, NaN or huge values: the queries
    before it do not see it, and their results are what they are without it."""
    from low_bit_fake_quant import paged_attention, write_kv_cache
    q, cache, table, lens, starts = problem(gpu, lens=[130, 75], counts=[n, n], dtype=dtype, garbage=False)
    run = lambda: paged_attention(q, cache, table, lens, starts, max_query_len=n, return_lse=True)  # noqa: E731
    out, lse = run()
    x = torch.ones(2, 2, 128, device=gpu)
    x[:, :, ::3] = bad
    slots = torch.tensor([int(table[b, (L - 1) // 16]) * 16 + (L - 1) % 16 for b, L in enumerate((130, 75))], device=gpu)
    write_kv_cache(x, x, cache, slots)
    got, gl = run()
    want, wlse, tol, ltol = ref.attend(q, cache, table, lens, starts)
    before = [i for i in range(2 * n) if i % n != n - 1]
    ref.check(got[before], want[before], tol[before], "before")
    ref.check(gl[before], wlse[before], ltol[before], "before lse")
    ref.check(out[before], want[before], tol[before], "without")


@pytest.mark.parametrize("n,L", [(1, 20), (1, 5000), (40, 100), (40, 5000)])
def test_a_nan_in_a_query_stays_in_its_row(gpu, n, L):
    q, cache, table, lens, starts = problem(gpu, lens=[L, L], counts=[n, n], garbage=False)
    q[n - 1, 1, 7] = math.nan
    q[n, 2, 100] = math.inf  # its scores are +-inf: NaN, or 0 where all are -inf, as for a row that sees nothing
    from low_bit_fake_quant import paged_attention
    out, lse = paged_attention(q, cache, table, lens, starts, max_query_len=n, return_lse=True)
    bad = torch.zeros(q.shape[:2], dtype=torch.bool, device=gpu)
    bad[n - 1, 1] = bad[n, 2] = True
    assert torch.isnan(out[n - 1, 1]).all() and torch.isnan(lse[n - 1, 1])
    want, wlse, tol, ltol = ref.attend(torch.nan_to_num(q, 0, 0, 0), cache, table, lens, starts)
    ref.check(out[~bad], want[~bad], tol[~bad], "others")
    ref.check(lse[~bad], wlse[~bad], ltol[~bad], "others lse")


@pytest.mark.parametrize("n", [1, 40])
def test_a_few_large_and_many_small_weights(gpu, n):
    """One key holds half the weight, thousands share the rest, each 2^-12 and less of it."""
    from low_bit_fake_quant import write_kv_cache
    q, cache, table, lens, starts = problem(gpu, lens=[6000], counts=[n], garbage=False, qscale=1.0)
    k = torch.zeros(6000, 2, 128)
    k[0] = q[:, ::2].mean(0).sign().cpu().float()
    q.copy_(k[0].repeat_interleave(2, 0).to(q.dtype)[None] * (12.5 / math.sqrt(128) * 0.8))
    g = torch.Generator().manual_seed(1)
    v = torch.randn(6000, 2, 128, generator=g)
    at = torch.arange(6000)
    write_kv_cache(k.to(gpu), v.to(gpu), cache, (table.cpu().long()[0, at // 16] * 16 + at % 16).to(gpu))
    run_and_check((q, cache, table, lens, starts), "one and many", hint=n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [1, 40])
def test_scales_of_k_and_v_further_apart_than_fp16_reaches(gpu, n, d, dtype):
    """K rows over 2^-30 ... 2^3 and V rows over 2^-40 ... 2^20, and either alone: the
    chunk kernel's loop for such parts, for K, for V and for both."""
    from low_bit_fake_quant import write_kv_cache
    for kspan, vspan in (((-30, 3), (0, 0)), ((0, 0), (-40, 20)), ((-30, 3), (-40, 20))):
        args = problem(gpu, lens=[150, 90], counts=[n, n], d=d, dtype=dtype, garbage=False)
        g = torch.Generator().manual_seed(5)
        for b, L in enumerate((150, 90)):
            k, v = (torch.randn(L, 2, d, generator=g) * torch.exp2(torch.randint(*(s[0], s[1] + 1), (L, 1, 1), generator=g).float())
                    for s in (kspan, vspan))
            at = torch.arange(L)
            write_kv_cache(k.to(gpu), v.to(gpu), args[1], (args[2].cpu().long()[b, at // 16] * 16 + at % 16).to(gpu))
        run_and_check(args, f"K 2^{kspan} V 2^{vspan}", hint=n)


@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("span", [(-3, 3), (-30, 30), (8, 14), (-20, -12)])
def test_values_of_very_different_sizes(gpu, n, span):
    """V rows over many powers of two: no scale may over- or underflow on the way."""
    vs = lambda T, g: torch.exp2(torch.randint(span[0], span[1] + 1, (T,), generator=g).float())  # noqa: E731
    args = problem(gpu, lens=[150, 90], counts=[n, n], vscale=vs, seed=n)
    run_and_check(args, f"values 2^{span}", hint=n)


@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_peaked_scores_and_scales(gpu, n, dtype):
    """Scores of hundreds: one key takes all, and maxima grow along the keys."""
    args = problem(gpu, lens=[400, 130], counts=[n, n], qscale=30.0, dtype=dtype)
    run_and_check(args, "peaked", hint=n)
    run_and_check(args, "flat", hint=n, sm_scale=1e-6)
    run_and_check(args, "sm_scale", hint=n, sm_scale=0.7)


@pytest.mark.parametrize("n", [1, 40])
def test_layouts_of_queries_and_output(gpu, n):
    from low_bit_fake_quant import paged_attention
    q, cache, table, lens, starts = problem(gpu, lens=[100, 50], counts=[n, n], tail=2)
    T, hq, d = q.shape
    want, wl = paged_attention(q, cache, table, lens, starts, max_query_len=n, return_lse=True)
    assert not want[-2:].any() and torch.isneginf(wl[-2:]).all()
    packed = torch.cat([q, q + 1], 1)[:, :hq]
    heads = q.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.empty(T * hq * d + 1, dtype=q.dtype, device=gpu)[1:].view(T, hq, d).copy_(q)
    last = q.transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.empty(table.shape[0], 2 * table.shape[1], dtype=torch.int32, device=gpu)
    wide[:, ::2] = table
    for x in (packed, heads, odd, last):
        assert torch.equal(paged_attention(x, cache, wide[:, ::2], lens, starts, max_query_len=n), want)
    big = torch.full((T, hq + 3, d), 7.0, dtype=q.dtype, device=gpu)
    out = big[:, 1:1 + hq]
    got, l2 = paged_attention(q, cache, table, lens, starts, max_query_len=n, out=out, return_lse=True)
    assert got.data_ptr() == out.data_ptr() and torch.equal(out[:-2], want[:-2]) and torch.equal(l2, wl)
    assert (out[-2:] == 7).all() and (big[:, 0] == 7).all() and (big[:, 1 + hq:] == 7).all()


@pytest.mark.parametrize("n,L", [(1, 3000), (60, 3000), (300, 300)])
def test_graph_replays_two_graphs_and_streams(gpu, n, L):
    """Two captured calls with their own workspaces, replayed in turn with eager
    calls between them, on new inputs: each equals the eager call bit for bit."""
    from low_bit_fake_quant import paged_attention
    sets = [problem(gpu, lens=[L, L // 2], counts=[n, n], seed=s, tail=1, garbage=False) for s in (1, 2)]
    call = lambda a: paged_attention(*a, max_query_len=n, return_lse=True)  # noqa: E731
    for a in sets:
        call(a)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for a in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(a))
        graphs.append(g)
    side = torch.cuda.Stream(device=gpu)
    for rep in range(4):
        for a in sets:
            a[0].copy_(cpu_randn(*a[0].shape, seed=20 + rep).to(gpu))
            a[3].copy_(torch.tensor([L - 3 * rep, L // 2 - rep], dtype=torch.int32).to(gpu))
        side.wait_stream(torch.cuda.current_stream(gpu))
        for g in graphs:
            g.replay()
        with torch.cuda.stream(side):
            eager = [call(a) for a in sets]
        side.synchronize()
        torch.cuda.synchronize()
        for a, o, e in zip(sets, outs, eager):
            assert torch.equal(o[0], e[0]) and torch.equal(o[1], e[1]), rep
            w = call(a)
            assert torch.equal(o[0], w[0]) and torch.equal(o[1], w[1]), rep


@pytest.mark.parametrize("n,L", [(4, 700), (90, 700)])
def test_a_replay_with_other_chunk_lengths(gpu, n, L):
    """The split of the tokens over the sequences is read on the device: a captured call follows it."""
    from low_bit_fake_quant import paged_attention
    a = problem(gpu, lens=[L, L // 2, L], counts=[n, n, n], hq=8, seed=3, garbage=False)
    call = lambda: paged_attention(*a, max_query_len=3 * n, return_lse=True)  # noqa: E731
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = call()
    for starts in ((0, n, 2 * n, 3 * n), (0, 0, 3 * n, 3 * n), (0, 1, 2, 3 * n - 1), (1, 2 * n, 2 * n, 2 * n + 1)):
        a[4].copy_(torch.tensor(starts, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        want = call()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), starts
        ref.check(got[0], *[x for i, x in enumerate(ref.attend(*a)) if i in (0, 2)], str(starts))


def test_repeated_calls_give_the_same_bits(gpu):
    from low_bit_fake_quant import paged_attention
    for n, L in ((1, 6000), (64, 2000), (500, 500)):
        a = problem(gpu, lens=[L, L], counts=[n, n], garbage=False)
        first = paged_attention(*a, max_query_len=n)
        for _ in range(3):
            assert torch.equal(paged_attention(*a, max_query_len=n), first)


def test_prompt_then_tokens_as_a_model_runs_them(gpu):
    """Norm and rotation, cache write and attention together: a prompt in two chunks
    and then token by token gives, at every position, what attention over the values
    read back from the cache gives."""
    from low_bit_fake_quant import (empty_kv_cache, paged_attention, qk_norm_rope, read_kv_cache, rotary_table,
                                    write_kv_cache)
    B, hq, hk, d, page, total = 3, 8, 2, 128, 16, 75
    cos, sin = rotary_table(total, d, device=gpu)
    wq, wk = (1 + 0.1 * cpu_randn(d, seed=s, dtype=torch.float32).to(gpu) for s in (1, 2))
    qkv = cpu_randn(B, total, hq + 2 * hk, d, seed=3).to(gpu)
    cols = -(-total // page)
    cache = empty_kv_cache(B * cols, page, hk, d, device=gpu)
    table = torch.randperm(B * cols, generator=torch.Generator().manual_seed(2)).view(B, cols).int().to(gpu)
    outs, qs, done = [], [], 0
    for n in (40, 30, 1, 1, 1, 2):
        x = qkv[:, done:done + n]
        at = torch.arange(done, done + n, device=gpu)
        q, k = qk_norm_rope(x[:, :, :hq], x[:, :, hq:hq + hk], wq, wk, cos, sin, at, pairs="halves")
        slots = table.long()[:, at // page] * page + at % page
        write_kv_cache(k.flatten(0, 1), x[:, :, hq + hk:].flatten(0, 1), cache, slots.flatten())
        done += n
        lens = torch.full((B,), done, dtype=torch.int32, device=gpu)
        starts = torch.arange(0, B * n + 1, n, dtype=torch.int32, device=gpu)
        outs.append(paged_attention(q.flatten(0, 1), cache, table, lens, starts, max_query_len=n).view(B, n, hq, d))
        qs.append(q)
    assert done == total
    got, q = torch.cat(outs, 1), torch.cat(qs, 1)
    lens = torch.full((B,), total, dtype=torch.int32, device=gpu)
    want, _, tol, _ = ref.attend(q.flatten(0, 1), cache, table, lens,
                                 torch.arange(0, B * total + 1, total, dtype=torch.int32))
    ref.check(got.flatten(0, 1), want, tol, "chunks and tokens")
    # and the whole as one chunk
    starts = torch.arange(0, B * total + 1, total, dtype=torch.int32, device=gpu)
    ref.check(paged_attention(q.flatten(0, 1).contiguous(), cache, table, lens, starts), want, tol, "one chunk")
    k, _ = read_kv_cache(cache, table, lens, total, dtype=torch.float32)
    assert torch.equal(k[1].double(), ref.rows_of(cache[0], cache[1], table[1], total))


def test_refusals(gpu):
    from low_bit_fake_quant import paged_attention
    q, cache, table, lens, starts = problem(gpu, lens=[20], counts=[2])

    def call(q=q, cache=cache, table=table, lens=lens, starts=starts, **kw):
        return paged_attention(q, cache, table, lens, starts, **kw)

    for kw, err, msg in (
            (dict(q=q.float()), TypeError, "bfloat16 or float16"), (dict(q=q[..., :64]), ValueError, "q must be"),
            (dict(q=q[:, :3]), ValueError, "multiple of the cache's"), (dict(q=q.cpu()), ValueError, "must live on"),
            (dict(table=table.long()), TypeError, "int32"), (dict(table=table[:, :0]), ValueError, "no columns"),
            (dict(lens=lens.long()), TypeError, "seq_lens must be"), (dict(starts=starts[:1]), ValueError, "query_starts"),
            (dict(sm_scale=0.0), ValueError, "sm_scale"), (dict(sm_scale=-1.0), ValueError, "sm_scale"),
            (dict(sm_scale=math.nan), ValueError, "sm_scale"), (dict(sm_scale=2.0 ** 16), ValueError, "sm_scale"), (dict(window=0), ValueError, "window"),
            (dict(max_query_len=-1), ValueError, "max_query_len"), (dict(out=q[:1].clone()), ValueError, "out must be"),
            (dict(out=q[:1].expand(2, -1, -1)), ValueError, "out must have"),
            (dict(q=q.clone().requires_grad_()), ValueError, "no backward pass"),
            (dict(out=q.clone().requires_grad_()), ValueError, "no backward pass")):
        with pytest.raises(err, match=msg):
            call(**kw)
    assert paged_attention(q[:0], cache, table, lens, starts * 0).shape == (0, 4, 128)
    o, l = paged_attention(q, cache, table[:0], lens[:0], starts[:1], return_lse=True)
    assert not o.any() and torch.isneginf(l).all()


def test_an_output_that_autograd_has_saved(gpu):
    """Writing into `out` counts as a change in place: a backward pass that needs the old values says so."""
    from low_bit_fake_quant import paged_attention
    args = problem(gpu, lens=[20], counts=[2])
    out = torch.zeros_like(args[0])
    w = torch.ones_like(out, requires_grad=True)
    y = (out * w).sum()
    paged_attention(*args, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        paged_attention(*args, out=torch.zeros_like(args[0]))


def test_out_of_memory_is_torchs_error(gpu):
    from low_bit_fake_quant import read_kv_cache
    _, cache, table, lens, _ = problem(gpu, lens=[20], counts=[1])
    with pytest.raises(torch.OutOfMemoryError):
        read_kv_cache(cache, table, lens, 1 << 34, dtype=torch.float32)
