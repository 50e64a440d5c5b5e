"""Paged attention over the cache in 4 bits.  The tests that the 8-bit cache has, on caches of
4-bit codes (the reference sees the same values as 8-bit codes), and those that are this
format's own."""

import math

import pytest
import torch

import kv4_reference as ref4
import kv_reference as ref
import test_gpu_cache_gradients as gradients
import test_gpu_paged_attention as eight
import test_gpu_paged_large_values as large
import test_gpu_paged_out as outs
import test_gpu_paged_padding as padding
from conftest import cpu_randn

pytestmark = pytest.mark.gpu


def problem(dev, *, lens, counts, hq=4, hk=2, d=128, page=16, dtype=torch.bfloat16, tail=0, seed=0, qscale=2.0,
            vscale=None, cols=None, garbage=True):
    """test_gpu_paged_attention.problem in 4 bits."""
    from low_bit_fake_quant import empty_kv_cache, write_kv_cache
    B = len(lens)
    cols = cols or max(1, -(-max(lens) // page))
    pages = B * cols + 2
    g = torch.Generator().manual_seed(seed)
    cache = (ref4.garbage(pages, page, hk, d, dev, seed) if garbage else
             empty_kv_cache(pages, page, hk, d, device=dev, bits=4))
    if garbage:
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


def attend(q, cache, table, lens, starts, *, causal=True, window=None, sm_scale=None):
    """kv_reference.attend of the same values, whose bound is added to what it leaves out.  Many E2M1 values are 0, so
    what a row's large weights multiply may be nothing at all, and its result the product of a weight that fp16 holds as
    one of its smallest numbers: the chunk kernel's largest weight is 2^7 at least, so fp16's step there, 2^-24, rounds
    the others by up to 2^-32 of it.  Added up: 2^-32 sum |V_j| over the keys that are seen (l >= 1).

    And the query's terms leave up to 2^-19 of the largest of 32 columns (2^-3 2^-15 of a scale that the largest is
    twice of at least): scores off by dq = 2^-19 sum of that |k_j| sm_scale, the result by 2 dq max |V_j|, its lse by dq."""
    if cache[0].dtype == torch.float4_e2m1fn_x2:
        cache = ref4.widen(cache)
    out, lse, tol, ltol = plain(q, cache, table, lens, starts, causal=causal, window=window, sm_scale=sm_scale)
    for b in range(table.shape[0]):
        r0, r1 = int(starts[b]), int(starts[b + 1])
        v = torch.nan_to_num(ref.rows_of(cache[2], cache[3], table[b], int(lens[b]))).abs()
        if r1 > r0 and v.shape[0]:
            seen = ref.visible(r1 - r0, v.shape[0], causal, window, q.device).any(0)
            k = torch.nan_to_num(ref.rows_of(cache[0], cache[1], table[b], int(lens[b]))).abs()
            g, d = q.shape[1] // v.shape[1], q.shape[2]
            tol[r0:r1] += 2.0 ** -32 * v[seen].sum(0).repeat_interleave(g, 0)
            if seen.any():
                top = torch.nan_to_num(q[r0:r1].double()).abs().unflatten(-1, (-1, 32)).amax(-1).repeat_interleave(32, -1)
                kt = k[seen].permute(1, 2, 0).repeat_interleave(g, 0).contiguous()
                dq = 2.0 ** -19 * torch.bmm(top.transpose(0, 1).contiguous(), kt).amax(-1).t() * (sm_scale or 1.0 / math.sqrt(d))
                tol[r0:r1] += 2 * dq[..., None] * v[seen].amax(0).repeat_interleave(g, 0)
                ltol[r0:r1] += dq
    return out, lse, tol, ltol


plain = ref.attend


@pytest.fixture(autouse=True)
def in_4_bits(monkeypatch):
    for module in (eight, gradients, large, outs, padding):
        monkeypatch.setattr(module, "problem", problem)
    monkeypatch.setattr(ref, "attend", attend)


for _module in (eight, large, outs, padding):
    for _name, _test in vars(_module).copy().items():
        # (the two that build their own caches, and those of the allocator, have nothing of the format)
        if _name.startswith("test_") and _name not in ("test_prompt_then_tokens_as_a_model_runs_them",
                                                       "test_out_of_memory_is_torchs_error"):
            globals()[_name] = _test
test_a_cache_that_asks_for_a_gradient_is_refused = gradients.test_a_cache_that_asks_for_a_gradient_is_refused
test_cache_calls_refuse_tangents = gradients.test_cache_calls_refuse_tangents


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [1, 40])
def test_scales_further_apart_than_fp16_reaches(gpu, n, d, dtype):
    """V rows over 2^-10 ... 2^40 and K rows over 2^-12 ... 2^3, and either alone (below 1e-4 the scale stays)."""
    from low_bit_fake_quant import write_kv_cache
    for kspan, vspan in (((-12, 3), (0, 0)), ((0, 0), (-10, 40)), ((-12, 3), (-10, 40))):
        args = problem(gpu, lens=[150, 90], counts=[n, n], d=d, dtype=dtype, garbage=False)
        g = torch.Generator().manual_seed(5)
        for b, L in enumerate((150, 90)):
            k, v = (torch.randn(L, 2, d, generator=g) * torch.exp2(torch.randint(*(s[0], s[1] + 1), (L, 1, 1), generator=g).float())
                    for s in (kspan, vspan))
            at = torch.arange(L)
            write_kv_cache(k.to(gpu), v.to(gpu), args[1], (args[2].cpu().long()[b, at // 16] * 16 + at % 16).to(gpu))
        eight.run_and_check(args, f"K 2^{kspan} V 2^{vspan}", hint=n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("low,high", [(100, 103), (100, 136), (100, 137), (1, 254)])
def test_scale_bytes_of_a_cache_filled_elsewhere(gpu, n, d, dtype, low, high):
    """Any V scales from 2^-126 to 2^127, and the widest span that fp16 holds next to one more."""
    q, cache, table, lens, starts = problem(gpu, lens=[150, 90], counts=[n, n], d=d, dtype=dtype, garbage=False)
    g = torch.Generator().manual_seed(low + high)
    pick = torch.randint(low, high + 1, cache[3].shape, generator=g, dtype=torch.uint8)
    pick[..., 0, 0], pick[..., 1, 0] = low, high
    cache[3].copy_(pick.to(gpu))
    eight.run_and_check((q, cache, table, lens, starts), f"scales {low} ... {high}", hint=n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("kind", ["outliers", "tiny", "huge", "one", "hidden"])
def test_queries_of_very_different_columns(gpu, n, d, dtype, kind):
    """A few columns a thousand times the others; values next to the dtype's smallest and largest; one column."""
    q, cache, table, lens, starts = problem(gpu, lens=[150, 90], counts=[n, n], d=d, dtype=dtype, garbage=False, qscale=1.0)
    g = torch.Generator().manual_seed(3)
    if kind == "outliers":
        q.mul_(torch.where(torch.rand(d, generator=g) < 0.1, 30.0, 0.03).to(gpu).to(dtype))
        sm = 0.05
    elif kind == "tiny":
        q.mul_(2.0 ** (-22 if dtype == torch.float16 else -124))
        sm = 2.0 ** 15
    elif kind == "huge":
        q.mul_(2.0 ** (13 if dtype == torch.float16 else 100))
        sm = 2.0 ** (-16 if dtype == torch.float16 else -64)
    elif kind == "hidden":  # one column of 32 is thousands of times the others, and K is 0 there
        q[..., ::32] *= 4000 if dtype == torch.bfloat16 else 1000
        cache[0].view(torch.uint8)[..., ::16] &= 0xF0
        sm = 0.1
    else:
        q[..., 1:] = 0
        sm = 1.0
    if kind == "huge" and dtype == torch.bfloat16:
        cache[1].fill_(90)  # (scores of 2^100 2^-37 2^-64)
    eight.run_and_check((q, cache, table, lens, starts), kind, hint=n, sm_scale=sm)


@pytest.mark.parametrize("n,L,cols,hk,d,dtype,causal,before", [
    (2200, 2500, None, 16, 128, torch.bfloat16, False, 0), (2200, 4480, None, 16, 128, torch.float16, True, 0),
    (2200, 2500, 300, 16, 128, torch.bfloat16, False, 5), (2100, 2200, None, 24, 64, torch.float16, False, 0),
    (2200, 30, 300, 16, 128, torch.bfloat16, False, 0)])
def test_two_unequal_parts(gpu, n, L, cols, hk, d, dtype, causal, before):
    """Row tiles of one sequence that fill more than half of the chip, but not all; also where the sequence is much shorter
    than its table, and behind rows of no sequence."""
    from low_bit_fake_quant import paged_attention
    q, cache, table, lens, starts = problem(gpu, lens=[L], counts=[n], hq=hk, hk=hk, d=d, dtype=dtype, page=64, cols=cols,
                                            tail=before, garbage=False)
    q, starts = torch.roll(q, before, 0), starts + before
    out, lse = paged_attention(q, cache, table, lens, starts, causal=causal, return_lse=True)
    for h in range(0, hk, 8):
        part = type(cache)(*(t.view(torch.uint8)[:, h:h + 8].contiguous().view(t.dtype) for t in cache))
        want, wlse, tol, ltol = attend(q[:, h:h + 8].contiguous(), part, table, lens, starts, causal=causal)
        ref.check(out[:, h:h + 8], want, tol, "out")
        ref.check(lse[:, h:h + 8], wlse, ltol, "lse")


@pytest.mark.parametrize("n", [1, 3, 17, 100, 700])
def test_equals_the_8_bit_cache_of_the_same_values(gpu, n):
    from low_bit_fake_quant import paged_attention
    q, cache, table, lens, starts = problem(gpu, lens=[1500, 900, 33], counts=[n, n, 1], hq=8, page=32, garbage=False)
    got = paged_attention(q, cache, table, lens, starts, max_query_len=n)
    want = paged_attention(q, ref4.widen(cache), table, lens, starts, max_query_len=n)
    _, _, tol, _ = plain(q, ref4.widen(cache), table, lens, starts)
    ref.check(got, want.double(), 2 * tol, "two caches")


def test_prompt_then_tokens_as_a_model_runs_them(gpu):
    """Rotation and cache write in one call, then attention: a prompt in two chunks and then token by token gives, at
    every position, what attention over the values read back from the cache gives; so does fake_quant_attention's input."""
    from low_bit_fake_quant import append_kv_cache, empty_kv_cache, paged_attention, read_kv_cache, rotary_table
    B, hq, hk, d, page, total = 3, 8, 2, 128, 16, 75
    cos, sin = rotary_table(total, d, device=gpu)
    qkv = cpu_randn(B, total, hq + 2 * hk, d, seed=3).to(gpu)
    cols = -(-total // page)
    cache = empty_kv_cache(B * cols, page, hk, d, device=gpu, bits=4)
    table = torch.randperm(B * cols, generator=torch.Generator().manual_seed(2)).view(B, cols).int().to(gpu)
    results, qs, done = [], [], 0
    for n in (40, 30, 1, 1, 1, 2):
        x = qkv[:, done:done + n].flatten(0, 1)
        at = torch.arange(done, done + n, device=gpu)
        slots = table.long()[:, at // page] * page + at % page
        q = append_kv_cache(x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:], cache, slots.flatten(), cos, sin, at.repeat(B),
                            pairs="halves")
        done += n
        lens = torch.full((B,), done, dtype=torch.int32, device=gpu)
        starts = torch.arange(0, B * n + 1, n, dtype=torch.int32, device=gpu)
        results.append(paged_attention(q, cache, table, lens, starts, max_query_len=n).view(B, n, hq, d))
        qs.append(q.view(B, n, hq, d))
    assert done == total
    got, q = torch.cat(results, 1), torch.cat(qs, 1)
    lens = torch.full((B,), total, dtype=torch.int32, device=gpu)
    starts = torch.arange(0, B * total + 1, total, dtype=torch.int32, device=gpu)
    want, _, tol, _ = attend(q.flatten(0, 1), cache, table, lens, starts)
    ref.check(got.flatten(0, 1), want, tol, "chunks and tokens")
    ref.check(paged_attention(q.flatten(0, 1).contiguous(), cache, table, lens, starts), want, tol, "one chunk")
    k, _ = read_kv_cache(cache, table, lens, total, dtype=torch.float32)
    wide = ref4.widen(cache)
    assert torch.equal(k[1].double(), ref.rows_of(wide[0], wide[1], table[1], total))
    # the values are what the whole-tensor attention takes
    kk, vv = (x.repeat_interleave(hq // hk, 2) for x in read_kv_cache(cache, table, lens, total))
    one = paged_attention(q.flatten(0, 1).contiguous(), cache, table, lens, starts, causal=False).view(B, total, hq, d)
    s = torch.matmul(q.float().transpose(1, 2), kk.float().permute(0, 2, 3, 1).contiguous()) / math.sqrt(d)
    o = torch.matmul(s.softmax(-1), vv.float().transpose(1, 2).contiguous()).transpose(1, 2)
    assert (one.float() - o).abs().max() <= 2.0 ** -8 * o.abs().max() * 1.5
