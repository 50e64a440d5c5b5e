"""Paged attention where the values that queries see reach the largest that the
cache holds, 448 * 2^119: an average of them is a finite bf16 number, whichever kernel
forms it, in however many parts of the keys.  Bounds: kv_reference.attend."""

import pytest
import torch

import kv_reference as ref
from test_gpu_paged_attention import problem

pytestmark = pytest.mark.gpu

TOP = 448.0 * 2.0 ** 119


def fill_values(args, lens, v):
    """V of the sequences' tokens, in order, is v (tokens, hk, d); K stays."""
    from low_bit_fake_quant import PagedKVCache, write_kv_cache
    _, cache, table, _, _ = args
    t, page = table.cpu().long(), cache.k_codes.shape[2]
    slots = torch.cat([t[b, torch.arange(n) // page] * page + torch.arange(n) % page for b, n in enumerate(lens)])
    spare = PagedKVCache(cache.k_codes.clone(), cache.k_scale.clone(), cache.v_codes, cache.v_scale)
    write_kv_cache(v.to(cache.k_codes.device), v.to(cache.k_codes.device), spare, slots.to(cache.k_codes.device))


def values(kind, tokens, hk, d):
    g = torch.Generator().manual_seed(11)
    x = torch.randn(tokens, hk, d, generator=g)
    if kind == "largest":  # of one sign a column: an average has the same size
        return torch.where(torch.arange(d) % 2 == 0, TOP, -TOP).expand(tokens, hk, d).contiguous()
    if kind == "mixed":
        return x.sign() * TOP
    if kind == "wide":  # scales further apart than fp16 reaches, in every part
        return x.sign() * torch.exp2(torch.where(torch.arange(tokens) % 2 == 0, 127.0, -10.0))[:, None, None]
    return x * 2.0 ** {"2^113": 113, "2^122": 122}[kind]


def check(got, want, tol, what):
    """ref.check; a value whose bound reaches past fp16's largest on both sides of 0 may be either infinity."""
    assert not torch.isnan(got).any(), f"{what}: NaN"
    top = torch.finfo(got.dtype).max
    either = (tol - want.abs() >= top) & torch.isinf(got)
    ref.check(got[~either], want[~either], tol[~either], what)


@pytest.mark.parametrize("kind", ["largest", "mixed", "2^113", "2^122", "wide"])
@pytest.mark.parametrize("d,dtype", [(128, torch.bfloat16), (64, torch.bfloat16), (128, torch.float16), (64, torch.float16)])
@pytest.mark.parametrize("n,L", [(1, 90), (1, 5000), (40, 100), (40, 5000)])
def test_averages_of_the_largest_values(gpu, n, L, d, dtype, kind):
    """One token and a chunk, their keys in one part and in several."""
    from low_bit_fake_quant import paged_attention
    lens = [L, L - L // 3]
    args = problem(gpu, lens=lens, counts=[n, n], d=d, dtype=dtype, page=64, garbage=False, qscale=0.05)
    fill_values(args, lens, values(kind, sum(lens), 2, d))
    out, lse = paged_attention(*args, max_query_len=n, return_lse=True)
    want, wlse, tol, ltol = ref.attend(*args)
    check(out, want, tol, kind)
    ref.check(lse, wlse, ltol, kind + " lse")


@pytest.mark.parametrize("L", [100, 5000])
def test_maxima_that_grow_along_the_keys(gpu, L):
    """A row's weights may reach 2^15 times its reference before that moves."""
    from low_bit_fake_quant import paged_attention, write_kv_cache
    lens, n = [L, L], 40
    args = problem(gpu, lens=lens, counts=[n, n], page=64, garbage=False)
    fill_values(args, lens, values("largest", 2 * L, 2, 128))
    q, cache, table, _, _ = args
    q.fill_(1.0)
    k = torch.full((L, 2, 128), 0.0)
    k[:] = (torch.arange(L).clamp(max=127)[:, None, None] // 64 * 2.0 ** -4)  # the second tile's scores: 1.02 * 8 larger
    keep = cache.v_codes.clone(), cache.v_scale.clone()
    for b in range(2):
        at = torch.arange(L)
        write_kv_cache(k.to(gpu), k.to(gpu), cache, (table.cpu().long()[b, at // 64] * 64 + at % 64).to(gpu))
    cache.v_codes.view(torch.uint8).copy_(keep[0].view(torch.uint8))
    cache.v_scale.copy_(keep[1])
    for scale in (None, 1.0):
        out = paged_attention(*args, max_query_len=n, sm_scale=scale)
        want, _, tol, _ = ref.attend(*args, sm_scale=scale)
        ref.check(out, want, tol, f"scale {scale}")


@pytest.mark.parametrize("n", [1, 40])
def test_the_width_of_the_table_changes_rounding_only(gpu, n):
    """The same keys in one part, and (a wide table) in several."""
    from low_bit_fake_quant import paged_attention
    lens = [120, 100]
    q, cache, table, sl, starts = problem(gpu, lens=lens, counts=[n, n], page=16, cols=400, garbage=False, qscale=0.05)
    fill_values((q, cache, table, sl, starts), lens, values("largest", sum(lens), 2, 128))
    want, _, tol, _ = ref.attend(q, cache, table, sl, starts)
    for t in (table[:, :8], table):
        ref.check(paged_attention(q, cache, t, sl, starts, max_query_len=n), want, tol, f"{t.shape[1]} columns")
