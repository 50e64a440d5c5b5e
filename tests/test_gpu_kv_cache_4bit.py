"""The paged cache in 4 bits: written rows equal the definition in 64 bits bit for bit, at
every middle between two codes too; slots that are not written stay as they are, and values
come back as code * 2^e."""

import math

import pytest
import torch

import kv4_reference as ref
from conftest import cpu_randn
from test_gpu_kv_cache import DTYPES, slots_for

pytestmark = pytest.mark.gpu

F4 = torch.float4_e2m1fn_x2


def bytes_of(cache):
    return [t.view(torch.uint8).clone() for t in cache]


def by_slot(t):
    """(pages, h, page, w) -> (slots, h, w) bytes"""
    t = t.view(torch.uint8).transpose(1, 2)
    return t.reshape(-1, *t.shape[2:])


@pytest.mark.parametrize("T,h,d,page,dtype", [
    (1, 1, 64, 16, "bf16"), (7, 3, 128, 16, "fp16"), (64, 2, 128, 64, "fp32"), (65, 5, 64, 32, "fp16"),
    (129, 8, 128, 128, "bf16"), (200, 1, 64, 1024, "fp32"), (63, 12, 128, 16, "bf16")])
def test_written_rows_equal_the_definition(gpu, T, h, d, page, dtype):
    from low_bit_fake_quant import write_kv_cache
    pages = -(-2 * T // page) + 1
    cache = ref.garbage(pages, page, h, d, gpu)
    before = bytes_of(cache)
    scale = torch.logspace(-6, 4, T).view(T, 1, 1)
    k, v = ((cpu_randn(T, h, d, seed=s, dtype=torch.float32) * scale).to(DTYPES[dtype]).to(gpu) for s in (1, 2))
    slots = slots_for(T, pages * page, 5).to(gpu)
    if T > 3:
        slots[1], slots[2] = -1, pages * page  # neither is in the cache
    write_kv_cache(k, v, cache, slots)
    live = (slots >= 0) & (slots < pages * page)
    at = slots[live]
    rest = torch.ones(pages * page, dtype=torch.bool, device=gpu)
    rest[at] = False
    for i, x in ((0, k), (2, v)):
        val, e = ref.encode(x)
        assert torch.equal(ref.values(by_slot(cache[i])[at]), val[live])
        assert torch.equal(by_slot(cache[i + 1])[at].long() - 127, e[live])
        for j in (i, i + 1):
            assert torch.equal(by_slot(cache[j])[rest], by_slot(before[j])[rest])


def test_every_middle_and_its_neighbours(gpu):
    """All values, the middles between them (ties to the even code) and the floats next to both, at three scales."""
    from low_bit_fake_quant import empty_kv_cache, write_kv_cache
    v = torch.tensor(ref.VALUES)
    x = torch.cat([v, (v[:-1] + v[1:]) / 2])
    x = torch.cat([x, torch.nextafter(x, torch.tensor(0.0)), torch.nextafter(x, torch.tensor(9.0))])
    x = torch.cat([x, -x]).clamp(-6, 6)
    rows = torch.zeros(-(-x.numel() // 31), 32)
    rows[:, 0] = 6.0  # fixes the scale
    flat = torch.zeros(rows.shape[0] * 31)
    flat[:x.numel()] = x
    rows[:, 1:] = flat.view(-1, 31)
    rows = torch.cat([rows, rows * 2.0 ** -9, rows * 2.0 ** 60])
    rows = torch.cat([rows, torch.zeros(-rows.shape[0] % 2, 32)]).view(-1, 1, 64).to(gpu)
    cache = empty_kv_cache(-(-rows.shape[0] // 16), 16, 1, 64, device=gpu, bits=4)
    write_kv_cache(rows, -rows, cache, torch.arange(rows.shape[0], device=gpu))
    for i, r in ((0, rows), (2, -rows)):
        val, e = ref.encode(r)
        assert torch.equal(ref.values(by_slot(cache[i])[:rows.shape[0]]), val)
        assert torch.equal(by_slot(cache[i + 1])[:rows.shape[0]].long() - 127, e)


def test_amax_next_to_six_times_a_power_of_two(gpu):
    """The scale changes from one float to the next there, over every exponent that fp32 has (floor 1e-4)."""
    from low_bit_fake_quant import empty_kv_cache, write_kv_cache
    x = torch.ldexp(torch.tensor(6.0), torch.arange(-20, 126))
    x = torch.cat([x, torch.nextafter(x, torch.tensor(0.0)), torch.nextafter(x, torch.tensor(math.inf))])
    T = x.numel()
    rows = (x[:, None] * torch.linspace(-1, 1, 64)[None]).view(T, 1, 64).to(gpu)
    cache = empty_kv_cache(-(-T // 16), 16, 1, 64, device=gpu, bits=4)
    write_kv_cache(rows, rows, cache, torch.arange(T, device=gpu))
    val, e = ref.encode(rows)
    assert torch.equal(by_slot(cache[1])[:T].long() - 127, e)
    assert torch.equal(ref.values(by_slot(cache[0])[:T]), val)


def test_zero_nan_and_infinite_rows(gpu):
    from low_bit_fake_quant import empty_kv_cache, read_kv_cache, write_kv_cache
    x = cpu_randn(6, 2, 128, seed=4, dtype=torch.float32)
    x[0] = 0
    x[1, :, 5] = math.nan
    x[2, :, 40] = math.inf
    x[3, :, 70] = -math.inf
    x[4] = 3.4e38
    x[5, :, 100:] = 1e-44
    cache = empty_kv_cache(1, 16, 2, 128, device=gpu, bits=4)
    write_kv_cache(x.to(gpu), -x.to(gpu), cache, torch.arange(6, device=gpu))
    k, v = read_kv_cache(cache, torch.zeros(1, 1, dtype=torch.int32, device=gpu),
                         torch.tensor([6], dtype=torch.int32, device=gpu), 6, dtype=torch.float32)
    top = 6 * 2.0 ** 125
    for got, t in ((k, x), (v, -x)):
        got = got[0].cpu()
        assert torch.isfinite(got).all()
        clean = torch.nan_to_num(t, nan=0.0, posinf=top, neginf=-top)
        val, e = ref.encode(clean)
        want = (val * torch.exp2(e.double()).repeat_interleave(32, -1)).float()
        nan = torch.isnan(t)
        assert torch.equal(got[~nan], want[~nan])
        assert torch.equal(got[nan].double(), -6 * torch.exp2(e.double()).repeat_interleave(32, -1)[nan])


@pytest.mark.parametrize("layout", ["packed", "head_major", "unaligned", "expanded", "last_strided"])
def test_layouts_of_the_rows(gpu, layout):
    from low_bit_fake_quant import empty_kv_cache, write_kv_cache
    T, h, d = 37, 4, 128
    base = cpu_randn(T, 3 * h, d, seed=6).to(gpu)
    if layout == "packed":
        k, v = base[:, h:2 * h], base[:, 2 * h:]
    elif layout == "head_major":
        k, v = (base[:, i * h:(i + 1) * h].transpose(0, 1).contiguous().transpose(0, 1) for i in (0, 1))
    elif layout == "unaligned":
        flat = torch.empty(T * h * d + 1, dtype=base.dtype, device=gpu)
        k = flat[1:].view(T, h, d).copy_(base[:, :h])
        v = base[:, h:2 * h]
    elif layout == "expanded":
        k, v = base[:1, :h].expand(T, h, d), base[:, :1].expand(T, h, d)
    else:
        k = base[:, :h].transpose(1, 2).contiguous().transpose(1, 2)
        v = base[:, :2 * h, ::2].repeat_interleave(2, -1)[:, :h]
    want, got = (empty_kv_cache(3, 16, h, d, device=gpu, bits=4) for _ in range(2))
    slots = slots_for(T, 48, 7).to(gpu)
    write_kv_cache(k.contiguous().clone(), v.contiguous().clone(), want, slots)
    write_kv_cache(k, v, got, slots)
    for a, b in zip(bytes_of(got), bytes_of(want)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("h,d,page,lens,max_len,dtype", [
    (1, 64, 16, [1], 1, "fp32"), (3, 128, 16, [0, 17, 48, 5], 40, "bf16"), (2, 64, 64, [64, 63, 65, 130], 131, "fp16"),
    (5, 128, 32, [33, -4, 1000], 70, "fp32"), (4, 128, 128, [200], 300, "bf16")])
def test_read_gives_code_times_scale_and_zeros_behind(gpu, h, d, page, lens, max_len, dtype):
    from low_bit_fake_quant import read_kv_cache
    B, cols = len(lens), -(-max(*lens, 1) // page) if max(lens) < 900 else 2
    pages = B * cols + 2
    cache = ref.garbage(pages, page, h, d, gpu)
    for t in (cache[1], cache[3]):
        t.clamp_(1, 254)  # (a scale of 255 is not a number, one of 0 is below fp32's normal ones)
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(1))[:B * cols].view(B, cols).int().to(gpu)
    if cols > 1:
        table[-1, 1] = -1
        table[0, -1] = pages if lens[0] <= (cols - 1) * page else table[0, -1]
    k, v = read_kv_cache(cache, table, torch.tensor(lens, dtype=torch.int32, device=gpu), max_len, dtype=DTYPES[dtype])
    for b, n in enumerate(lens):
        n = max(0, min(n, max_len, cols * page))
        for got, i in ((k, 0), (v, 2)):
            want = torch.zeros(max_len, h, d, dtype=torch.float64, device=gpu)
            for j in range(n):
                pid = int(table[b, j // page])
                if 0 <= pid < pages:
                    two = torch.exp2(cache[i + 1][pid, :, j % page].double() - 127).repeat_interleave(32, -1)
                    want[j] = ref.values(cache[i].view(torch.uint8)[pid, :, j % page].contiguous()) * two
            # fp32 holds code * 2^e up to its largest (6 * 2^126 and more is infinite), so one rounding is the whole of it
            assert torch.equal(got[b], want.float().to(DTYPES[dtype])), (b, i)


def test_offsets_past_32_bits(gpu):
    """Code tensors of over 2^32 bytes: the last pages are written, read and attended."""
    from low_bit_fake_quant import append_kv_cache, empty_kv_cache, paged_attention, read_kv_cache, rotary_table
    h, d, page = 8, 128, 64
    pages = (1 << 32) // (h * d // 2 * page) + 3
    cache = empty_kv_cache(pages, page, h, d, device=gpu, bits=4)
    assert cache.k_codes.numel() > 1 << 32
    T = 100
    k, v = (cpu_randn(T, h, d, seed=s).to(gpu) for s in (1, 2))
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device=gpu)
    at = torch.arange(T, device=gpu)
    cos, sin = rotary_table(1, d, device=gpu)
    append_kv_cache(None, k, v, cache, table[0].long()[at // page] * page + at % page, cos, sin, -1 - at)
    lens = torch.tensor([T], dtype=torch.int32, device=gpu)
    gk, gv = read_kv_cache(cache, table, lens, T, dtype=torch.float32)
    for got, x in ((gk, k), (gv, v)):
        val, e = ref.encode(x)
        assert torch.equal(got[0].double(), val * torch.exp2(e.double()).repeat_interleave(32, -1))
    small = type(cache)(*(t.view(torch.uint8)[-2:].clone().view(t.dtype) for t in cache))
    for n in (1, 40):
        q = cpu_randn(n, 2 * h, d, seed=9).to(gpu)
        starts = torch.tensor([0, n], dtype=torch.int32, device=gpu)
        got = paged_attention(q, cache, table, lens, starts)
        want = paged_attention(q, small, table - (pages - 2), lens, starts)
        assert torch.equal(got, want)


def test_graph_replays_and_other_streams(gpu):
    from low_bit_fake_quant import empty_kv_cache, read_kv_cache, write_kv_cache
    T, h, d, page = 70, 3, 64, 16
    k, v = (cpu_randn(T, h, d, seed=s).to(gpu) for s in (1, 2))
    slots = slots_for(T, 96, 3).to(gpu)
    table = torch.arange(6, dtype=torch.int32, device=gpu)[None]
    lens = torch.tensor([96], dtype=torch.int32, device=gpu)
    cache, other = (empty_kv_cache(6, page, h, d, device=gpu, bits=4) for _ in range(2))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        write_kv_cache(k, v, cache, slots)
        rk, rv = read_kv_cache(cache, table, lens, 96)
    side = torch.cuda.Stream(device=gpu)
    for rep in range(4):
        k.copy_(cpu_randn(T, h, d, seed=10 + rep).to(gpu))
        slots.copy_(slots_for(T, 96, 3 + rep).to(gpu))
        for c in (cache, other):
            for t in c:
                t.view(torch.uint8).fill_(100)
        g.replay()
        side.wait_stream(torch.cuda.current_stream(gpu))
        with torch.cuda.stream(side):
            write_kv_cache(k, v, other, slots)
            wk, wv = read_kv_cache(other, table, lens, 96)
        side.synchronize()
        torch.cuda.synchronize()
        assert torch.equal(rk, wk) and torch.equal(rv, wv)
        for a, b in zip(bytes_of(cache), bytes_of(other)):
            assert torch.equal(a, b)


def test_empty_calls_and_refusals(gpu):
    from low_bit_fake_quant import empty_kv_cache, read_kv_cache, write_kv_cache
    c = empty_kv_cache(2, 16, 2, 64, device=gpu, bits=4)
    assert c.k_codes.shape == (2, 2, 16, 32) and c.k_codes.dtype == F4 and c.k_scale.eq(127).all()
    x = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device=gpu)
    write_kv_cache(x, x, c, torch.zeros(0, dtype=torch.int64, device=gpu))
    k, _ = read_kv_cache(c, torch.zeros(1, 0, dtype=torch.int32, device=gpu),
                         torch.tensor([9], dtype=torch.int32, device=gpu), 3)
    assert k.shape == (1, 3, 2, 64) and not k.any()
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=gpu)
    s = torch.arange(3, device=gpu)
    eight = empty_kv_cache(2, 16, 2, 64, device=gpu)
    half = empty_kv_cache(2, 16, 2, 32 * 2, device=gpu)._replace(k_codes=eight.k_codes[..., :32].contiguous())
    for bad, err, msg in (
            (lambda: write_kv_cache(x[..., :32], x[..., :32], c, s), ValueError, r"k and v must be \(T, 2, 64\)"),
            (lambda: write_kv_cache(x, x, c._replace(v_codes=c.v_codes.view(torch.uint8)), s), TypeError, "float4"),
            (lambda: write_kv_cache(x, x, c._replace(k_codes=c.k_codes.view(torch.uint8)), s), ValueError, "D must be"),
            (lambda: write_kv_cache(x, x, c._replace(v_codes=eight.v_codes), s), ValueError, "cache tensors must be codes"),
            (lambda: write_kv_cache(x, x, half, s), ValueError, "D must be"),
            (lambda: write_kv_cache(x, x, c._replace(k_scale=c.k_scale[..., :1].contiguous()), s), ValueError,
             "cache tensors must be codes"),
            (lambda: write_kv_cache(x.requires_grad_(), x, c, s), ValueError, "no backward pass")):
        with pytest.raises(err, match=msg):
            bad()
