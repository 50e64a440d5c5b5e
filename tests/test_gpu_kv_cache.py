"""Writing the quantised paged cache and reading it back: codes and scales equal
the package's MXFP8 quantiser and the definition in 64 bits bit for bit, slots that
are not written stay as they are, and values come back as code * 2^e."""

import math

import pytest
import torch

import kv_reference as ref
from conftest import cpu_randn

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def filled(pages, page, h, d, dev, seed=3):
    """A cache of arbitrary bytes (NaN codes and scales among them)."""
    from low_bit_fake_quant import PagedKVCache
    g = torch.Generator().manual_seed(seed)
    by = lambda *s: torch.randint(0, 256, s, generator=g, dtype=torch.uint8).to(dev)  # noqa: E731
    f8 = torch.float8_e4m3fn
    return PagedKVCache(by(pages, h, page, d).view(f8), by(pages, h, page, d // 32), by(pages, h, page, d).view(f8),
                        by(pages, h, page, d // 32))


def bytes_of(cache):
    return [t.view(torch.uint8).clone() for t in cache]


def slots_for(T, total, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(total, generator=g)[:T]


CASES = [(1, 1, 64, 16, "bf16"), (7, 3, 128, 16, "fp16"), (64, 2, 128, 64, "fp32"), (65, 5, 64, 32, "fp16"),
         (129, 8, 128, 128, "bf16"), (200, 1, 64, 1024, "fp32"), (63, 12, 128, 16, "bf16")]


@pytest.mark.parametrize("T,h,d,page,dtype", CASES)
def test_written_rows_equal_the_quantiser_and_the_definition(gpu, T, h, d, page, dtype):
    from low_bit_fake_quant import mxfp8_qk_quant, write_kv_cache
    pages = -(-2 * T // page) + 1
    cache = filled(pages, page, h, d, gpu)
    before = bytes_of(cache)
    scale = torch.logspace(-6, 4, T).view(T, 1, 1)
    k, v = ((cpu_randn(T, h, d, seed=s, dtype=torch.float32) * scale).to(DTYPES[dtype]).to(gpu) for s in (1, 2))
    slots = slots_for(T, pages * page, 5).to(gpu)
    if T > 3:
        slots[1], slots[2] = -1, pages * page  # neither is in the cache
    write_kv_cache(k, v, cache, slots)
    live = (slots >= 0) & (slots < pages * page)
    at = slots[live]
    for i, x in ((0, k), (2, v)):
        codes, sc = mxfp8_qk_quant(x[None])
        val, e = ref.mx_encode(x)
        c = cache[i].view(torch.uint8).transpose(1, 2).reshape(-1, h, d)
        s = cache[i + 1].transpose(1, 2).reshape(-1, h, d // 32)
        assert torch.equal(c[at], codes[0].view(torch.uint8)[live])
        assert torch.equal(torch.exp2(s[at].double() - 127), sc[0][live].double())
        assert torch.equal(s[at].long() - 127, e[live])
        assert torch.equal(ref.mx_decode(c[at], torch.full_like(s[at], 127)), val[live])
        rest = torch.ones(pages * page, dtype=torch.bool, device=gpu)
        rest[at] = False
        b = before[i].transpose(1, 2).reshape(-1, h, d)
        bs = before[i + 1].transpose(1, 2).reshape(-1, h, d // 32)
        assert torch.equal(c[rest], b[rest]) and torch.equal(s[rest], bs[rest])


def test_zero_nan_and_infinite_rows(gpu):
    from low_bit_fake_quant import empty_kv_cache, mxfp8_qk_quant, read_kv_cache, write_kv_cache
    x = cpu_randn(6, 2, 128, seed=4, dtype=torch.float32)
    x[0] = 0
    x[1, :, 5] = math.nan
    x[2, :, 40] = math.inf
    x[3, :, 70] = -math.inf
    x[4] = 3.4e38
    x[5, :, 100:] = 1e-44
    x = x.to(gpu)
    cache = empty_kv_cache(1, 16, 2, 128, device=gpu)
    write_kv_cache(x, -x, cache, torch.arange(6, device=gpu))
    for i, t in ((0, x), (2, -x)):
        # infinities are held as the largest finite value, 448 * 2^119
        codes, sc = mxfp8_qk_quant(t.clamp(-448 * 2.0 ** 119, 448 * 2.0 ** 119)[None])
        assert torch.equal(cache[i].view(torch.uint8)[0, :, :6].transpose(0, 1), codes[0].view(torch.uint8))
        assert torch.equal(torch.exp2(cache[i + 1][0, :, :6].transpose(0, 1).double() - 127), sc[0].double())
    k, v = read_kv_cache(cache, torch.zeros(1, 1, dtype=torch.int32, device=gpu),
                         torch.tensor([6], dtype=torch.int32, device=gpu), 6, dtype=torch.float32)
    assert torch.isfinite(k).all() and torch.isfinite(v).all()
    assert (k[0, 2, :, 40] == 448 * 2.0 ** 119).all() and (k[0, 3, :, 70] == -448 * 2.0 ** 119).all()


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
    want, got = (empty_kv_cache(3, 16, h, d, device=gpu) for _ in range(2))
    slots = slots_for(T, 48, 7).to(gpu)
    write_kv_cache(k.contiguous().clone(), v.contiguous().clone(), want, slots)
    write_kv_cache(k, v, got, slots)
    for a, b in zip(bytes_of(got), bytes_of(want)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("h,d,page,lens,max_len,dtype", [
    (1, 64, 16, [1], 1, "fp32"), (3, 128, 16, [0, 17, 48, 5], 40, "bf16"), (2, 64, 64, [64, 63, 65, 130], 131, "fp16"),
    (5, 128, 32, [33, -4, 1000], 70, "fp32"), (4, 128, 128, [200], 300, "bf16")])
def test_read_gives_code_times_scale_and_zeros_behind(gpu, h, d, page, lens, max_len, dtype):
    from low_bit_fake_quant import empty_kv_cache, read_kv_cache, write_kv_cache
    B, cols = len(lens), -(-max(*lens, 1) // page) if max(lens) < 900 else 2
    pages = B * cols + 2
    cache = filled(pages, page, h, d, gpu)
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(1))[:B * cols].view(B, cols).int().to(gpu)
    T = pages * page
    x = cpu_randn(T, 2 * h, d, seed=8, dtype=torch.float32).to(gpu) * 5
    write_kv_cache(x[:, :h], x[:, h:], cache, torch.arange(T, device=gpu))
    if cols > 1:
        table[-1, 1] = -1
        table[0, -1] = pages if lens[0] <= (cols - 1) * page else table[0, -1]
    k, v = read_kv_cache(cache, table, torch.tensor(lens, dtype=torch.int32, device=gpu), max_len, dtype=DTYPES[dtype])
    for b, n in enumerate(lens):
        n = max(0, min(n, max_len, cols * page))
        for got, i in ((k, 0), (v, 2)):
            want = torch.zeros(max_len, h, d, dtype=torch.float64, device=gpu)
            want[:n] = torch.nan_to_num(ref.rows_of(cache[i], cache[i + 1], table[b], n))
            # fp32 holds code * 2^e, so one rounding to the output dtype is the whole of it
            assert torch.equal(got[b], want.float().to(DTYPES[dtype])), (b, i)
    assert empty_kv_cache(1, 16, h, d, device=gpu)[1].eq(127).all()


def test_offsets_past_32_bits(gpu):
    """Code tensors of over 2^32 bytes: the last pages are written, read and attended."""
    from low_bit_fake_quant import empty_kv_cache, paged_attention, read_kv_cache, write_kv_cache
    h, d, page = 8, 128, 64
    pages = (1 << 32) // (h * d * page) + 3
    cache = empty_kv_cache(pages, page, h, d, device=gpu)
    assert cache.k_codes.numel() > 1 << 32
    T = 100
    k, v = (cpu_randn(T, h, d, seed=s).to(gpu) for s in (1, 2))
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device=gpu)
    at = torch.arange(T, device=gpu)
    write_kv_cache(k, v, cache, table[0].long()[at // page] * page + at % page)
    lens = torch.tensor([T], dtype=torch.int32, device=gpu)
    gk, gv = read_kv_cache(cache, table, lens, T, dtype=torch.float32)
    for got, x in ((gk, k), (gv, v)):
        val, e = ref.mx_encode(x)
        assert torch.equal(got[0].double(), val * torch.exp2(e.double()).repeat_interleave(32, -1))
    small = type(cache)(*(t[-2:].clone() for t in cache))
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
    cache, other = (empty_kv_cache(6, page, h, d, device=gpu) for _ in range(2))
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
    c = empty_kv_cache(2, 16, 2, 64, device=gpu)
    x = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device=gpu)
    write_kv_cache(x, x, c, torch.zeros(0, dtype=torch.int64, device=gpu))
    k, _ = read_kv_cache(c, torch.zeros(1, 2, dtype=torch.int32, device=gpu),
                         torch.zeros(1, dtype=torch.int32, device=gpu), 0)
    assert k.shape == (1, 0, 2, 64)
    k, _ = read_kv_cache(c, torch.zeros(1, 0, dtype=torch.int32, device=gpu),
                         torch.tensor([9], dtype=torch.int32, device=gpu), 3)
    assert k.shape == (1, 3, 2, 64) and not k.any()
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=gpu)
    s = torch.arange(3, device=gpu)
    for bad, err, msg in (
            (lambda: write_kv_cache(x[:, :1], x[:, :1], c, s), ValueError, "k and v must be"),
            (lambda: write_kv_cache(x, x.float(), c, s), TypeError, "one dtype"),
            (lambda: write_kv_cache(x.double(), x.double(), c, s), TypeError, "unsupported dtype"),
            (lambda: write_kv_cache(x, x, c, s.int()), TypeError, "slots must be"),
            (lambda: write_kv_cache(x, x, c, s[:2]), ValueError, "slots must have shape"),
            (lambda: write_kv_cache(x, x, c, s.cpu()), ValueError, "slots must live on"),
            (lambda: write_kv_cache(x.cpu(), x, c, s), ValueError, "must live on the cache's"),
            (lambda: write_kv_cache(x.requires_grad_(), x, c, s), ValueError, "no backward pass"),
            (lambda: write_kv_cache(x, x, c._replace(k_scale=c.k_scale[:1]), s), ValueError, "cache tensors must be codes"),
            (lambda: write_kv_cache(x, x, c._replace(v_codes=c.v_codes.view(torch.uint8)), s), TypeError, "float8"),
            (lambda: write_kv_cache(x, x, c._replace(v_codes=c.v_codes.transpose(1, 2).contiguous().transpose(1, 2)), s),
             ValueError, "contiguous"),
            (lambda: read_kv_cache(c, torch.zeros(1, 2, dtype=torch.int64, device=gpu), s[:1].int(), 1), TypeError, "int32"),
            (lambda: read_kv_cache(c, torch.zeros(1, 2, dtype=torch.int32, device=gpu), s.int(), 1), ValueError, "seq_lens"),
            (lambda: read_kv_cache(c, torch.zeros(1, 2, dtype=torch.int32, device=gpu), s[:1].int(), 1,
                                   dtype=torch.float64), TypeError, "unsupported dtype")):
        with pytest.raises(err, match=msg):
            bad()
    with torch.no_grad():
        write_kv_cache(x, x, c, s)
