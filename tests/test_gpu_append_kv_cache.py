"""append_kv_cache: the rotation is fp32, each product and the sum rounded, so Q is that
rounded to its dtype and the cache holds exactly what write_kv_cache makes of the rotated
K; against the definition in 64 bits Q is within its roundings."""

import math

import pytest
import torch

import kv_reference as ref8
from conftest import cpu_randn
from test_gpu_kv_cache import DTYPES, slots_for
from test_gpu_kv_cache_4bit import bytes_of

pytestmark = pytest.mark.gpu


def turned(x, cos, sin, positions, pairs):
    """fp32 rotation in the operator's order of roundings; negative positions stay."""
    on = (positions >= 0)[:, None, None]
    at = positions.clamp(min=0).long()
    y = ref8.rotate(x.float(), cos[at][:, None], sin[at][:, None], pairs)
    return torch.where(on, y, x.float())


def inputs(dev, T, hq, hk, d, dtype, rot, *, limit=5000, packed=True, seed=0):
    from low_bit_fake_quant import rotary_table
    x = cpu_randn(T, hq + 2 * hk, d, seed=seed, dtype=torch.float32) * torch.logspace(-2, 2, T).view(T, 1, 1)
    x = x.to(dtype).to(dev)
    q, k, v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    if not packed:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    cos, sin = rotary_table(limit, rot, device=dev)
    g = torch.Generator().manual_seed(seed)
    positions = torch.randint(0, limit, (T,), generator=g).to(dev)
    return q, k, v, cos, sin, positions


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
@pytest.mark.parametrize("T,hq,hk,d,rot,page,dtype", [
    (1, 1, 1, 64, 64, 16, "bf16"), (5, 4, 2, 128, 128, 16, "fp16"), (33, 3, 3, 128, 96, 64, "fp32"),
    (65, 14, 2, 64, 16, 32, "bf16"), (17, 32, 8, 128, 128, 16, "bf16"), (31, 5, 5, 64, 48, 128, "fp32"),
    (130, 7, 1, 128, 64, 256, "fp16"), (700, 12, 12, 128, 128, 64, "bf16"), (5000, 6, 2, 64, 64, 16, "fp16")])
def test_queries_and_cache(gpu, T, hq, hk, d, rot, page, dtype, pairs, bits):
    from low_bit_fake_quant import append_kv_cache, empty_kv_cache, write_kv_cache
    t = DTYPES[dtype]
    q, k, v, cos, sin, pos = inputs(gpu, T, hq, hk, d, t, rot, packed=T % 2 == 1)
    pages = -(-2 * T // page) + 1
    slots = slots_for(T, pages * page, 5).to(gpu)
    if T > 4:
        pos[1], pos[2] = -1, -7
        slots[2], slots[3] = -1, pages * page + 5
    got, want = (empty_kv_cache(pages, page, hk, d, device=gpu, bits=bits) for _ in range(2))
    out = append_kv_cache(q, k, v, got, slots, cos, sin, pos.int() if T % 3 == 0 else pos, pairs=pairs)
    assert out.shape == q.shape and out.dtype == t and out.is_contiguous()
    assert torch.equal(out, turned(q, cos, sin, pos, pairs).to(t))
    write_kv_cache(turned(k, cos, sin, pos, pairs), v.float(), want, slots)
    for a, b in zip(bytes_of(got), bytes_of(want)):
        assert torch.equal(a, b)
    # 64 bits: two products and a sum round to fp32, then to the dtype
    z = turned64(q, cos, sin, pos, pairs)
    size = turned64(q.abs(), cos.abs(), -sin.abs(), pos, pairs).abs() + turned64(q.abs(), cos.abs(), sin.abs(), pos, pairs).abs()
    tol = z.abs() * ref8.U[t] + 3 * 2.0 ** -24 * size * 1.01 + {"fp16": 2.0 ** -24, "bf16": 2.0 ** -133, "fp32": 2.0 ** -149}[dtype]
    assert ((out.double() - z).abs() <= tol).all()


def turned64(x, cos, sin, positions, pairs):
    on = (positions >= 0)[:, None, None]
    at = positions.clamp(min=0).long()
    return torch.where(on, ref8.rotate(x.double(), cos[at][:, None].double(), sin[at][:, None].double(), pairs), x.double())


@pytest.mark.parametrize("bits", [4, 8])
def test_positions_past_the_table(gpu, bits):
    """NaN in Q's rotated columns, nothing of the token in the cache, the others as without it."""
    from low_bit_fake_quant import append_kv_cache, empty_kv_cache
    q, k, v, cos, sin, pos = inputs(gpu, 20, 4, 2, 128, torch.bfloat16, 64, limit=50)
    slots = torch.arange(20, device=gpu)
    clean, cache = (empty_kv_cache(2, 16, 2, 128, device=gpu, bits=bits) for _ in range(2))
    want = append_kv_cache(q, k, v, clean, slots, cos, sin, pos)
    pos[7], pos[11] = 50, 1 << 40
    got = append_kv_cache(q, k, v, cache, slots, cos, sin, pos)
    bad = torch.zeros(20, dtype=torch.bool, device=gpu)
    bad[7] = bad[11] = True
    assert torch.isnan(got[bad][..., :64]).all() and torch.equal(got[bad][..., 64:], q[bad][..., 64:])
    assert torch.equal(got[~bad], want[~bad])
    empty = bytes_of(empty_kv_cache(2, 16, 2, 128, device=gpu, bits=bits))
    for a, b, z in zip(bytes_of(cache), bytes_of(clean), empty):
        for s in range(32):
            w = z if s in (7, 11) else b
            assert torch.equal(a[s // 16, :, s % 16], w[s // 16, :, s % 16])
    # an empty table: every position is past it
    before = bytes_of(cache)
    none = append_kv_cache(q, k, v, cache, slots, cos[:0], sin[:0], pos)
    assert torch.isnan(none[..., :64]).all()
    for a, b in zip(bytes_of(cache), before):
        assert torch.equal(a, b)


def test_columns_that_are_not_rotated_do_not_reach_each_other(gpu):
    from low_bit_fake_quant import append_kv_cache, empty_kv_cache, rotary_table
    for pairs in ("adjacent", "halves"):
        q = torch.ones(4, 1, 128, dtype=torch.bfloat16, device=gpu)
        q[0, 0, 3], q[1, 0, 70], q[2, 0, 127] = math.inf, math.nan, -math.inf
        cos, sin = rotary_table(4, 64, device=gpu)
        pos = torch.tensor([-1, 0, 1, 2], device=gpu)
        c = empty_kv_cache(1, 16, 1, 128, device=gpu)
        got = append_kv_cache(q, q, q, c, torch.arange(4, device=gpu), cos, sin, pos, pairs=pairs)
        want = turned(q, cos, sin, pos, pairs).to(q.dtype)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
        assert torch.equal(torch.isnan(got).sum((1, 2)).cpu(), torch.tensor([0, 1, 0, 0]))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
def test_infinities_and_nan_reach_the_cache_as_by_a_write(gpu, pairs, bits):
    from low_bit_fake_quant import append_kv_cache, empty_kv_cache, write_kv_cache
    q, k, v, cos, sin, pos = inputs(gpu, 12, 2, 2, 128, torch.float32, 96, packed=False)
    for i, x in enumerate((math.inf, -math.inf, math.nan, 3.4e38, -3.4e38, 1e-44)):
        k[i, 0, 5 * i], k[i, 1, 100], v[i, :, 7 * i] = x, x, x
    slots = torch.arange(12, device=gpu)
    got, want = (empty_kv_cache(1, 16, 2, 128, device=gpu, bits=bits) for _ in range(2))
    append_kv_cache(q, k, v, got, slots, cos, sin, pos, pairs=pairs)
    write_kv_cache(turned(k, cos, sin, pos, pairs), v, want, slots)
    for a, b in zip(bytes_of(got), bytes_of(want)):
        assert torch.equal(a, b)


def test_layouts_no_queries_and_strided_tables(gpu):
    from low_bit_fake_quant import append_kv_cache, empty_kv_cache
    T, hq, hk, d = 37, 4, 2, 128
    q, k, v, cos, sin, pos = inputs(gpu, T, hq, hk, d, torch.bfloat16, 64, limit=90, packed=False)
    slots = slots_for(T, 48, 7).to(gpu)
    first = empty_kv_cache(3, 16, hk, d, device=gpu, bits=4)
    want = append_kv_cache(q, k, v, first, slots, cos, sin, pos)
    heads = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    last = lambda x: x.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    odd = lambda x: torch.empty(x.numel() + 1, dtype=x.dtype, device=gpu)[1:].view(x.shape).copy_(x)  # noqa: E731
    wide = torch.empty(90, 65, device=gpu)
    wide[:, 1:33], wide[:, 33:] = cos, sin
    two = torch.stack((pos, pos), 1)[:, 0]
    for f in (heads, last, odd):
        c = empty_kv_cache(3, 16, hk, d, device=gpu, bits=4)
        assert torch.equal(append_kv_cache(f(q), f(k), f(v), c, torch.stack((slots, slots), 1)[:, 1], wide[:, 1:33],
                                           wide[:, 33:], two), want)
        for a, b in zip(bytes_of(c), bytes_of(first)):
            assert torch.equal(a, b)
    c = empty_kv_cache(3, 16, hk, d, device=gpu, bits=4)
    assert append_kv_cache(None, k, v, c, slots, cos, sin, pos) is None
    for a, b in zip(bytes_of(c), bytes_of(first)):
        assert torch.equal(a, b)
    one = empty_kv_cache(3, 16, hk, d, device=gpu, bits=4)
    append_kv_cache(None, k[:1].expand(T, -1, -1), v[:1].expand(T, -1, -1), one, slots, cos, sin, pos[:1].expand(T))
    rows = one.k_codes.view(torch.uint8).transpose(1, 2).reshape(48, -1)[slots]
    assert (rows == rows[:1]).all()


def test_graph_replays_two_graphs_and_streams(gpu):
    from low_bit_fake_quant import append_kv_cache, empty_kv_cache
    sets = []
    for s in (1, 2):
        a = inputs(gpu, 24, 8, 2, 128, torch.bfloat16, 128, seed=s)
        sets.append((a, empty_kv_cache(4, 16, 2, 128, device=gpu, bits=4 * s), slots_for(24, 64, s).to(gpu)))
    call = lambda a, c, s: append_kv_cache(*a[:3], c, s, *a[3:], pairs="halves")  # noqa: E731
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(*x))
        graphs.append(g)
    side = torch.cuda.Stream(device=gpu)
    for rep in range(4):
        for a, c, s in sets:
            a[0].copy_(cpu_randn(*a[0].shape, seed=30 + rep).to(gpu))
            a[5].copy_(torch.randint(0, 5000, (24,), generator=torch.Generator().manual_seed(rep)).to(gpu))
            s.copy_(slots_for(24, 64, 10 + rep).to(gpu))
            for t in c:
                t.view(torch.uint8).fill_(99)
        for g in graphs:
            g.replay()
        side.wait_stream(torch.cuda.current_stream(gpu))
        with torch.cuda.stream(side):
            others = [type(c)(*(torch.full_like(t.view(torch.uint8), 99).view(t.dtype) for t in c)) for _, c, _ in sets]
            eager = [call(a, o, s) for (a, _, s), o in zip(sets, others)]
        side.synchronize()
        torch.cuda.synchronize()
        for (_, c, _), o, got, want in zip(sets, others, outs, eager):
            assert torch.equal(got, want)
            for x, y in zip(bytes_of(c), bytes_of(o)):
                assert torch.equal(x, y)


def test_writing_counts_as_a_change_in_place(gpu):
    from low_bit_fake_quant import append_kv_cache, empty_kv_cache
    q, k, v, cos, sin, pos = inputs(gpu, 3, 2, 1, 64, torch.bfloat16, 64)
    c = empty_kv_cache(1, 16, 1, 64, device=gpu, bits=4)
    before = [t._version for t in c]
    append_kv_cache(q, k, v, c, torch.arange(3, device=gpu), cos, sin, pos)
    assert all(t._version > b for t, b in zip(c, before))


def test_empty_calls_and_refusals(gpu):
    import torch.autograd.forward_ad as forward_ad

    from low_bit_fake_quant import append_kv_cache, empty_kv_cache
    q, k, v, cos, sin, pos = inputs(gpu, 6, 4, 2, 64, torch.bfloat16, 64, limit=9)
    c = empty_kv_cache(2, 16, 2, 64, device=gpu, bits=4)
    s = torch.arange(6, device=gpu)
    keep = bytes_of(c)

    def call(q=q, k=k, v=v, cache=c, slots=s, cos=cos, sin=sin, positions=pos, **kw):
        return append_kv_cache(q, k, v, cache, slots, cos, sin, positions, **kw)

    e = call(q=q[:0], k=k[:0], v=v[:0], slots=s[:0], positions=pos[:0])
    assert e.shape == (0, 4, 64)
    for kw, err, msg in (
            (dict(k=k[:, :1], v=v[:, :1]), ValueError, "k and v must be"), (dict(v=v.float()), TypeError, "one dtype"),
            (dict(q=q.float()), TypeError, "one dtype"), (dict(q=q[:5]), ValueError, "q must be"),
            (dict(q=q[:, :0]), ValueError, "q must be"), (dict(q=q[..., :32]), ValueError, "q must be"),
            (dict(q=q.cpu()), ValueError, "q must live on"), (dict(k=k.cpu()), ValueError, "must live on the cache's"),
            (dict(q=q.double(), k=k.double(), v=v.double()), TypeError, "unsupported dtype"),
            (dict(slots=s.int()), TypeError, "slots must be"), (dict(slots=s[:5]), ValueError, "slots must have shape"),
            (dict(positions=pos.float()), TypeError, "positions must be int32 or int64"),
            (dict(positions=pos[:5]), ValueError, "positions must have shape"),
            (dict(positions=pos[None]), ValueError, "positions must have shape"),
            (dict(positions=pos.cpu()), ValueError, "positions must live on"),
            (dict(cos=cos[:, :5], sin=sin[:, :5]), ValueError, "multiple of 16"), (dict(cos=cos[:3]), ValueError, "must be \\(P, R/2\\)"),
            (dict(cos=cos.double()), TypeError, "float32"), (dict(sin=sin.cpu()), ValueError, "cos and sin must live on"),
            (dict(pairs="both"), ValueError, "pairs must be"),
            (dict(q=q.clone().requires_grad_()), ValueError, "no backward pass"),
            (dict(v=v.clone().requires_grad_()), ValueError, "no backward pass"),
            (dict(cos=cos.clone().requires_grad_()), ValueError, "no backward pass")):
        with pytest.raises(err, match=msg):
            call(**kw)
    with forward_ad.dual_level():
        for name, x in (("q", q), ("k", k), ("v", v), ("cos", cos)):
            with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
                call(**{name: forward_ad.make_dual(x.clone(), torch.ones_like(x))})
    for a, b in zip(keep, bytes_of(c)):
        assert torch.equal(a, b)
    with torch.no_grad():
        call(q=q.clone().requires_grad_())
