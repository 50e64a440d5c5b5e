"""The 4-bit cache's and append_kv_cache's host side without a GPU: structs, refusals, the
plain restatement of the format."""

import ctypes

import pytest
import torch

import kv4_reference as ref
import kv_reference as ref8
from test_cache_operators_cpu import FAKE, _fields, _refused, lib  # noqa: F401  (lib: a fixture)


def test_structs_match_the_header():
    from low_bit_fake_quant import _lib
    assert _fields("lbfq_kv_append_params") == [f[0] for f in _lib.KvAppendParams._fields_]


def test_append_entry_refuses(lib):  # noqa: F811
    from low_bit_fake_quant import _lib
    p = _lib.KvAppendParams(q=FAKE, k=FAKE, v=FAKE, dtype=2, T=3, Hq=4, Hk=2, D=128, q_t=512, q_h=128, k_t=256, k_h=128,
                            v_t=256, v_h=128, cos=FAKE, sin=FAKE, table_len=9, rot=64, positions=FAKE, pos_t=1, q_out=FAKE,
                            slots=FAKE, k_codes=FAKE, k_scale=FAKE, v_codes=FAKE, v_scale=FAKE, num_pages=4, page_shift=4,
                            bits=4)
    _refused(lib, lambda x: lib.lbfq_kv_append(x, None), p,
             [("D", 32, "D must be"), ("page_shift", 3, "pages hold"), ("page_shift", 11, "pages hold"),
              ("num_pages", 0, "number of pages"), ("Hk", 0, "number of heads"), ("Hq", -1, "number of heads"),
              ("Hq", 1 << 16, "number of heads"), ("v_codes", None, "missing cache"), ("k_scale", FAKE + 1, "16-byte"),
              ("dtype", 3, "bad dtype"), ("T", 0, "number of tokens"), ("slots", None, "missing tensor"),
              ("positions", None, "missing tensor"), ("cos", None, "missing tensor"), ("q", None, "missing tensor"),
              ("q_out", None, "missing tensor"), ("v_t", 4, "16-byte"), ("q_h", 1, "16-byte"), ("q_out", FAKE + 8, "16-byte"),
              ("sin", FAKE + 4, "16-byte"), ("rot", 24, "rot must be"), ("rot", 0, "rot must be"), ("rot", 144, "rot must be"),
              ("table_len", -1, "bad table"), ("T", 1 << 39, "too large"), ("bits", 5, "4 or 8 bits")])
    assert lib.lbfq_kv_append(None, None) == -1


def test_other_entries_refuse_other_widths(lib):  # noqa: F811
    from low_bit_fake_quant import _lib
    cache = dict(k_codes=FAKE, k_scale=FAKE, v_codes=FAKE, v_scale=FAKE, num_pages=4, page_shift=4)
    w = _lib.KvWriteParams(k=FAKE, v=FAKE, dtype=1, T=3, H=2, D=64, k_t=128, k_h=64, v_t=128, v_h=64, slots=FAKE, **cache)
    r = _lib.KvReadParams(B=1, H=2, D=64, max_len=5, block_table=FAKE, table_stride=1, table_cols=1, seq_lens=FAKE,
                          k_out=FAKE, v_out=FAKE, dtype=0, **cache)
    a = _lib.PagedParams(q=FAKE, dtype=2, T=2, Hq=4, Hk=2, D=128, B=1, q_t=512, q_h=128, block_table=FAKE, table_stride=9,
                         table_cols=9, seq_lens=FAKE, query_starts=FAKE, sm_scale=0.1, causal=1, out=FAKE, out_t=512,
                         out_h=128, **cache)
    for fn, p in ((lib.lbfq_kv_write, w), (lib.lbfq_kv_read, r), (lib.lbfq_paged_attention, a)):
        _refused(lib, lambda x: fn(x, None), p, [("bits", b, "4 or 8 bits") for b in (-4, 1, 6, 16)])
    a.bits = 5
    assert lib.lbfq_paged_attention_workspace_bytes(ctypes.byref(a)) == 0


def test_python_entries_refuse_cpu_tensors():
    from low_bit_fake_quant import append_kv_cache, empty_kv_cache, paged_attention, read_kv_cache, rotary_table, write_kv_cache
    c = empty_kv_cache(2, 16, 1, 64, device="cpu", bits=4)
    assert c.k_codes.shape == (2, 1, 16, 32) and c.k_codes.dtype == torch.float4_e2m1fn_x2 and c.v_scale.shape == (2, 1, 16, 2)
    x, i = torch.zeros(1, 1, 64, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    t = torch.zeros(1, 2, dtype=torch.int32)
    for call in (lambda: write_kv_cache(x, x, c, i.long()), lambda: read_kv_cache(c, t, i, 1),
                 lambda: paged_attention(x, c, t, i, torch.zeros(2, dtype=torch.int32)),
                 lambda: append_kv_cache(x, x, x, c, i.long(), *rotary_table(2, 64), i)):
        with pytest.raises(ValueError, match="CUDA device"):
            call()
    for bits in (0, 2, 16):
        with pytest.raises(ValueError, match="bits must be"):
            empty_kv_cache(2, 16, 1, 64, device="cpu", bits=bits)


def test_the_64_bit_format():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(50, 128, generator=g) * torch.logspace(-8, 6, 50)[:, None]
    x[0] = 0
    x[1, :32] = 6.0 * 2 ** -3  # amax / 6 a power of two exactly
    val, e = ref.encode(x)
    assert set(val.abs().unique().tolist()) <= set(ref.VALUES) and (e[0] == -15).all() and (e[1, 0] == -3).all()
    q = x.double() / torch.exp2(e.double()).repeat_interleave(32, -1)
    # the nearest of all values, and the even code of two
    table = torch.tensor(ref.VALUES, dtype=torch.float64)
    apart = (q.abs()[..., None] - table).abs()
    assert torch.equal(apart.amin(-1), (q.abs() - val.abs()).abs())
    middle = torch.tensor([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 4]).float()
    assert ref.encode(middle)[0][0, :7].tolist() == [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0]
    # every value of 4 bits is one of 8
    every = torch.arange(256, dtype=torch.uint8).view(2, 128)
    v = ref.values(every)
    assert torch.equal(ref8.mx_decode(v.to(torch.float8_e4m3fn), torch.full((2, 8), 127, dtype=torch.uint8)), v)
