"""The cache operators' host side without a GPU: the ctypes structs mirror the
header, the C entries refuse bad parameters before any launch, the Python entries
refuse CPU tensors, and the plain restatement of the format is right."""

import ctypes
import os
import re

import pytest
import torch

import kv_reference as ref
from conftest import REPO


def _fields(struct):
    text = open(os.path.join(REPO, "include", "lbfq.h")).read()
    body = re.search(r"typedef struct \{((?:(?!typedef struct).)*?)\}\s*" + struct, text, flags=re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    names = []
    for decl in body.split(";"):
        if decl.strip():
            parts = decl.replace("const", " ").split()
            names += [n.strip().lstrip("*").strip() for n in " ".join(parts[1:]).split(",")]
    return names


def test_structs_match_the_header():
    from low_bit_fake_quant import _lib
    for struct, cls in (("lbfq_qk_norm_params", _lib.QkNormParams), ("lbfq_qk_norm_grads", _lib.QkNormGrads),
                        ("lbfq_kv_write_params", _lib.KvWriteParams), ("lbfq_kv_read_params", _lib.KvReadParams),
                        ("lbfq_paged_params", _lib.PagedParams)):
        assert _fields(struct) == [f[0] for f in cls._fields_], struct


@pytest.fixture
def lib():
    from low_bit_fake_quant import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built (run __graft_entry__.build())")
    return _lib.load(require_gpu=False)


def _refused(lib, fn, p, changes):
    """Each change of one field of valid parameters is refused (no pointer is
    followed on these paths; fake addresses are enough)."""
    for field, value, msg in changes:
        saved = getattr(p, field)
        setattr(p, field, value)
        assert fn(ctypes.byref(p)) == -1, field
        assert msg in lib.lbfq_last_error().decode(), field
        setattr(p, field, saved)


FAKE = 0x1000


def test_qk_norm_entries_refuse(lib):
    from low_bit_fake_quant import _lib
    p = _lib.QkNormParams(q=FAKE, k=FAKE, dtype=2, B=1, S=4, Hq=2, Hk=1, D=128, q_b=0, q_s=256, q_h=128, k_s=128,
                          k_h=128, cos=FAKE, sin=FAKE, table_len=4, rot=128, eps=1e-6, q_out=FAKE, k_out=FAKE)
    bad = [("D", 96, "D must be"), ("dtype", 5, "bad dtype"), ("S", 0, "empty"), ("Hk", 0, "empty"), ("q", None, "missing"),
           ("rot", 24, "rot must be"), ("rot", 256, "rot must be"), ("table_len", 3, "the table has 3"),
           ("q_s", 129, "16-byte"), ("q", FAKE + 2, "16-byte"), ("cos", FAKE + 4, "16-byte"), ("B", 1 << 50, "too large"),
           ("Hq", 1 << 30, "too large")]
    _refused(lib, lambda x: lib.lbfq_qk_norm_rope(x, None), p, bad + [("q_out", None, "missing output")])
    g = _lib.QkNormGrads(dyq=FAKE, dyk=FAKE, dq=FAKE, dk=FAKE)
    _refused(lib, lambda x: lib.lbfq_qk_norm_rope_bwd(x, ctypes.byref(g), None), p, bad)
    _refused(lib, lambda x: lib.lbfq_qk_norm_rope_bwd(ctypes.byref(p), x, None), g,
             [("dyq", None, "missing gradient"), ("dq_weight", FAKE, "missing workspace"), ("dyk_h", 3, "16-byte"),
              ("dyk", FAKE + 8, "16-byte")])
    assert lib.lbfq_qk_norm_rope(None, None) == -1 and lib.lbfq_qk_norm_rope_bwd(ctypes.byref(p), None, None) == -1
    assert lib.lbfq_qk_norm_rope_bwd_rows(None) == 0
    assert lib.lbfq_qk_norm_rope_bwd_rows(ctypes.byref(p)) == 1


def test_cache_entries_refuse(lib):
    from low_bit_fake_quant import _lib
    cache = dict(k_codes=FAKE, k_scale=FAKE, v_codes=FAKE, v_scale=FAKE, num_pages=4, page_shift=4)
    bad = [("D", 32, "D must be"), ("page_shift", 3, "pages hold"), ("page_shift", 11, "pages hold"),
           ("num_pages", 0, "number of pages"), ("H", 0, "number of heads"), ("v_codes", None, "missing cache"),
           ("k_scale", FAKE + 1, "16-byte"), ("dtype", 3, "bad dtype")]
    w = _lib.KvWriteParams(k=FAKE, v=FAKE, dtype=1, T=3, H=2, D=64, k_t=128, k_h=64, v_t=128, v_h=64, slots=FAKE, **cache)
    _refused(lib, lambda x: lib.lbfq_kv_write(x, None), w,
             bad + [("T", 0, "number of tokens"), ("slots", None, "missing tensor"), ("v_t", 4, "16-byte"),
                    ("T", 1 << 39, "too large")])
    r = _lib.KvReadParams(B=1, H=2, D=64, max_len=5, block_table=FAKE, table_stride=1, table_cols=1, seq_lens=FAKE,
                          k_out=FAKE, v_out=FAKE, dtype=0, **cache)
    _refused(lib, lambda x: lib.lbfq_kv_read(x, None), r,
             bad + [("max_len", 0, "number of tokens"), ("B", 0, "number of tokens"), ("seq_lens", None, "missing tensor"),
                    ("table_cols", -1, "block table"), ("B", 1 << 31, "too large")])
    a = _lib.PagedParams(q=FAKE, dtype=2, T=2, Hq=4, Hk=2, D=128, B=1, q_t=512, q_h=128, block_table=FAKE, table_stride=9,
                         table_cols=9, seq_lens=FAKE, query_starts=FAKE, sm_scale=0.1, causal=1, out=FAKE, out_t=512,
                         out_h=128, **cache)
    _refused(lib, lambda x: lib.lbfq_paged_attention(x, None), a,
             [b for b in bad if b[0] not in ("H", "dtype", "v_codes")] +
             [("dtype", 0, "bf16 or fp16"), ("Hq", 3, "multiple of the key heads"), ("T", 0, "number of tokens"),
              ("table_cols", 0, "block table"), ("table_cols", 1 << 28, "block table"), ("q", None, "missing tensor"),
              ("v_codes", None, "missing tensor"), ("out_h", 4, "16-byte"), ("q", FAKE + 2, "16-byte"),
              ("sm_scale", 0.0, "sm_scale"), ("sm_scale", float("inf"), "sm_scale"), ("sm_scale", float("nan"), "sm_scale"),
              ("window", -1, "window")])
    # a long table: the keys are split, and the parts need a workspace
    a.table_cols = 4000
    need = lib.lbfq_paged_attention_workspace_bytes(ctypes.byref(a))
    assert need > 0
    a.workspace_bytes = need
    assert lib.lbfq_paged_attention(ctypes.byref(a), None) == -1 and b"workspace" in lib.lbfq_last_error()
    a.workspace, a.workspace_bytes = FAKE, need - 1
    assert lib.lbfq_paged_attention(ctypes.byref(a), None) == -1 and b"workspace" in lib.lbfq_last_error()
    assert lib.lbfq_paged_attention_workspace_bytes(None) == 0
    # sizes that the launch refuses need none, and are not divided by
    a.window = 5
    for name, bad in (("Hq", 1), ("Hk", 0), ("T", 1 << 62), ("T", 1 << 29), ("B", 0), ("table_cols", 1 << 62), ("page_shift", 60),
                      ("num_pages", 1 << 62)):
        old = getattr(a, name)
        setattr(a, name, bad)
        assert lib.lbfq_paged_attention_workspace_bytes(ctypes.byref(a)) == 0, name
        assert lib.lbfq_paged_attention(ctypes.byref(a), None) == -1, name
        setattr(a, name, old)
    assert lib.lbfq_paged_attention_workspace_bytes(ctypes.byref(a)) >= 0
    # more workgroups than a launch may have
    a.window, a.B, a.T, a.max_query_len, a.Hk, a.Hq = 0, 1 << 23, 1 << 23, 1, 2, 4
    assert lib.lbfq_paged_attention(ctypes.byref(a), None) == -1 and b"too large" in lib.lbfq_last_error()
    for p, fn in ((w, lib.lbfq_kv_write), (r, lib.lbfq_kv_read)):
        p.T = p.B = 1 << 29
        assert fn(ctypes.byref(p), None) == -1 and b"too large" in lib.lbfq_last_error()


def test_a_missing_host_module_is_said_loudly(lib, monkeypatch):
    import sys

    from low_bit_fake_quant import _lib
    monkeypatch.setattr(_lib, "_torch_ops", None)
    monkeypatch.setitem(sys.modules, "low_bit_fake_quant._lbfq_torch", None)
    monkeypatch.delattr(sys.modules["low_bit_fake_quant"], "_lbfq_torch", raising=False)
    with pytest.raises(_lib.HipLibraryError, match="build it"):
        _lib.torch_ops()


def test_python_entries_refuse_cpu_tensors():
    from low_bit_fake_quant import empty_kv_cache, paged_attention, qk_norm_rope, read_kv_cache, rotary_table, write_kv_cache
    c = empty_kv_cache(2, 16, 1, 64, device="cpu")
    x, i = torch.zeros(1, 1, 64, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    t = torch.zeros(1, 2, dtype=torch.int32)
    for call in (lambda: write_kv_cache(x, x, c, i.long()), lambda: read_kv_cache(c, t, i, 1),
                 lambda: paged_attention(x, c, t, i, torch.zeros(2, dtype=torch.int32)),
                 lambda: qk_norm_rope(x, x, None, None, *rotary_table(2, 64))):
        with pytest.raises(ValueError, match="CUDA device"):
            call()
    for kw, msg in (((2, 24, 1, 64), "page_size"), ((2, 16, 1, 96), "D must be"), ((0, 16, 1, 64), "positive"),
                    ((2, 16, 0, 64), "positive")):
        with pytest.raises(ValueError, match=msg):
            empty_kv_cache(*kw, device="cpu")


def test_the_64_bit_format_agrees_with_torch_and_the_oracle():
    from oracle import quant as oquant
    g = torch.Generator().manual_seed(0)
    x = torch.randn(50, 128, generator=g) * torch.logspace(-8, 6, 50)[:, None]
    x[0] = 0
    x[1, :32] = 448.0 * 2 ** -3  # amax / 448 a power of two exactly
    val, e = ref.mx_encode(x)
    q = (x.unflatten(-1, (-1, 32)) * torch.exp2(-e.float())[..., None]).flatten(-2)
    assert torch.equal(q.clamp(-448, 448).to(torch.float8_e4m3fn).double(), val)
    assert (val.abs() <= 448).all()
    codes, scale = oquant.mxfp8_qk_quant(x[None, :, None])
    assert torch.equal(torch.as_tensor(scale).reshape(50, 4).double(), torch.exp2(e.double()))
    every = torch.arange(256, dtype=torch.uint8)
    every = every[(every & 127) != 127]
    dec = ref.mx_decode(torch.cat([every, every[:2]]).view(torch.float8_e4m3fn).view(8, 32),
                        torch.full((8, 1), 130, dtype=torch.uint8)).flatten()[:254]
    assert torch.equal(dec, every.view(torch.float8_e4m3fn).double() * 8)


def test_rotary_table_angles_are_formed_in_64_bits():
    from low_bit_fake_quant import rotary_table
    cos, sin = rotary_table(200000, 64)
    import math
    for pos, i in ((199999, 0), (123457, 3), (1, 31)):
        a = pos * 10000.0 ** (-2 * i / 64)
        assert abs(cos[pos, i].item() - math.cos(a)) < 2 ** -23 and abs(sin[pos, i].item() - math.sin(a)) < 2 ** -23
