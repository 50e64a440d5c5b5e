"""Two unequal parts of a sequence's keys (paged attention over 4 bits): which calls get them, and how long they are."""

import ctypes

import pytest

from test_paged_plan_cpu import FAKE, lib  # noqa: F401  (lib: a fixture)


def plan(lib, T, keys, *, B=1, hint=0, hq=16, hk=16, d=128, causal=False, window=None, bits=4, dtype=2, page=64):  # noqa: F811
    """(parts, of 65536 what the first has or 0) of a call whose table holds `keys`."""
    from low_bit_fake_quant import _lib
    p = _lib.PagedParams(q=FAKE, dtype=dtype, T=T, Hq=hq, Hk=hk, D=d, B=B, q_t=hq * d, q_h=d, k_codes=FAKE, k_scale=FAKE,
                         v_codes=FAKE, v_scale=FAKE, num_pages=4, page_shift=page.bit_length() - 1, block_table=FAKE,
                         table_stride=keys // page, table_cols=keys // page, seq_lens=FAKE, query_starts=FAKE,
                         max_query_len=hint, sm_scale=0.1, causal=causal, window=window or 0, out=FAKE, out_t=hq * d, out_h=d,
                         bits=bits)
    share = ctypes.c_int(-1)
    parts = lib.lbfq_paged_attention_parts(ctypes.byref(p), ctypes.byref(share))
    need = lib.lbfq_paged_attention_workspace_bytes(ctypes.byref(p))
    assert need == (0 if parts <= 1 else parts * T * hq * (4 * d + 8) + 16)
    return parts, share.value


@pytest.mark.parametrize("T,keys,kw", [
    (4680, 32768, dict(hq=12, hk=12)), (3800, 32768, dict(hq=12, hk=12)), (2700, 8192, {}), (2900, 8192, dict(causal=True)),
    (1400, 8192, dict(hq=32, hk=8)), (2700, 6144, dict(hq=24, hk=24, d=64, dtype=1))])
def test_row_tiles_that_fill_more_than_half_of_the_chip_have_them(lib, T, keys, kw):  # noqa: F811
    parts, share = plan(lib, T, keys, **kw)
    assert parts == 2 and 32768 <= share < 65536


@pytest.mark.parametrize("T,keys,kw", [
    (4680, 32768, dict(hq=12, hk=12, bits=8)),  # 8 bits
    (5000, 8192, dict(causal=True)),  # a prompt, whose row tiles differ
    (8192, 8192, {}), (1000, 8192, {}),  # row tiles for more than the chip, and for less than half of it
    (4680, 32768, dict(hq=12, hk=12, B=2)),  # several sequences
    (4680, 256, dict(hq=12, hk=12)), (16, 8192, dict(hint=1, hk=8))])
def test_others_have_equal_parts(lib, T, keys, kw):  # noqa: F811
    parts, share = plan(lib, T, keys, **kw)
    assert parts >= 1 and share == 0


def test_the_second_part_is_never_the_longer_one(lib):  # noqa: F811
    """(the second part of a sequence is cut off at the first one's length)"""
    seen = 0
    for T in range(1, 9000, 61):
        for keys in (256, 1024, 2048, 4096, 8192, 16384, 32768, 65536, 1 << 20):
            for hq, hk in ((12, 12), (32, 8), (40, 40), (8, 1), (16, 16), (5, 5)):
                for d in (64, 128):
                    parts, share = plan(lib, T, keys, hq=hq, hk=hk, d=d)
                    assert share == 0 or (parts == 2 and 32768 <= share < 65536), (T, keys, hq, hk, d)
                    seen += share > 0
    assert seen > 100


def test_bad_parameters_have_no_parts(lib):  # noqa: F811
    from low_bit_fake_quant import _lib
    share = ctypes.c_int(-1)
    assert lib.lbfq_paged_attention_parts(ctypes.byref(_lib.PagedParams(bits=5)), ctypes.byref(share)) == 0 and share.value == 0
    assert lib.lbfq_paged_attention_parts(None, None) == 0
