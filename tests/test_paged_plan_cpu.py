"""How many parts paged attention cuts the keys into, seen by the workspace that it asks
for: no more where the token buffer is padded or nothing is said of its sequence's
length, and none that would make a call too large."""

import ctypes
import os

import pytest

FAKE = 0x1000
GIB = 1 << 30


@pytest.fixture
def lib():
    from low_bit_fake_quant import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built (run __graft_entry__.build())")
    return _lib.load(require_gpu=False)


def need(lib, T, keys, *, B=1, hint=0, hq=32, hk=8, d=128, causal=1, window=0, page=64):
    from low_bit_fake_quant import _lib
    p = _lib.PagedParams(q=FAKE, dtype=2, T=T, Hq=hq, Hk=hk, D=d, B=B, q_t=hq * d, q_h=d, k_codes=FAKE, k_scale=FAKE,
                         v_codes=FAKE, v_scale=FAKE, num_pages=4, page_shift=page.bit_length() - 1, block_table=FAKE,
                         table_stride=keys // page, table_cols=keys // page, seq_lens=FAKE, query_starts=FAKE,
                         max_query_len=hint, sm_scale=0.1, causal=causal, window=window, out=FAKE, out_t=hq * d, out_h=d)
    return lib.lbfq_paged_attention_workspace_bytes(ctypes.byref(p))


@pytest.mark.parametrize("T,keys", [(8192, 2048), (16384, 2048), (32768, 2048), (65536, 4096), (200000, 4096), (1 << 21, 4096)])
def test_a_padded_buffer_of_one_sequence_needs_no_more_parts(lib, T, keys):
    """The row tiles of the buffer fill the chip by themselves."""
    assert need(lib, T, keys) == need(lib, T, keys, hint=keys) == 0


@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("B", [1, 3, 64])
@pytest.mark.parametrize("hint", [0, 1, 4, 100])
def test_the_workspace_is_bounded(lib, hint, B, causal):
    for T in (B, 100, 1000, 4097, 50000, 1 << 20):
        for keys in (64, 1024, 32768, 1 << 20):
            for window in (0, 512):
                assert 0 <= need(lib, T, keys, B=B, hint=hint, causal=causal, window=window) <= GIB, (T, keys, window)


def test_calls_of_2_26_rows_and_more_are_taken_in_one_part(lib):
    """(several parts would be refused: the launch that joins them has a wave a row)"""
    for B, hint in ((1, 0), (1, 1), (2, 0), (5, 1)):
        assert need(lib, 1 << 21, 1 << 20, B=B, hint=hint) == 0
        assert need(lib, 1 << 21, 1 << 20, B=B, hint=hint, window=100) == 0


def test_calls_that_need_parts_have_them(lib):
    """A few tokens over many keys, on a chip of 256 CUs."""
    row = 4 * 128 + 8
    assert need(lib, 1, 1 << 16, hint=1) >= 32 * row * 32
    assert need(lib, 100, 1 << 16) >= 3200 * row * 16
    assert need(lib, 2048, 1 << 16, B=2) >= 2048 * 32 * row * 2


@pytest.mark.parametrize("B,T,keys,hq,hk,parts", [(16, 485, 2048, 32, 8, 2), (8, 477, 4032, 32, 8, 3), (2, 1421, 16000, 32, 8, 4),
                                                  (2, 432, 5056, 32, 8, 4)])
def test_parts_of_several_sequences_are_the_fastest(lib, B, T, keys, hq, hk, parts):
    """(the times of 1 to 8 parts stand above the rule)"""
    assert need(lib, T, keys, B=B, hq=hq, hk=hk) == parts * T * hq * (4 * 128 + 8) + 16
