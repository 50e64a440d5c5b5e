"""How many parts paged attention cuts the keys into, seen by the workspace that it asks
for: no more where the token buffer is padded or nothing is said of its sequence's length."""

import ctypes
import os

import pytest

FAKE = 0x1000


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


def test_calls_that_need_parts_have_them(lib):
    """A few tokens over many keys, on a chip of 256 CUs."""
    row = 4 * 128 + 8
    assert need(lib, 1, 1 << 16, hint=1) >= 32 * row * 32
    assert need(lib, 100, 1 << 16) >= 3200 * row * 16
    assert need(lib, 2048, 1 << 16, B=2) >= 2048 * 32 * row * 2
