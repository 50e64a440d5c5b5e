"""The parts that paged attention over 4 bits cuts the keys into, seen by the workspace that it asks for."""

import pytest

import test_paged_plan_cpu as eight
from test_paged_plan_cpu import GIB, lib  # noqa: F401  (lib: a fixture)


@pytest.fixture(autouse=True)
def in_4_bits(monkeypatch):
    from low_bit_fake_quant import _lib
    whole = _lib.PagedParams
    monkeypatch.setattr(_lib, "PagedParams", lambda **kw: whole(bits=4, **kw))


test_a_padded_buffer_of_one_sequence_needs_no_more_parts = eight.test_a_padded_buffer_of_one_sequence_needs_no_more_parts
test_the_workspace_is_bounded = eight.test_the_workspace_is_bounded
test_calls_of_2_26_rows_and_more_are_taken_in_one_part = eight.test_calls_of_2_26_rows_and_more_are_taken_in_one_part


def parts(lib, T, keys, **kw):  # noqa: F811
    need = eight.need(lib, T, keys, **kw)
    return (need - 16) // (T * kw.get("hq", 32) * (4 * kw.get("d", 128) + 8)) if need else 1


@pytest.mark.parametrize("B,keys,hq,hk,want", [(1, 704, 32, 8, 1), (1, 5056, 32, 8, 16), (1, 40000, 32, 8, 32), (24, 4032, 32, 8, 1),
                                               (48, 16000, 32, 8, 4), (8, 8000, 40, 40, 1), (12, 16000, 12, 12, 4), (128, 8000, 32, 8, 1)])
def test_parts_of_single_tokens(lib, B, keys, hq, hk, want):  # noqa: F811
    assert parts(lib, B, keys, B=B, hint=1, hq=hq, hk=hk) == want


# (the last: 19 row tiles and sequences' ends, 8 heads: the largest s with 120 s s 152 <= 64 * 4032)
@pytest.mark.parametrize("B,T,keys,hq,hk,causal,want", [(1, 4680, 32768, 12, 12, 0, 2), (1, 4680, 9408, 12, 12, 0, 1),
                                                        (1, 700, 8000, 12, 12, 0, 6), (1, 8192, 8192, 32, 8, 1, 1),
                                                        (8, 477, 4032, 32, 8, 1, 3)])
def test_parts_of_chunks(lib, B, T, keys, hq, hk, causal, want):  # noqa: F811
    assert parts(lib, T, keys, B=B, hq=hq, hk=hk, causal=causal) == want
