"""Parts of single tokens over 4 bits: as many as even out the sequences of a batch, none where there are enough of those
to do it by themselves."""

import pytest

import test_paged_plan_unequal_cpu as plans
from test_paged_plan_cpu import lib  # noqa: F401  (a fixture)


@pytest.mark.parametrize("B,keys,hk,want", [
    (48, 11968, 8, 1), (48, 12032, 8, 3), (48, 20032, 8, 5), (96, 20032, 8, 4), (128, 11968, 8, 1), (128, 12032, 8, 3),
    (128, 20032, 8, 3), (192, 12032, 8, 2), (192, 40000, 8, 2), (256, 11968, 8, 1), (256, 12032, 8, 1), (256, 40000, 8, 1),
    (512, 12032, 8, 1), (512, 20032, 1, 5), (64, 12032, 40, 1), (32, 12032, 40, 2), (2, 40000, 8, 16), (3000, 12032, 8, 1)])
def test_parts_go_by_what_the_sequences_fill(lib, B, keys, hk, want):  # noqa: F811
    parts, share = plans.plan(lib, B, keys, B=B, hint=1, hq=hk, hk=hk)
    assert (parts, share) == (want, 0)
