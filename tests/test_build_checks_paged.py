"""The 4-bit cache's attention kernels, as built: none keeps anything in scratch memory, and both units were looked at."""

import os

import pytest

from test_build_checks import OBJS, mfma_check

UNITS = ("lbfq_paged4.o", "lbfq_paged4_chunk.o")
BUILT = {os.path.basename(o): o for o in OBJS}

needs_build = pytest.mark.skipif(not OBJS, reason="no built objects")


@needs_build
@pytest.mark.parametrize("unit", UNITS)
def test_no_scratch_memory(unit):
    """A wait for scratch memory is also one for the copies into LDS that are on their way."""
    import build_lib
    assert unit in BUILT, f"{unit} is not in the build directory"
    s_path = build_lib.device_asm(BUILT[unit])
    if not os.path.exists(s_path):
        pytest.skip("no device assembly (built without -save-temps)")
    with open(s_path) as f:
        text = f.read()
    assert text.count("; -- End function") >= 4  # bf16 and fp16, heads of 64 and 128
    assert mfma_check.scratch_kernels(text, "paged") == []
