"""The 4-bit cache's attention kernels, as built: none keeps anything in scratch memory or converts 32 values over its own
operands, and both units were looked at."""

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


@needs_build
@pytest.mark.skipif(not mfma_check.tools_available(), reason="no LLVM tools")
@pytest.mark.parametrize("unit", UNITS)
def test_conversions_do_not_lie_over_their_operands(unit):
    assert unit in BUILT, f"{unit} is not in the build directory"
    asm = mfma_check.disassemble(BUILT[unit])
    assert "v_cvt_scalef32_2xpk16" in asm and mfma_check.wide_conversion_overlaps(asm) == []
