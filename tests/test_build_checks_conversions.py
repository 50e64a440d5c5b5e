"""The build's check of conversions of 32 values: their result must not lie over an operand."""

from test_build_checks import OBJS, mfma_check

import pytest


def test_parser_flags_results_over_operands():
    asm = ("\tv_cvt_scalef32_2xpk16_fp6_f32 v[36:41], v[34:49], v[2:17], 1.0  // 0\n"
           "\tv_cvt_scalef32_2xpk16_fp6_f32 v[18:23], v[2:17], v[50:65], v18\n"
           "\tv_cvt_scalef32_2xpk16_fp6_f32 v[82:87], v[50:65], v[34:49], v94\n"
           "\tv_cvt_scalef32_pk32_f32_fp6 v[2:33], v[82:87], v94\n"
           "\tv_cvt_scalef32_pk32_f32_fp6 v[2:33], v[30:35], v94\n"
           "\tv_cvt_scalef32_pk_bf16_fp4 v1, v1, v2\n")
    bad = mfma_check.wide_conversion_overlaps(asm)
    assert len(bad) == 3 and "v[36:41]" in bad[0] and "v18" in bad[1] and "v[30:35]" in bad[2]


@pytest.mark.skipif(not OBJS or not mfma_check.tools_available(), reason="no built objects or no LLVM tools")
def test_built_objects_have_none():
    for o in OBJS:
        if "paged4" in o:
            asm = mfma_check.disassemble(o)
            assert "v_cvt_scalef32_2xpk16" in asm and not mfma_check.wide_conversion_overlaps(asm)
