"""The build's check on generated assembly that matrix-core instructions are never masked off."""
import importlib

import pytest

GOOD = """
_Zkernel: ; @_Zkernel
	s_and_saveexec_b64 s[0:1], vcc
	s_cbranch_execz .LBB0_2
	v_mfma_f32_16x16x32_bf16 v[0:3], v[8:11], v[4:7], v[0:3]
.LBB0_2:
	s_or_b64 exec, exec, s[0:1]
	s_and_saveexec_b64 s[0:1], vcc
	ds_write_b128 v1, v[0:3]
	s_or_b64 exec, exec, s[0:1]
	v_mfma_f32_16x16x4_f32 v[0:3], v8, v4, v[0:3]
	s_endpgm
"""


def test_masked_mfma_is_found(pkg):
    build = importlib.import_module(pkg.__name__ + ".build")
    assert build.check_no_masked_mfma(GOOD, "good") == 2
    bad = GOOD.replace("	s_cbranch_execz .LBB0_2\n", "")
    with pytest.raises(RuntimeError, match="_Zkernel: `v_mfma_f32_16x16x32_bf16.*executes whatever"):
        build.check_no_masked_mfma(bad, "bad")
