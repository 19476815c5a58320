"""The build's check that no matrix-core instruction runs with an empty lane mask: the forms in which a listing narrows
EXEC, the branches that do and do not skip on it, and the other side of a condition."""
import importlib

import pytest

MFMA = "v_mfma_f32_16x16x32_bf16 v[0:3], v[8:11], v[4:7], v[0:3]"


def listing(body):
    return "_Zkernel: ; @_Zkernel\n" + "".join(line + "\n" if line.startswith(".") else f"\t{line}\n" for line in body.strip().split("; "))


SOUND = [
    MFMA,
    f"s_and_saveexec_b64 s[0:1], vcc; s_cbranch_execz .L1; {MFMA}; .L1:; s_or_b64 exec, exec, s[0:1]; {MFMA}",
    f"s_and_saveexec_b64 s[0:1], vcc; ds_write_b128 v1, v[0:3]; s_or_b64 exec, exec, s[0:1]; {MFMA}",
    f"s_and_saveexec_b64 s[0:1], vcc; ds_write_b128 v1, v[0:3]; s_mov_b64 exec, -1; {MFMA}",
    # both sides, each behind a branch of its own
    f"s_and_saveexec_b64 s[0:1], vcc; s_xor_b64 s[0:1], exec, s[0:1]; s_cbranch_execz .L1; {MFMA}; .L1:; "
    f"s_or_saveexec_b64 s[0:1], s[0:1]; s_xor_b64 exec, exec, s[0:1]; s_cbranch_execz .L2; {MFMA}; .L2:; s_or_b64 exec, exec, s[0:1]; {MFMA}",
    # a loop that lanes leave one by one
    f".L1:; {MFMA}; s_andn2_b64 exec, exec, s[2:3]; s_cbranch_execnz .L1; s_or_b64 exec, exec, s[2:3]; s_endpgm",
    # a branch on an EXEC that nothing has narrowed is not taken
    f"s_cbranch_execz .L1; s_branch .L2; .L1:; s_and_b64 exec, exec, vcc; {MFMA}; .L2:; {MFMA}",
    # the masks that registers hold are no EXEC
    f"s_and_b64 s[0:1], exec, vcc; s_andn2_b64 vcc, exec, s[0:1]; s_cbranch_vccnz .L1; {MFMA}; .L1:; s_endpgm",
]

MASKED = [
    ("s_and_saveexec", f"s_and_saveexec_b64 s[0:1], vcc; {MFMA}"),
    # neither a label nor a branch on something else skips an empty EXEC
    ("s_and_saveexec", f"s_and_saveexec_b64 s[0:1], vcc; .L1:; {MFMA}; s_or_b64 exec, exec, s[0:1]"),
    ("s_and_saveexec", f"s_and_saveexec_b64 s[0:1], vcc; s_cbranch_scc1 .L1; {MFMA}; .L1:; s_or_b64 exec, exec, s[0:1]"),
    ("s_and_saveexec", f"s_and_saveexec_b64 s[0:1], vcc; s_cbranch_vccz .L1; s_nop 0; .L1:; {MFMA}"),
    # where the branch on an empty EXEC arrives
    ("s_and_saveexec", f"s_and_saveexec_b64 s[0:1], vcc; s_cbranch_execz .L1; s_nop 0; .L1:; {MFMA}"),
    ("s_and_b64 exec", f"s_and_b64 exec, exec, vcc; {MFMA}"),
    ("s_andn2_b64 exec", f"s_andn2_b64 exec, exec, s[0:1]; {MFMA}"),
    ("s_andn2_saveexec", f"s_andn2_saveexec_b64 s[0:1], vcc; {MFMA}"),
    ("v_cmpx", f"v_cmpx_gt_u32 v1, v2; {MFMA}"),
    ("s_mov_b64 exec", f"s_mov_b64 exec, s[4:5]; {MFMA}"),
    # the other side of a condition
    ("s_xor_b64 exec", f"s_and_saveexec_b64 s[0:1], vcc; s_cbranch_execz .L1; s_nop 0; .L1:; s_or_saveexec_b64 s[0:1], s[0:1]; "
                       f"s_xor_b64 exec, exec, s[0:1]; {MFMA}; s_or_b64 exec, exec, s[0:1]"),
    # an inner restoring is not the outer one
    ("s_and_saveexec", f"s_and_saveexec_b64 s[0:1], vcc; s_and_saveexec_b64 s[2:3], vcc; s_nop 0; s_or_b64 exec, exec, s[2:3]; {MFMA}"),
    # behind a loop, before what the lanes had is back
    ("s_andn2_b64 exec", f".L1:; s_nop 0; s_andn2_b64 exec, exec, s[2:3]; s_cbranch_execnz .L1; {MFMA}"),
    # on one path of two
    ("s_and_saveexec", f"s_cbranch_scc1 .L1; s_and_saveexec_b64 s[0:1], vcc; .L1:; {MFMA}"),
]


@pytest.fixture(scope="module")
def check(pkg):
    return importlib.import_module(pkg.__name__ + ".build").check_no_masked_mfma


@pytest.mark.parametrize("body", SOUND)
def test_sound_listings_pass(check, body):
    assert check(listing(body), "sound") == body.count("v_mfma")


@pytest.mark.parametrize("by,body", MASKED)
def test_masked_listings_are_refused(check, by, body):
    with pytest.raises(RuntimeError, match=f"_Zkernel: `v_mfma.*executes whatever `{by}"):
        check(listing(body), "masked")
