"""No result of a matrix instruction is used before it is there, along any way through any kernel of the built library."""

import pytest

from swiftlet_amd import build
from tests import matrix_waits as M


def body(*lines):
    text = "0000000000000000 <f>:\n" + "".join(f"\t{line}  // {4 * i:012X}: 00000000\n" for i, line in enumerate(lines))
    (name, code), = M.functions(text)
    return code


MFMA = "v_mfma_f32_16x16x32_f16 v[0:3], v[8:11], v[12:15], 0"


@pytest.mark.parametrize("lines,uses", [
    ([MFMA, "s_nop 7", "v_add_f32_e32 v5, v0, v6", "s_endpgm"], 0),
    ([MFMA, "s_nop 6", "v_add_f32_e32 v5, v0, v6", "s_endpgm"], 1),
    ([MFMA, "s_nop 6", "v_mov_b32_e32 v0, v6", "s_endpgm"], 0),
    ([MFMA, "s_nop 6", "global_store_dword v0, v6, s[0:1]", "s_endpgm"], 1),
    ([MFMA, "v_add_f32_e32 v5, v4, v6", "s_endpgm"], 0),
    ([MFMA, "v_mfma_f32_16x16x32_f16 v[0:3], v[8:11], v[12:15], v[0:3]", "s_nop 7", "v_add_f32_e32 v5, v0, v6", "s_endpgm"], 0),
    ([MFMA, "v_mfma_f32_16x16x32_f16 v[4:7], v[0:3], v[12:15], 0", "s_endpgm"], 1),
    (["v_mfma_f32_16x16x4_f32 v[0:3], v8, v12, 0", "s_nop 8", "v_add_f32_e32 v5, v3, v6", "s_endpgm"], 1),
    # a branch that skips the waits, ahead and back
    ([MFMA, "s_cbranch_scc1 1", "s_nop 7", "v_add_f32_e32 v5, v0, v6", "s_endpgm"], 1),
    ([MFMA, "s_nop 6", "s_cbranch_scc1 1", "s_nop 7", "v_add_f32_e32 v5, v0, v6", "s_endpgm"], 0),
    (["v_add_f32_e32 v5, v0, v6", MFMA, "s_cbranch_scc1 65533", "s_endpgm"], 1),
    ([MFMA, "s_branch 1", "s_endpgm", "v_add_f32_e32 v5, v0, v6", "s_endpgm"], 1)], ids=str)
def test_what_it_finds(lines, uses):
    assert len(M.early(body(*lines))) == uses


def test_the_library():
    if not M.OBJDUMP.exists():
        pytest.skip("no llvm-objdump")
    if not build.LIB.exists():
        build.build()
    seen, bad = 0, []
    for text in M.listings(build.LIB):
        if "v_mfma" in text:
            for name, code in M.functions(text):
                seen += sum("mfma" in op for _, op, _ in code)
                bad += [f"{name}: {made} -> {used} after {waited}" for made, used, waited in M.early(code)]
    assert seen > 1000  # the library was read at all
    assert not bad, "\n".join(bad)
