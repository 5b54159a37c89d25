"""The build's assembly check on the block kernels that write their MFMAs as inline assembly, which nothing pads for
the compiler: accumulation registers, and the kernels as built here."""
import re

import pytest

from tcc_spmm_amd import asm_check, build

MFMA = "\tv_mfma_scale_f32_16x16x128_f8f6f4 a[0:3], v[0:7], v[8:15], a[0:3], v16, v17 op_sel_hi:[0,0,0]\n"


def _listing(body: str) -> str:
    return "_ZN4test12multiplyWideEv:\n" + body + "\ts_endpgm\n.Lfunc_end0:\n"


def test_accumulation_registers_are_results():
    early = _listing(MFMA + "\ts_nop 3\n\tv_accvgpr_read_b32 v20, a2\n")
    late = _listing(MFMA + "\ts_nop 15\n\ts_nop 3\n\tv_accvgpr_read_b32 v20, a2\n")
    assert len(asm_check.check(early, "multiplyWide")) == 1
    assert asm_check.check(late, "multiplyWide") == []
    # v2 is another register than a2
    assert asm_check.check(_listing(MFMA + "\tv_mov_b32_e32 v20, v30\n"), "multiplyWide") == []


def test_only_the_named_kernels_are_looked_at():
    other = _listing(MFMA + "\tv_accvgpr_read_b32 v20, a2\n").replace("multiplyWide", "multiplyRows")
    assert asm_check.check(other + _listing(MFMA), "multiplyWide") == []
    assert asm_check.check(other, "multiplyWide") == ["no kernels found in the assembly"]


@pytest.mark.parametrize("src", list(build.INLINE_MFMA), ids=lambda src: src.stem)
def test_kernels_as_built(src):
    """They pass; with a read planted right behind each of their MFMAs in the listing they do not."""
    build.BUILD.mkdir(exist_ok=True)
    build.check_inline_mfma(src)
    listing = (build.BUILD / f"{src.stem}-gfx950.s").read_text()
    name = build.INLINE_MFMA[src]
    planted, count = re.subn(r"(\tv_mfma_\S+ a\[(\d+):\d+\].*\n)", r"\1\tv_accvgpr_read_b32 v0, a\2\n", listing)
    assert count > 64 and any("MFMA result read" in p for p in asm_check.check(planted, name))
