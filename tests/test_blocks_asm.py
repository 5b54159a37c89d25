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


def _ring(between, wait=8, extra=""):
    """A loop of one counted wait: `between` loads to LDS a turn, and before it eight."""
    row = "\tbuffer_load_dwordx4 v9, s[4:7], 0 offen lds\n"
    body = row * 8 + ".LBB0_1:\n" + extra + f"\t;;#ASMSTART\n\ts_waitcnt vmcnt({wait}) lgkmcnt(0)\n\ts_barrier\n\t;;#ASMEND\n"
    return _listing(body + row * between + "\ts_cbranch_scc1 .LBB0_1\n")


def test_counted_waits_are_held_to_their_counts():
    load = "\tglobal_load_ushort v3, v4, s[2:3]\n"
    check = lambda text, waits: asm_check.check_counted_waits(text, "multiplyWide", waits)  # noqa: E731
    assert check(_ring(4), {8: (8, {4, 8})}) == []
    assert check(_ring(4, extra=load), {9: (8, {4, 8})})[0].endswith("no count is known of")
    assert check(_ring(4, 9, load), {9: (8, {4, 8})}) == []
    # the load that was counted on is not there
    assert check(_ring(4, 9), {9: (8, {4, 8})}) == [
        "_ZN4test12multiplyWideEv: `s_waitcnt vmcnt(9) lgkmcnt(0)` may leave 9 loads to LDS outstanding, not 8"]
    # a load to LDS too few, or one that is not a load to LDS any more
    assert "3 loads to LDS between" in check(_ring(3), {8: (8, {4, 8})})[0]
    assert check("", {8: (8, {4})}) == ["no kernels found in the assembly"]


@pytest.mark.parametrize("src", list(build.COUNTED_WAITS), ids=lambda src: src.stem)
def test_counted_waits_as_built(src):
    """They pass; a memory load taken out of a loop, moved to the other side of the next wait, or made an ordinary one
    does not, whichever it is."""
    build.BUILD.mkdir(exist_ok=True)
    build.check_inline_mfma(src)
    listing = (build.BUILD / f"{src.stem}-gfx950.s").read_text()
    for kernels, waits in build.COUNTED_WAITS[src].items():
        lines = listing.split("\n")
        starts = [i for i, line in enumerate(lines) if re.match(r"^_Z\S+:", line) and kernels in line]
        checked = 0
        for start in starts:
            end = next(i for i in range(start, len(lines)) if lines[i].startswith(".Lfunc_end"))
            kernel = lines[start:end + 1]
            ring = [i for i, line in enumerate(kernel) if re.search(r"s_waitcnt vmcnt\([1-9]\d*\) lgkmcnt", line)
                    and "s_barrier" in kernel[i + 1]]
            if not ring:  # a form of two stages, whose waits are for everything
                continue
            for at in (i for i in range(ring[0] + 2, ring[-1]) if " lds" in kernel[i] or "load_ushort" in kernel[i]):
                gone = kernel[:at] + kernel[at + 1:]
                wait = next(i for i in ring if i > at) - 1
                late = gone[:wait + 1] + [kernel[at]] + gone[wait + 1:]
                plain = kernel[:at] + [kernel[at].replace(" lds", "")] + kernel[at + 1:]
                for text in (gone, late) + ((plain,) if " lds" in kernel[at] else ()):
                    assert asm_check.check_counted_waits("\n".join(text), kernels, waits), kernel[at]
                checked += 1
        assert checked > 10


INLINE = "\t;;#ASMSTART\n" + MFMA + "\t;;#ASMEND\n"


@pytest.mark.parametrize("writes", ["v_mov_b32_e32 v3, v30", "v_and_or_b32 v16, v30, v31, v32", "v_accvgpr_write_b32 a2, 0",
                                    "v_perm_b32 v15, v30, v31, s0"])
def test_an_inline_mfma_right_behind_its_operand(writes):
    """Any operand, the sum and the scales among them; not for other registers, or two wait states later, or where the
    compiler itself places the MFMA."""
    check = lambda between, mfma=INLINE: asm_check.check(_listing(f"\t{writes}\n" + between + mfma), "multiplyWide")  # noqa: E731
    assert len(check("")) == 1 and "0 wait states before" in check("")[0]
    assert len(check("\ts_mov_b32 s0, s1\n")) == 1
    assert len(check(".LBB0_2:\n\ts_nop 0\n")) == 1  # a label is no instruction
    assert check("\ts_nop 1\n") == [] and check("\ts_mov_b32 s0, s1\n\tds_read_b32 v40, v41\n") == []
    assert check("", MFMA) == []
    other = writes.replace(" v3,", " v33,").replace(" v16,", " v36,").replace(" a2,", " a22,").replace(" v15,", " v35,")
    assert asm_check.check(_listing(f"\t{other}\n" + INLINE), "multiplyWide") == []


@pytest.mark.parametrize("src", list(build.INLINE_MFMA), ids=lambda src: src.stem)
def test_operands_as_built(src):
    """With a write of an operand planted right in front of every inline MFMA the kernels do not pass."""
    build.BUILD.mkdir(exist_ok=True)
    build.check_inline_mfma(src)
    listing = (build.BUILD / f"{src.stem}-gfx950.s").read_text()
    planted, count = re.subn(r"(\t;;?#ASMSTART\n\tv_mfma_\S+ a\[\d+:\d+\], v\[(\d+):)", r"\tv_mov_b32_e32 v\2, 0\n\1", listing)
    problems = asm_check.check(planted, build.INLINE_MFMA[src])
    assert count > 64 and sum("wait states before" in p for p in problems) >= count
