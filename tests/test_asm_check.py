"""The build's scan of inline-asm MFMAs (raftinfer_amd/asm_check.py) on small
listings whose answer is fixed by counting wait states, and on the built
prefill kernel itself."""
import pathlib

from raftinfer_amd import asm_check
from raftinfer_amd.asm_check import RESULT_WAIT_STATES, asm_mfma_hazards

MFMA = """\t;;#ASMSTART
\ts_nop 1
\tv_mfma_f32_32x32x16_bf16 a[16:31], v[30:33], v[6:9], a[16:31]
\t;;#ASMEND
"""


def test_copy_right_after_an_asm_mfma_is_flagged():
    text = MFMA + "\tv_accvgpr_mov_b32 a2, a17\n"
    hazards = asm_mfma_hazards(text)
    assert len(hazards) == 1 and "a[16:31]" in hazards[0] and "after 0 wait states" in hazards[0]


def test_reads_after_the_drain_or_of_other_registers_pass():
    drained = MFMA + "\ts_nop 7\n\ts_nop 7\n\ts_nop 3\n\tv_accvgpr_read_b32 v0, a16\n"
    assert asm_mfma_hazards(drained) == []
    other = MFMA + "\tv_accvgpr_read_b32 v0, a32\n\tv_accvgpr_mov_b32 a1, a15\n"
    assert asm_mfma_hazards(other) == []


def test_wait_states_are_counted_exactly():
    # s_nop n gives n + 1 wait states; one short of the latency is flagged, the latency is not
    short = MFMA + "\ts_nop 7\n" * 2 + f"\ts_nop {RESULT_WAIT_STATES - 16 - 2}\n" + "\tv_add_f32 v1, a20, v2\n"
    assert len(asm_mfma_hazards(short)) == 1
    enough = MFMA + "\ts_nop 7\n" * 2 + f"\ts_nop {RESULT_WAIT_STATES - 16 - 1}\n" + "\tv_add_f32 v1, a20, v2\n"
    assert asm_mfma_hazards(enough) == []


def test_compiler_mfmas_and_mfma_chains_are_not_flagged():
    # a compiler-placed MFMA (outside ASMSTART/ASMEND) is the compiler's own business, and an
    # accumulator chain is checked by the hardware
    text = "\tv_mfma_f32_32x32x16_bf16 a[0:15], v[4:7], v[8:11], 0\n\tv_accvgpr_read_b32 v0, a0\n"
    text += MFMA + MFMA
    assert asm_mfma_hazards(text) == []


def test_vector_results_operand_writes_and_owned_registers():
    mfma = MFMA.replace("\ts_nop 1\n", "").replace("a[16:31]", "v[40:55]")
    for line in ("\tv_mov_b32_e32 v1, v41\n", "\tv_mov_b32_e32 v55, v1\n", "\tds_write_b32 v1, v50\n"):
        assert len(asm_mfma_hazards(mfma + line)) == 1, line
        assert asm_mfma_hazards(mfma + "\ts_nop 7\n" * 3 + line) == [], line
    # an operand written by the vector unit right before, then two wait states before
    write = "\tv_add_f32_e32 v32, v1, v2\n"
    assert len(asm_mfma_hazards(write + "\ts_nop 0\n" + mfma)) == 1
    assert asm_mfma_hazards(write + "\ts_nop 1\n" + mfma) == []
    # ... also the accumulator that goes in, and both registers of a swap
    for line in ("\tv_accvgpr_write_b32 a20, v9\n", "\tv_permlane32_swap_b32_e32 v1, v31\n",
                 "\tv_permlane32_swap_b32_e32 v9, v1\n", "\tv_swap_b32 v1, v7\n"):
        agpr = MFMA.replace("\ts_nop 1\n", "")
        assert len(asm_mfma_hazards(line + agpr)) == 1, line
        assert asm_mfma_hazards(line + "\ts_nop 1\n" + agpr) == [], line
    for line in ("\tv_permlane32_swap_b32_e32 v1, v41\n", "\tv_permlane16_swap_b32_e32 v41, v1\n"):
        assert len(asm_mfma_hazards(mfma + line)) == 1, line
    # registers named in hexadecimal, and the rule for kernels that own the accumulation registers
    assert len(asm_mfma_hazards(MFMA.replace("a[16:31]", "a[0x80:0x8f]") + "\tv_accvgpr_read_b32 v0, a[0x81]\n")) == 1
    spill = "\tv_accvgpr_write_b32 a3, v9\n"
    assert asm_mfma_hazards(spill) == []
    assert len(asm_mfma_hazards(spill, owned_agprs=True)) == 1
    assert asm_mfma_hazards("\t;;#ASMSTART\n" + spill + "\t;;#ASMEND\n", owned_agprs=True) == []


def test_built_prefill_kernel_has_no_hazard():
    s = pathlib.Path(asm_check.__file__).resolve().parent / "_build" / "attention_prefill_mfma.hip.s"
    if not s.exists():
        import pytest
        pytest.skip("the library has not been built here")
    assert asm_mfma_hazards(s.read_text()) == []
    wide = s.with_name("attention_prefill_wide.hip.s")
    assert asm_mfma_hazards(wide.read_text(), owned_agprs=True) == []


def test_what_is_under_way_follows_branches():
    read = "\tv_add_f32 v1, a20, v2\n"
    gap = "\ts_nop 7\n" * 3
    # to a label further down, past code that falls out of the listing's order
    ahead = MFMA + "\ts_cbranch_scc1 .LBB0_2\n" + gap + "\ts_endpgm\n.LBB0_2:\n" + read
    assert len(asm_mfma_hazards(ahead)) == 1
    assert asm_mfma_hazards(ahead.replace(".LBB0_2:\n", ".LBB0_2:\n" + gap)) == []
    # back to a loop's head: the read stands in front of the MFMA
    loop = "\ts_nop 0\n.LBB0_1:\n" + read + MFMA + "\ts_cbranch_scc0 .LBB0_1\n\ts_endpgm\n"
    assert len(asm_mfma_hazards(loop)) == 1
    assert asm_mfma_hazards(loop.replace(MFMA, MFMA + gap)) == []
    # over two branches, whose own wait states count
    chain = MFMA + "\ts_branch .LBB0_4\n.LBB0_3:\n" + read + "\ts_endpgm\n.LBB0_4:\n\ts_branch .LBB0_3\n"
    hazards = asm_mfma_hazards(chain)
    assert len(hazards) == 1 and "after 2 wait states" in hazards[0]


def test_nothing_falls_through_an_unconditional_branch():
    read = "\tv_add_f32 v1, a20, v2\n"
    for end in ("\ts_branch .LBB0_9\n", "\ts_endpgm\n"):
        assert asm_mfma_hazards(MFMA + end + ".LBB0_1:\n" + read) == [], end
    # the longest wait of all ways into a label is the one that counts
    both = MFMA + "\ts_cbranch_scc1 .LBB0_1\n" + "\ts_nop 7\n" * 2 + ".LBB0_1:\n" + read
    hazards = asm_mfma_hazards(both)
    assert len(hazards) == 1 and "after 1 wait states" in hazards[0]


def test_built_paged_kernel_has_no_hazard():
    s = pathlib.Path(asm_check.__file__).resolve().parent / "_build" / "paged_prefill.hip.s"
    if not s.exists():
        import pytest
        pytest.skip("the library has not been built here")
    assert asm_mfma_hazards(s.read_text(), owned_agprs=True) == []


# ------------------------------------------ waits of loads through scalar registers

LOAD = "\tglobal_load_lds_dwordx4 v4, s[10:11] offset:1024\n"


def test_a_load_into_lds_waits_for_m0():
    from raftinfer_amd.asm_check import scalar_wait_hazards
    assert len(scalar_wait_hazards("\ts_mov_b32 m0, s5\n" + LOAD)) == 1
    assert len(scalar_wait_hazards("\ts_add_i32 m0, s5, 16\n\tbuffer_load_dword v1, s[4:7], 0 offen lds\n")) == 1
    assert scalar_wait_hazards("\ts_mov_b32 m0, s5\n\ts_nop 0\n" + LOAD) == []
    assert scalar_wait_hazards("\ts_mov_b32 m0, s5\n\tglobal_load_dwordx4 v[4:7], v4, s[10:11]\n" + LOAD) == []
    # over a branch, which is a wait state itself
    assert scalar_wait_hazards("\ts_mov_b32 m0, s5\n\ts_branch .L1\n\ts_nop 0\n.L1:\n" + LOAD) == []


def test_a_memory_instruction_waits_for_a_vector_write_of_its_scalars():
    from raftinfer_amd.asm_check import scalar_wait_hazards
    write = "\tv_readfirstlane_b32 s11, v2\n"
    assert len(scalar_wait_hazards(write + "\ts_nop 3\n" + LOAD)) == 1
    assert scalar_wait_hazards(write + "\ts_nop 4\n" + LOAD) == []
    assert scalar_wait_hazards(write.replace("s11", "s12") + LOAD) == []
    # a scalar instruction's own write has no such wait
    assert scalar_wait_hazards(write + "\ts_add_u32 s11, s11, s3\n" + LOAD) == []
    assert len(scalar_wait_hazards(write + "\ts_cmp_eq_u32 s11, s3\n" + LOAD)) == 1
    assert len(scalar_wait_hazards("\tv_cmp_gt_u32_e64 s[10:11], v1, v2\n" + LOAD)) == 1
    # back to a loop's head, and over two branches
    loop = ".L1:\n" + LOAD + "\ts_nop 7\n" + write + "\ts_cbranch_scc0 .L1\n\ts_endpgm\n"
    assert len(scalar_wait_hazards(loop)) == 1
    assert len(scalar_wait_hazards(write + "\ts_branch .L2\n.L3:\n" + LOAD + "\ts_endpgm\n.L2:\n\ts_branch .L3\n")) == 1
    assert scalar_wait_hazards(write + "\ts_endpgm\n.L2:\n" + LOAD) == []


def test_asm_loads_into_lds_have_their_waits():
    """In the sources: behind its write of M0 every asm load waits, and where the wait is too short for a base that a vector
    instruction may write, the build checks the assembly."""
    import re
    from raftinfer_amd.build import ASM_CHECKED
    sources = pathlib.Path(asm_check.__file__).resolve().parent / "csrc"
    found = 0
    for path in sorted(sources.iterdir()):
        text = path.read_text()
        for line in text.splitlines():
            if "s_mov_b32 m0" in line:
                found += 1
                assert re.search(r"s_mov_b32 m0, %0\\n\\ts_nop (\d|%3)\\n\\tglobal_load_lds", line), (path.name, line)
        if path.suffix == ".hip" and re.search(r"load_lds_b128<0>|load_lds_b128_at<|load_rows<", text):
            assert path.name in ASM_CHECKED, path.name
    assert found >= 5


def test_built_kernels_wait_for_their_scalars():
    from raftinfer_amd.asm_check import scalar_wait_hazards
    from raftinfer_amd.build import ASM_CHECKED
    folder = pathlib.Path(asm_check.__file__).resolve().parent / "_build"
    for name in ASM_CHECKED:
        s = folder / (name + ".s")
        if not s.exists():
            import pytest
            pytest.skip("the library has not been built here")
        assert scalar_wait_hazards(s.read_text()) == [], name
