"""The scan of isa_check for scalar registers that the vector unit wrote just
before a vector-memory instruction reads them, on small listings."""

import pytest

from gfx950_gluon_tutorials_amd import isa_check

DMA = "\tbuffer_load_dwordx4 v1, s[4:7], s9 offen lds\n"


def _fn(body: str) -> str:
    return "k:\n" + body + "\n\ts_endpgm\n"


@pytest.mark.parametrize("write", ["v_readfirstlane_b32 s6, v2", "v_readlane_b32 s9, v250, 3", "v_readfirstlane_b32 m0, v2",
                                   "v_cmp_eq_u32_e64 s[4:5], v1, v2"])
def test_a_descriptor_offset_or_m0_needs_five_wait_states(write):
    assert len(isa_check.check_text(_fn(f"\t{write}\n\ts_nop 3\n" + DMA))) == 1
    assert isa_check.check_text(_fn(f"\t{write}\n\ts_nop 4\n" + DMA)) == []


def test_other_registers_and_scalar_writes_need_none():
    assert isa_check.check_text(_fn("\tv_readfirstlane_b32 s20, v2\n" + DMA)) == []
    assert isa_check.check_text(_fn("\ts_mov_b32 s6, s3\n\ts_mov_b32 m0, s2\n" + DMA)) == []
    assert isa_check.check_text(_fn("\tv_readfirstlane_b32 s6, v2\n\ts_mov_b32 s6, s3\n" + DMA)) == []


def test_across_a_back_edge():
    loop = ".LBB0_1:\n" + DMA + "\ts_nop 4\n\tv_readfirstlane_b32 s6, v2\n\ts_cbranch_scc1 .LBB0_1\n"
    assert len(isa_check.check_text(_fn(loop))) == 1


@pytest.mark.parametrize("reader", ["s_cmp_eq_u32 s6, 0", "s_cmp_lg_u64 s[6:7], 0", "s_cmpk_lt_u32 s6, 0x10", "s_bitcmp1_b32 s6, 3",
                                    "s_cmov_b32 s6, s3", "s_setreg_b32 hwreg(HW_REG_MODE, 0, 4), s6"])
def test_scalar_instructions_that_only_read_or_may_not_write_keep_the_record(reader):
    code = f"\tv_readfirstlane_b32 s6, v2\n\t{reader}\n"
    assert len(isa_check.check_text(_fn(code + DMA))) == 1
    assert isa_check.check_text(_fn(code + "\ts_nop 3\n" + DMA)) == []


def test_m0_compared_with_a_number():
    assert len(isa_check.check_text(_fn("\tv_readfirstlane_b32 m0, v2\n\ts_cmp_lt_i32 m0, 5\n" + DMA))) == 1


@pytest.mark.parametrize("write", ["v_add_co_u32_e64 v3, s[6:7], v2, v4", "v_subrev_co_u32_e64 v3, s[6:7], v2, v4",
                                   "v_addc_co_u32_e64 v3, s[4:5], v2, v4, s[20:21]", "v_div_scale_f32 v3, s[6:7], v2, v4, v2",
                                   "v_mad_u64_u32 v[10:11], s[6:7], v2, v4, 0", "v_mad_i64_i32 v[10:11], s[4:5], v2, v4, v[8:9]"])
def test_scalar_results_in_the_second_operand(write):
    assert len(isa_check.check_text(_fn(f"\t{write}\n\ts_nop 3\n" + DMA))) == 1
    assert isa_check.check_text(_fn(f"\t{write}\n\ts_nop 4\n" + DMA)) == []


@pytest.mark.parametrize("read", ["v_add_u32_e32 v3, s6, v2", "v_fma_f32 v3, s6, v2, v4", "v_cndmask_b32_e64 v3, v2, v4, s[6:7]",
                                  "v_addc_co_u32_e64 v3, s[20:21], v2, v4, s[6:7]", "v_writelane_b32 v3, s6, 5"])
def test_scalar_operands_that_are_read_are_no_results(read):
    assert isa_check.check_text(_fn(f"\t{read}\n" + DMA)) == []
