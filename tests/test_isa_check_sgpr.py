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
