"""isa_check over a function's control flow, on small listings."""

from gfx950_gluon_tutorials_amd import isa_check

MFMA = "\tv_mfma_f32_32x32x16_f16 a[0:15], v[0:3], v[4:7], a[0:15]\n"


def test_code_behind_an_early_end_is_scanned():
    """A kernel that returns early goes on behind its first s_endpgm."""
    early = "k:\n\ts_cbranch_scc1 .LBB0_2\n\ts_endpgm\n.LBB0_2:\n"
    bad = early + MFMA + "\tv_accvgpr_read_b32 v20, a15\n\ts_endpgm\n.Lfunc_end0:\n"
    good = early + MFMA + "\ts_nop 7\n\ts_nop 3\n\tv_accvgpr_read_b32 v20, a15\n\ts_endpgm\n.Lfunc_end0:\n"
    assert len(isa_check.check_text(bad)) == 1
    assert len(isa_check.check_text(good + bad.replace("k:", "j:"))) == 1
    assert isa_check.check_text(good) == []
    # What follows a function's end is no code of it.
    assert isa_check.check_text(good + "\t.section\t.rodata\n" + MFMA + "\tv_accvgpr_read_b32 v20, a15\n") == []
