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


# --- values loaded from scratch memory ----------------------------------------------------

LOAD, USE = "\tscratch_load_dword v7, off, off offset:16\n", "\tv_add_u32_e32 v0, s4, v7\n"
THEN, END = "\ts_and_saveexec_b64 s[{0}:{1}], vcc\n\ts_cbranch_execz .LBB0_{0}\n", "\ts_or_b64 exec, exec, s[{0}:{1}]\n"


def _then(n):
    return THEN.format(n, n + 1)


def _end(n):
    return END.format(n, n + 1)


def _check(body):
    return isa_check.check_text("k:\n" + body + "\ts_endpgm\n.Lfunc_end0:\n")


def test_a_reload_between_the_ends_of_two_branches():
    """The inner end is gone: what is reloaded there reaches the inner branch's lanes alone."""
    bad = _then(4) + _then(6) + "\tv_mov_b32_e32 v1, 0\n.LBB0_6:\n" + LOAD + ".LBB0_4:\n" + _end(4) + USE
    good = _then(4) + _then(6) + "\tv_mov_b32_e32 v1, 0\n.LBB0_6:\n" + _end(6) + ".LBB0_4:\n" + _end(4) + LOAD + USE
    assert len(_check(bad)) == 1 and "reloaded" in _check(bad)[0]
    assert _check(good) == []


def test_reloads_used_in_their_own_lanes():
    inside = _then(4) + LOAD + USE + ".LBB0_4:\n" + _end(4)
    nested = _then(4) + LOAD + _then(6) + USE + ".LBB0_6:\n" + _end(6) + USE + ".LBB0_4:\n" + _end(4)
    again = _then(4) + LOAD + ".LBB0_4:\n" + _end(4) + "\tv_mov_b32_e32 v7, 0\n" + USE
    for code in (inside, nested, again, LOAD + _then(4) + ".LBB0_4:\n" + _end(4) + USE):
        assert _check(code) == []
    assert len(_check(_then(4) + LOAD + _then(6) + ".LBB0_6:\n" + _end(6) + ".LBB0_4:\n" + _end(4) + USE)) == 1


def test_reloads_and_an_other_side():
    """then / else by the lanes that are left over, and masks that were spilled to lanes of a register."""
    other = "\ts_xor_b64 s[4:5], exec, s[4:5]\n"
    code = LOAD + _then(4) + other + "\tv_mov_b32_e32 v1, 0\n.LBB0_4:\n\ts_andn2_saveexec_b64 s[4:5], s[4:5]\n" + USE + _end(4) + USE
    assert _check(code) == []
    spill = "\tv_writelane_b32 v9, s4, 2\n\tv_writelane_b32 v9, s5, 3\n\ts_mov_b64 s[4:5], 0\n"
    back = "\tv_readlane_b32 s4, v9, 2\n\tv_readlane_b32 s5, v9, 3\n"
    assert _check(LOAD + _then(4) + spill + back + _end(4) + ".LBB0_4:\n" + USE) == []
    assert len(_check(LOAD + _then(4) + spill + back.replace(" 3", " 5") + _end(4) + ".LBB0_4:\n" + USE)) == 1


def test_reloads_in_a_loop():
    """Lanes leave it one by one; all are on again behind it."""
    loop = "\ts_mov_b64 s[6:7], 0\n.LBB0_1:\n{0}\tv_cmp_eq_u32_e32 vcc, v1, v2\n\ts_or_b64 s[6:7], vcc, s[6:7]\n" \
           "\ts_andn2_b64 exec, exec, s[6:7]\n\ts_cbranch_execnz .LBB0_1\n" + _end(6)
    assert _check(LOAD + loop.format(USE) + USE) == []
    assert len(_check(loop.format(LOAD) + USE)) == 1  # the last turn's lanes alone have its value
    assert _check(loop.format(LOAD + USE)) == []


def test_accumulating_reads_its_own_register():
    reload_in = _then(4) + LOAD + ".LBB0_4:\n" + _end(4)
    assert len(_check(reload_in + "\tv_fmac_f32_e32 v7, v1, v2\n")) == 1
    assert _check(reload_in + "\tv_fma_f32 v7, v1, v2, v3\n") == []
