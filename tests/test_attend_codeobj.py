"""CPU suite: what the compiler cannot see of the attention kernels' inline asm, on the disassembly of the built library."""
import codeobj


def _listing(texts):
    return ["%s   // %012X: 00000000" % (t, 0x1000 + 4 * i) for i, t in enumerate(texts)]


def test_fetches_have_their_wait_states(gpx, tmp_path):
    codeobj.guard_asm_fetches(gpx.LIB_PATH, tmp_path)


def test_guard_sees_a_missing_wait():
    load = "buffer_load_dwordx4 v5, s[4:7], 0 offen lds"
    for write in ("v_readfirstlane_b32 s6, v1", "v_cmp_eq_u32_e64 s[6:7], 0, v1", "v_add_co_u32 v1, s[4:5], v1, v2"):
        assert codeobj.scalar_hazard_violations(_listing([write, "s_mov_b32 m0, s9", "s_nop 0", load, "s_endpgm"]))
        assert codeobj.scalar_hazard_violations(_listing([write, "s_nop 3", load, "s_endpgm"]))
        assert not codeobj.scalar_hazard_violations(_listing([write, "s_nop 4", load, "s_endpgm"]))
    assert not codeobj.scalar_hazard_violations(_listing(["v_readfirstlane_b32 s8, v1", load, "s_endpgm"]))
    # along the short of two paths
    rows = _listing(["v_readfirstlane_b32 s6, v1", "s_cbranch_scc0 2", "s_nop 7", load, "s_endpgm"])
    rows[1] += " <kernel+0xC>"
    assert codeobj.scalar_hazard_violations(rows)
