"""How hmoe.isa_check cuts a listing into functions: a kernel may end in the middle of its listing, and what stands
behind that end is looked at too."""
from __future__ import annotations

from hmoe import isa_check

HEAD, END = "k:\n", "\ts_endpgm\n"
EARLY = HEAD + "\ts_cbranch_scc1 .LBB0_1\n" + END + ".LBB0_1:\n"
LOAD = "\tbuffer_load_dwordx4 v[4:7], v0, s[0:3], s4 offen\n"


def test_blocks_behind_an_end():
    assert isa_check.check_text(EARLY + END) == []
    assert isa_check.check_text(EARLY + "\ts_mov_b32 m0, -1\n" + END) != []
    assert isa_check.check_text(EARLY + LOAD + "\tv_mov_b32_e32 v20, v5\n\ts_waitcnt vmcnt(0)\n" + END) != []
    # a load before the end, its use behind it
    assert isa_check.check_text(HEAD + LOAD + "\ts_cbranch_scc1 .LBB0_1\n\ts_waitcnt vmcnt(0)\n" + END +
                                ".LBB0_1:\n\tv_mov_b32_e32 v20, v5\n\ts_waitcnt vmcnt(0)\n" + END) != []


def test_functions():
    text = EARLY + END + ".Lfunc_end0:\n\t.section .rodata\n\t.long 0\nk2:\n\ts_mov_b32 m0, -1\n" + END + ".Lfunc_end1:\n"
    assert [f[0] for f in isa_check._functions(text)] == ["k", "k2"]
    assert [len(f[1]) for f in isa_check._functions(text)] == [3, 2]
    assert [line.split(":")[0] for line in isa_check.check_text(text)] == ["k2"]
