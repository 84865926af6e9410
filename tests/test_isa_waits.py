"""The wait states that hand-written memory statements have to bring themselves (hmoe.isa_check.check_waits): small
listings with a known answer, and the listings that the build saved."""
from __future__ import annotations

import re

import pytest

from hmoe import isa_check
from hmoe.build import CHECKED_SOURCES, CSRC, OBJ, _device_listing

HEAD, END = "k:\n", "\ts_endpgm\n"


def block(*lines):
    return "\t;;#ASMSTART\n" + "".join(f"\t{x}\n" for x in lines) + "\t;;#ASMEND\n"


def bad(text: str) -> int:
    return len(isa_check.check_waits(text))


LOADS = ["global_load_lds_dwordx4 v[2:3], off", "global_load_lds_dword v2, s[8:9]",
         "buffer_load_dwordx4 v4, s[0:3], 0 offen lds"]


@pytest.mark.parametrize("load", LOADS)
def test_m0(load):
    assert bad(HEAD + block("s_mov_b32 m0, s6", load) + END) == 1
    assert bad(HEAD + block("s_mov_b32 m0, s6", "s_nop 0", load) + END) == 0
    assert bad(HEAD + block("s_mov_b32 m0, s6", "s_add_u32 s10, s10, 64", load) + END) == 0
    # the compiler's own loads are the compiler's affair
    assert bad(HEAD + f"\ts_mov_b32 m0, s6\n\t{load}\n" + END) == 0


def test_scalar_register_of_a_vector_instruction():
    load = "buffer_load_dwordx4 v4, s[0:3], 0 offen lds"
    write = "\tv_readfirstlane_b32 s2, v9\n"

    def with_(states):
        return HEAD + write + states + block("s_mov_b32 m0, s6", "s_nop 0", load) + END
    # two of the five lie in the block
    assert bad(with_("")) == 1 and bad(with_("\ts_nop 1\n")) == 1 and bad(with_("\ts_nop 2\n")) == 0
    assert bad(with_("\tv_mov_b32_e32 v1, v2\n" * 3)) == 0
    # another register; a scalar instruction's write (the hardware waits for that itself)
    assert bad(with_("").replace("s2, v9", "s4, v9")) == 0
    assert bad(with_("").replace("v_readfirstlane_b32 s2, v9", "s_mov_b32 s2, s9")) == 0
    # a compare into a pair, a carry
    assert bad(with_("").replace("v_readfirstlane_b32 s2, v9", "v_cmp_gt_u32_e64 s[2:3], v1, v2")) == 1
    assert bad(with_("").replace("v_readfirstlane_b32 s2, v9", "v_add_co_u32_e64 v1, s[0:1], v1, v2")) == 1


def test_every_path_counts():
    load = block("s_mov_b32 m0, s6", "s_nop 0", "global_load_lds_dword v2, s[8:9]")
    write, nop = "\tv_readfirstlane_b32 s8, v9\n", "\ts_nop 4\n"
    # a branch around the wait, and a loop's back edge
    assert bad(HEAD + write + "\ts_cbranch_scc1 .LBB0_1\n" + nop + ".LBB0_1:\n" + load + END) == 1
    assert bad(HEAD + write + nop + "\ts_cbranch_scc1 .LBB0_1\n.LBB0_1:\n" + load + END) == 0
    assert bad(HEAD + ".LBB0_1:\n" + load + write + "\ts_cbranch_scc1 .LBB0_1\n" + END) == 1


def test_statements_wait():
    source = (CSRC / "hm_lds_dma.h").read_text()
    statements = re.findall(r'asm volatile\("(s_mov_b32 m0[^"]*)"', source)
    assert len(statements) == 5 and all("\\n\\ts_nop 0\\n" in s for s in statements)


@pytest.mark.parametrize("source", sorted(CHECKED_SOURCES))
def test_built_listings_wait(source):
    listing = _device_listing(OBJ / source.replace(".hip", ".o"))
    if not listing.exists():
        pytest.skip("no saved listing (library not built here)")
    text = listing.read_text()
    assert "lds" in text and isa_check.check_waits(text) == [] and isa_check.check_text(text) == []
