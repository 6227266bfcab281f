"""Wait states of the LDS DMAs that take their address from a scalar base (CPU only, reads qengine_amd/csrc).

A vector memory instruction may read a scalar register that a vector instruction wrote five wait states before at the earliest
(GFX9). The compiler keeps to that for instructions of its own, but does not look into inline asm: a base that it reloads from
a spill (v_readlane) right before the statement would be read too early. So the statement itself waits: the scalar write of m0
and s_nop 4 make six.
"""
import re

from test_source_rules import asm_statements


def test_scalar_bases_are_waited_for():
    found = 0
    for f, body in asm_statements():
        lines = [x.strip() for x in body.split("\n") if x.strip()]
        for i, x in enumerate(lines):
            if x.startswith("global_load_lds") and not x.endswith("off"):
                found += 1
                nops = sum(int(m.group(1)) + 1 for m in (re.match(r"s_nop (\d+)$", y) for y in lines[:i]) if m)
                assert nops >= 5, (f, body)
    assert found
