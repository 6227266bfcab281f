"""The rows that the attention kernels take for a sequence and the order of a batch's blocks (qengine_amd/csrc/seq_rows.hpp),
compiled by g++ with overflow as an error, against Python's whole numbers. CPU only."""
import itertools
import os
import random
import re
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "qengine_amd", "csrc")
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")


@pytest.fixture(scope="module")
def rows(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("rows") / "seq_rows_host")
    subprocess.run(["g++", "-std=c++17", "-O1", "-ftrapv", "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(ROCM, "include"),
                    os.path.join(HERE, "seq_rows_host.cpp"), "-o", exe], check=True)

    def run(lines):
        r = subprocess.run([exe], input="\n".join(lines) + "\n", capture_output=True, text=True, timeout=60)
        assert r.returncode == 0, r.stderr
        return [None if x == "none" else tuple(map(int, x.split())) for x in r.stdout.splitlines()]
    return run


LOW, HIGH = -2 ** 31, 2 ** 31 - 1


def test_rows_stay_inside(rows):
    ends = [LOW, LOW + 1, LOW + 64, -2 ** 30, -1, 0, 1, 63, 64, 1000, 2 ** 30, HIGH - 1, HIGH]
    cases = [(a, b, t) for a, b in itertools.product(ends, ends) for t in (0, 1, 64, 1000, 2 ** 30, HIGH)]
    for (a, b, t), (first, n) in zip(cases, rows(["rows %d %d %d" % x for x in cases])):
        lo, hi = min(max(a, 0), t), min(max(b, 0), t)
        assert (first, n) == (lo, max(0, hi - lo)), (a, b, t)


def test_kernels_subtract_no_starts_of_their_own():
    """the attention kernels take lengths from rows_of alone"""
    for f in ("attn_prompt.hip", "attn_tree.hip", "attn_tree.hpp", "attn_wide.hip"):
        txt = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, f)).read())
        for m in re.finditer(r"\bcu\[", txt):
            line = txt[txt.rfind("\n", 0, m.start()) + 1:txt.find("\n", m.start())]
            assert "rows_of(a.cu[" in line, (f, line)


@pytest.mark.parametrize("n", [1, 2, 5, 64, 65, 300])
def test_every_block_has_its_place(rows, n):
    rng = random.Random(n)
    blocks = [rng.choice([0, 0, 1, 2, 3, 17, 40]) for _ in range(n)]
    text = "%d %s" % (n, " ".join(map(str, blocks)))
    got = rows(["place %d %s" % (i, text) for i in range(sum(blocks) + 3)])
    want = [(level, r) for level in range(40, -1, -1) for r in range(sum(b > level for b in blocks))]
    assert got == want + [None] * 3


@pytest.mark.parametrize("n,most", [(4096, 2 ** 24), (4096, 2 ** 23 + 5), (65, 2 ** 24), (700, 2 ** 20)])
def test_starts_that_do_not_ascend_end_the_search(rows, n, most):
    """sequences that overlap, so that their blocks sum past 2^31: every block of the grid finds one that exists, or none"""
    rng = random.Random(most)
    blocks = [rng.choice([0, most, most, most - 1, rng.randrange(most)]) for _ in range(n)]
    text = "%d %s" % (n, " ".join(map(str, blocks)))
    slots = [0, 1, 5, n, 12345, 2 ** 20, 2 ** 24, 2 ** 24 + 4095]
    for slot, at in zip(slots, rows(["place %d %s" % (i, text) for i in slots])):
        level, rank = at
        assert 0 <= rank < sum(b > level for b in blocks), (slot, at)
