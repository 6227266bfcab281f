"""Which kernel a grouped 8-bit product takes (qengine_amd/csrc/f8_choice.hpp), compiled by g++. CPU only."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CUS = 256


@pytest.fixture(scope="module")
def choose(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("choice") / "f8_choice_host")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", os.path.join(HERE, "f8_choice_host.cpp"), "-o", exe], check=True)

    def run(calls):
        text = "".join("%d %d %d %d %d %d\n" % c for c in calls)
        r = subprocess.run([exe], input=text, capture_output=True, text=True, timeout=60, check=True)
        return [int(v) for v in r.stdout.split()]
    return run


# experts, rows, n, k, and us by blocks of 64, 128 and 256 rows on an MI355X (ragged segments, rows by index)
MEASURED = [
    (8, 256, 256, 4096, 14.5, 29.9, 47.0),
    (8, 256, 512, 4096, 14.5, 30.0, 47.0),
    (8, 256, 1024, 4096, 15.0, 30.2, 47.8),
    (8, 256, 2048, 4096, 16.0, 30.9, 47.6),
    (8, 1024, 256, 4096, 14.8, 30.8, 48.8),
    (8, 1024, 512, 4096, 15.8, 31.2, 49.0),
    (8, 1024, 1024, 4096, 16.8, 32.3, 50.2),
    (8, 1024, 2048, 4096, 29.7, 33.5, 50.8),
    (8, 2048, 256, 4096, 15.5, 31.1, 49.4),
    (8, 2048, 512, 4096, 16.3, 32.2, 49.7),
    (8, 2048, 1024, 4096, 23.8, 32.7, 50.8),
    (8, 2048, 2048, 4096, 40.9, 40.3, 51.6),
    (8, 4096, 256, 4096, 15.7, 31.5, 50.9),
    (8, 4096, 512, 4096, 24.0, 33.1, 51.2),
    (8, 4096, 1024, 4096, 37.3, 40.0, 51.6),
    (8, 4096, 2048, 4096, 63.0, 69.2, 55.1),
    (8, 8192, 256, 4096, 24.8, 32.3, 50.6),
    (8, 8192, 512, 4096, 36.8, 39.5, 51.8),
    (8, 8192, 1024, 4096, 58.9, 68.9, 54.2),
    (8, 8192, 2048, 4096, 114.2, 112.6, 110.1),
    (8, 20000, 256, 4096, 40.1, 40.0, 51.5),
    (8, 20000, 512, 4096, 66.5, 70.5, 55.7),
    (8, 20000, 1024, 4096, 129.3, 136.4, 111.2),
    (8, 20000, 2048, 4096, 276.8, 250.4, 177.4),
    (32, 1024, 256, 2048, 9.8, 17.6, 27.2),
    (32, 1024, 1024, 2048, 14.9, 19.5, 29.2),
    (32, 1024, 2048, 2048, 24.6, 27.7, 37.0),
    (32, 4096, 256, 2048, 10.3, 18.7, 29.4),
    (32, 4096, 1024, 2048, 26.1, 25.1, 33.0),
    (32, 4096, 2048, 2048, 48.0, 49.9, 40.8),
    (32, 8192, 256, 2048, 16.0, 20.7, 31.7),
    (32, 8192, 1024, 2048, 37.5, 40.2, 34.9),
    (32, 8192, 2048, 2048, 79.4, 72.8, 70.6),
    (32, 20000, 256, 2048, 26.0, 25.3, 32.7),
    (32, 20000, 1024, 2048, 71.4, 77.8, 66.6),
    (32, 20000, 2048, 2048, 173.1, 159.1, 117.2),
    (60, 1024, 256, 2048, 10.5, 18.2, 27.6),
    (60, 1024, 1024, 2048, 24.0, 25.9, 35.5),
    (60, 1024, 2048, 2048, 50.3, 67.1, 72.5),
    (60, 8192, 256, 2048, 17.1, 20.5, 31.0),
    (60, 8192, 1024, 2048, 44.5, 48.1, 39.5),
    (60, 8192, 2048, 2048, 93.4, 97.5, 83.2),
    (60, 20000, 256, 2048, 27.4, 26.2, 33.6),
    (60, 20000, 1024, 2048, 87.0, 89.8, 73.4),
    (60, 20000, 2048, 2048, 185.5, 172.9, 144.7),
    (512, 4096, 1024, 2048, 183.3, 235.1, 280.9),
    (512, 20480, 1024, 2048, 214.7, 253.1, 292.1),
    (512, 40960, 1024, 2048, 270.6, 285.0, 324.5),
    (512, 81920, 1024, 2048, 423.0, 418.4, 366.4),
    (512, 40960, 2048, 512, 229.2, 220.6, 252.6),
    (128, 40000, 2048, 768, 198.2, 177.2, 150.8),
    (1, 4096, 4096, 4096, 150.6, 108.2, 66.6),
    (8, 32768, 4096, 4096, 1208.3, 831.5, 576.7),
    (60, 20000, 2816, 2048, 265.4, 243.8, 194.3),
]


def test_within_ten_per_cent_of_the_fastest(choose):
    got = choose([(r, n, k, e, CUS, 1) for e, r, n, k, *_ in MEASURED])
    slow = []
    for (e, r, n, k, *us), bt in zip(MEASURED, got):
        if us[(64, 128, 256).index(bt)] > 1.1 * min(us):
            slow.append((e, r, n, k, bt, us))
    assert not slow, slow


def test_rounds_of_an_xcd(choose):
    """blocks go to the XCDs in whole rows: tiles of 256 x 256 that are one round of the card may be two of an XCD (us measured by 64,
    128 and 256 rows: 20.1 / 23.8 / 29.1 and 45.6 / 43.6 / 60.2)"""
    assert choose([(1662, 5376, 288, 8, CUS, 1), (1171, 5984, 1904, 8, CUS, 1)]) in ([64, 64], [64, 128])


def test_few_rows_an_expert(choose):
    assert choose([(7, 1024, 2048, 1, CUS, 1), (4095, 1024, 2048, 512, CUS, 1), (1, 16, 16, 1024, CUS, 1)]) == [16] * 3


def test_no_large_blocks_where_offsets_do_not_fit(choose):
    calls = [(r, n, 4096, e, CUS, 0) for r in (4096, 1 << 20, 1 << 24) for n in (256, 1024) for e in (1, 8, 1024)]
    assert 256 not in choose(calls)
    assert choose([(1 << 20, 4096, 4096, 8, CUS, 1), (1 << 20, 4096, 4096, 8, CUS, 0)])[0] == 256


@pytest.mark.parametrize("cus", [32, 64, 256, 304])
def test_large_blocks_fill_the_card(choose, cus):
    """blocks that leave most CUs without work are not taken while smaller ones would give it to them"""
    calls = [(r, n, 4096, e, cus, 1) for e in (1, 2, 8, 30) for r in (240, 500, 1000, 2000, 4000) for n in (64, 200, 256, 512, 1000)]
    for (r, n, _, e, _, _), bt in zip(calls, choose(calls)):
        blocks = (r // 256 + min(r, e)) * -(-n // 256)
        small = max(r / 64, e) * -(-n // 128)
        assert bt != 256 or blocks * 4 > cus or small > 3 * cus, (r, n, e, bt)
