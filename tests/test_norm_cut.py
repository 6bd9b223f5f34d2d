"""How tsn_gate_add_norm cuts its rows into a launch (gate_norm_cut), on the host."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "thinksound-native_amd")


@pytest.fixture(scope="module")
def cut(tsn, tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("cut") / "norm_cut")
    subprocess.run(["/opt/rocm/bin/hipcc", "--offload-arch=gfx950", "-std=c++17", "-O1", "-Xclang", "-target-feature",
                    "-Xclang", "-packed-fp32-ops", "-x", "hip", os.path.join(ROOT, "tests", "norm_cut.cpp"),
                    "-I" + os.path.join(PKG, "csrc"), "-I" + os.path.join(ROOT, "include"), "-o", exe,
                    "-L" + os.path.join(PKG, "lib"), "-ltsn", "-Wl,-rpath," + os.path.join(PKG, "lib")],
                   check=True, capture_output=True, text=True)

    def ask(asked):
        r = subprocess.run([exe], input="".join("%d %d %d %d\n" % a for a in asked), capture_output=True, text=True, check=True)
        return [tuple(map(int, line.split())) for line in r.stdout.split("\n") if line]
    return ask


def test_launches_stay_below_2_32_threads(cut):
    """every row is taken, and no number of rows below 2^31 makes a launch of 2^32 threads or more"""
    near = [n + d for k in range(1, 9) for n in (k << 20, k << 21, k << 22, k << 23, k << 24, k << 27) for d in range(-9, 10)]
    rows = sorted({1, 2, 63, 64, 6352, 32771, *(n for n in near if n < 1 << 31), *((1 << 31) - d for d in range(1, 520))})
    asked = [(n, m, w, c) for n in rows for m in (1, 7, n) for w, c in ((1, 1), (2, 1), (4, 1), (8, 1), (8, 2), (16, 1))]
    got = cut(asked)
    assert len(got) == len(asked)
    for (n, m, w, c), (per, grid, block) in zip(asked, got):
        assert block == (64 * w if w > 1 else 256)
        assert 0 < grid * block < 1 << 32, (n, m, w, c, per, grid)
        groups = grid * (1 if w > 1 else 4)
        assert groups * per >= n and (groups - (1 if w > 1 else 4)) * per < n, (n, m, w, c, per, grid)


def test_rows_in_turn(cut):
    """a row a group where each has its own modulation, otherwise as many as fill the device once, 32 at most"""
    assert cut([(6352, 397, 2, 1), (6352, 1, 2, 1), (32771, 1, 4, 1), (32771, 5, 4, 1), (1, 1, 16, 1), (6352, 397, 8, 2)]) == \
        [(4, 1588, 128), (1, 6352, 128), (1, 32771, 256), (32, 1025, 256), (1, 1, 1024), (25, 255, 512)]
