"""Which kernel the 8-bit linear layer takes (csrc/linear_i8_rule.h, compiled as plain host code; no GPU): every tile has sizes
in the GPU tests that the rule sends to it, so that a threshold that moves cannot take a tile out of them unseen."""
import os
import subprocess

from linear_i8_tiles import TILES

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _rule(tmp_path, sizes):
    exe = str(tmp_path / "linear_i8_rule")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-I", os.path.join(REPO, "synerfgine_amd", "csrc"),
                    os.path.join(REPO, "tests", "native", "linear_i8_rule.cpp"), "-o", exe], check=True, capture_output=True)
    out = subprocess.run([exe], input="".join("%d %d %d %d\n" % s for s in sizes), capture_output=True, text=True, check=True, timeout=60)
    return out.stdout.split()


def test_every_tile_is_run(tmp_path):
    assert _rule(tmp_path, [t[1:] for t in TILES]) == [t[0] for t in TILES]
    for by_expert in (False, True):
        assert {t[0] for t in TILES if bool(t[4]) == by_expert} == {"64x64", "64x128", "128x128", "256x256"}


def test_the_other_kernels(tmp_path):
    sizes = [(1 << 20, 64, 64, 0), (100, 256, 4096, 0), (100000, 256, 4096, 0), (1, 4096, 4096, 0), (17, 4096, 4096, 0), (33, 4096, 1024, 0), (192, 1024, 2048, 16),
             (193, 1024, 2048, 16)]
    assert _rule(tmp_path, sizes) == ["rows", "rows", "256x256", "few", "split", "split", "few", "128x128"]
