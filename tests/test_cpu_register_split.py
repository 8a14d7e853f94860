"""The register shares of the kernels whose warps deal them out (setmaxnreg), on the
host: a kernel compiled to fewer registers than its shares add up to would wait
without a limit, and is refused before its launch."""

import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "comfyui-int-crush_b200", "csrc")

PROGRAM = """
#include <cstdio>
#include "register_split.h"

int main() {
  const ic::RegisterSplit product = {128, 40, 256, 232}, attention = {256, 72, 256, 184};
  int bad = 0;
  for (int regs = 1; regs <= 255; ++regs) {
    // what a block of 384 or 512 threads is given, against what its warps take
    const int given = (regs + 7) / 8 * 8;
    bad += product.fits(regs) != (384 * given >= 128 * 40 + 256 * 232);
    bad += attention.fits(regs) != (512 * given >= 256 * 72 + 256 * 184);
  }
  bad += product.fits(160) || !product.fits(161) || !product.fits(168) || attention.fits(120) || !attention.fits(128);
  std::printf("%d\\n", bad);
  return bad != 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a host C++ compiler")
def test_what_fits(tmp_path):
    source, program = tmp_path / "split.cpp", tmp_path / "split"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", CSRC, "-o", program, source], check=True)
    assert subprocess.run([program], timeout=60).returncode == 0


def test_every_split_is_checked_before_the_launch():
    """No literal shares, and as many checks as kernels that deal registers out."""
    for name in sorted(os.listdir(CSRC)):
        with open(os.path.join(CSRC, name)) as f:
            text = f.read()
        uses = re.findall(r'asm volatile\("setmaxnreg\.(?:inc|dec)[^"]*"([^;]*);', text)
        assert all('"n"(' in u and "REGS." in u for u in uses), name
        assert text.count("split_fits_once(kern") == len(uses) // 2, name
