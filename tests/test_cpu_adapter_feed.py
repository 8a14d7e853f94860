"""The producer of the streamed adapter kernels, run on the host against every
wait giving up: whatever happens, each copy that it issued has landed when it
returns (a CTA must not leave while a copy may still write to its shared
memory), and it waits for no copy that was not issued."""

import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "comfyui-int-crush_b200", "csrc")

PROGRAM = r"""
#include <cstdio>
#include <vector>
#include "lora_feed.h"

// The copies of one ring.  A stage that is free again had its copy read, so
// that copy had landed.
struct Ring {
  int stages, issued = 0;
  std::vector<bool> landed;
  bool take(int q) {
    if (q != issued) return false;
    if (q >= stages) landed[q - stages] = true;
    return true;
  }
  void load(int) { ++issued; landed.push_back(false); }
  bool wait(int q) {
    if (q < 0 || q >= issued) return false;
    landed[q] = true;
    return true;
  }
  bool all() const {
    for (bool l : landed) if (!l) return false;
    return true;
  }
};

template <int SA, int SB>
int cases() {
  int bad = 0;
  for (int blocks = 0; blocks <= 2 * SA + 3; ++blocks)
    for (int passes = 0; passes <= 3; ++passes)
      for (int stop = 0; stop <= blocks * (passes + 1) + 1; ++stop) {   // the wait that gives up
        Ring a{SA}, b{SB};
        int waits = 0;
        bool right = true;
        std::vector<int> block_of, pass_of;
        ic::lora_feed<SA, SB>(
            blocks, passes, [&](int q) { if (waits++ == stop) return false; right &= a.take(q); return true; },
            [&](int q) { a.load(q); }, [&](int q) { right &= a.wait(q); },
            [&](int q) { if (waits++ == stop) return false; right &= b.take(q); return true; },
            [&](int q, int i, int p) { b.load(q); block_of.push_back(i); pass_of.push_back(p); },
            [&](int q) { right &= b.wait(q); });
        for (int q = 0; q < b.issued; ++q) right &= block_of[q] == q / passes && pass_of[q] == q % passes;
        const bool finished = stop >= blocks * (passes + 1);
        if (finished) right &= a.issued == blocks && b.issued == blocks * passes;
        if (!right || !a.all() || !b.all()) {
          ++bad;
          std::printf("stages %d %d, %d blocks, %d passes, wait %d\n", SA, SB, blocks, passes, stop);
        }
      }
  return bad;
}

int main() { return cases<4, 6>() + cases<5, 4>() + cases<4, 4>() + cases<1, 1>() ? 1 : 0; }
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a host C++ compiler")
def test_every_copy_lands_before_the_feed_returns(tmp_path):
    source, program = tmp_path / "feed.cpp", tmp_path / "feed"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", CSRC, "-o", program, source], check=True)
    run = subprocess.run([program], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0, run.stdout[:2000]
