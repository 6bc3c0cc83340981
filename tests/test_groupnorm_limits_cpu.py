"""The largest sizes that group norm takes: its plan (vtl_b200/csrc/groupnorm_plan.h) counts them without overflow."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdio>
#include "groupnorm_plan.h"
int main() {
  const int C = kGnMaxChannels, Gs[] = {1, 2, 3, 1 << 20, C};
  for (int d = 0; d < 8; ++d)
    for (int G : Gs)
      for (int S = 1; S <= 2; ++S)
        for (int bwd = 0; bwd < 2; ++bwd) {
          const int c = G == C ? C : (C - d) / G * G;
          const GnPlan p = gn_plan(1, S, c, G, true, bwd ? kGnBwdThreads : kGnFwdThreads, 4, bwd ? 8 : 16, 148);
          if (p.on_chip && c / G > 8 * 512 * 4) return std::printf("a group of %d channels in a cluster\n", c / G), 1;
          // what the kernels for groups of any size round up
          if (c + 1023 < 0 || (c + 7) / 8 <= 0 || (c + 1023) / 1024 * 1024 - 1 < 0) return 1;
        }
  return C > 2000000000 ? 0 : 1;
}
"""


def test_plans_of_the_most_channels(tmp_path):
    src, exe = tmp_path / "limits.cpp", tmp_path / "limits"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-Wall", "-Werror", "-I",
                    os.path.join(ROOT, "vtl_b200", "csrc"), "-o", str(exe), str(src)], check=True)
    p = subprocess.run([str(exe)], capture_output=True, text=True)
    assert p.returncode == 0, p.stdout + p.stderr
