"""How group norm cuts its work (vtl_b200/csrc/groupnorm_plan.h), for many sizes, without a GPU: every position and channel
belongs to one CTA, and what a CTA takes fits its threads, its shared memory and the limits of a TMA box."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r'''
#include <cstdio>
#include <cstdlib>
#include "groupnorm_plan.h"
#define CHECK(x) if (!(x)) { std::printf("%s: B=%d S=%d width=%d G=%d aligned=%d bwd=%d\n", #x, B, S, width, G, aligned, bwd); std::exit(1); }
int main() {
  long plans = 0, on_chip = 0;
  const int Bs[] = {1, 7, 300}, Ss[] = {1, 2, 17, 64, 255, 257, 1000, 1024, 4095, 4096, 20000, 1000000};
  const int widths[] = {1, 2, 3, 4, 5, 8, 11, 16, 18, 31, 32, 48, 64, 100, 127, 128, 515, 1030, 2048, 4096, 5000, 8192, 40000};
  const int Gs[] = {1, 2, 3, 4, 8, 11, 30, 32, 64};
  for (int B : Bs) for (int S : Ss) for (int width : widths) for (int G : Gs) for (int aligned = 0; aligned < 2; ++aligned)
    for (int bwd = 0; bwd < 2; ++bwd) {
      const int C = width * G, threads = bwd ? kGnBwdThreads : kGnFwdThreads, middle = 4, most = bwd ? 8 : 16;
      const GnPlan p = gn_plan(B, S, C, G, aligned, threads, middle, most, 148);
      ++plans;
      CHECK(p.vec == (aligned && C % 4 == 0 ? 4 : 1));
      if (!p.on_chip) continue;
      ++on_chip;
      CHECK(p.groups >= 1 && p.groups <= G && p.groups <= kGnMaxGroups);
      CHECK((long long)(p.slabs - 1) * p.groups < G && (long long)p.slabs * p.groups >= G);
      CHECK(p.csplit * p.rsplit <= kGnMaxCluster);
      CHECK(p.vpt == 1 || p.vpt == middle || p.vpt == most);
      for (int slab = 0; slab < p.slabs; slab += p.slabs > 1 ? p.slabs - 1 : 1) {  // the first and the last
        const int groups = p.groups < G - slab * p.groups ? p.groups : G - slab * p.groups, channels = groups * width;
        CHECK(slab == 0 || p.csplit == 1 || groups == p.groups);
        CHECK((slab * p.groups * width) % p.vec == 0);
        int covered = 0;
        for (int c = 0; c < p.csplit; ++c) {
          const int first = c * p.channels, n = p.channels < channels - first ? p.channels : channels - first;
          CHECK(n > 0 && n % p.vec == 0 && first % p.vec == 0);
          covered += n;
          const int cols = n / p.vec, lanes = threads / gn_pow2(cols);
          CHECK(gn_pow2(cols) <= threads && lanes >= 1);
          long long rows = 0;
          for (int r = 0; r < p.rsplit; ++r) {
            const int r0 = (long long)r * p.rows < S ? r * p.rows : S, r1 = r0 + p.rows < S ? r0 + p.rows : S;
            rows += r1 - r0;
            CHECK(r1 - r0 <= lanes * p.vpt);
          }
          CHECK(rows == S);
        }
        CHECK(covered == channels);
        if (slab == p.slabs - 1) break;
      }
      if (p.tma) {
        CHECK(p.channels <= 256 && p.channels * 4 % 16 == 0 && p.box_rows <= 256 && p.box_rows % 8 == 0);
        CHECK(p.boxes * p.box_rows >= p.rows);
        CHECK((long long)p.boxes * p.box_rows * p.channels * 4 * (bwd ? 2 : 1) <= kGnMaxSmem);
      } else {
        CHECK((long long)threads * p.vpt * p.vec * 4 * (bwd ? 2 : 1) <= kGnMaxSmem);
      }
    }
  std::printf("%ld plans, %ld on chip\n", plans, on_chip);
  return on_chip > plans / 4 ? 0 : 1;
}
'''


def test_every_element_belongs_to_one_cta(tmp_path):
    src, exe = tmp_path / "plan.cpp", tmp_path / "plan"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-Wall", "-Werror", "-I",
                    os.path.join(ROOT, "vtl_b200", "csrc"), "-o", str(exe), str(src)], check=True)
    p = subprocess.run([str(exe)], capture_output=True, text=True)
    assert p.returncode == 0, p.stdout + p.stderr
