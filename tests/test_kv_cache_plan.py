"""CPU test of how the work of attention over a paged cache is dealt out (the library's own function, compiled for the host)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PLAN = r"""
#include "kv_plan.hpp"
#include <cassert>
#include <cstdio>
using namespace cuvs_b200::kv;
int main()
{
  // 148 SMs that hold 74, 33 and 15 clusters of 2, 4 and 8 blocks, as one B200 does, and others that they may hold
  const uint32_t machines[][4] = {{148, 74, 33, 15}, {148, 74, 36, 16}, {148, 70, 30, 8}, {148, 74, 37, 18}, {148, 0, 0, 0}};
  for (const auto& holds : machines) {
    for (uint64_t units = 1; units <= 2000; units++) {
      for (uint64_t most : {uint64_t(0), uint64_t(1), uint64_t(100), uint64_t(1500), uint64_t(3000), uint64_t(6144), uint64_t(20000), uint64_t(1) << 40}) {
        for (int i = 0; i < 4; i++) {
          plan p{};
          p.rows     = 8;
          p.chunk    = 16;
          p.resident = 3;
          p.large    = i & 1 ? 12 : 0;
          const bool shares = i & 2;
          deal_out(148, holds, p, units, most, shares);
          const uint64_t chunks = (most + p.chunk - 1) / p.chunk;
          assert(p.blocks >= 1);
          if (p.cluster == 0) {
            assert(shares && p.warps == uint32_t(kSmall) && p.blocks <= 148 * 3 && p.parts == (chunks > 1));
          } else {
            assert(p.blocks == units * p.cluster && !p.parts && (!shares || units <= 148));
            // all clusters at once, and no larger than there is work for
            if (p.cluster > 1) { assert(units <= holds[p.cluster == 8 ? 3 : p.cluster == 4 ? 2 : 1] && (p.cluster / 2) * p.warps < chunks); }
            if (shares) { assert((chunks + p.warps - 1) / p.warps <= 4 * p.cluster); }
          }
        }
      }
    }
  }
  auto cluster = [&](uint64_t units, uint64_t most) {
    plan p{};
    p.rows = 8, p.chunk = 16, p.resident = 3, p.large = 12;
    deal_out(148, machines[0], p, units, most, true);
    return p.cluster;
  };
  assert(cluster(8, 6144) == 8 && cluster(15, 3000) == 8);
  assert(cluster(16, 3000) == 4 && cluster(16, 6144) == 0);    // sixteen clusters of eight would be two waves
  assert(cluster(33, 1500) == 4 && cluster(34, 1500) == 2);    // and so would 34 of four
  assert(cluster(8, 8192) == 0 && cluster(148, 700) == 1);
  std::puts("ok");
}
"""


def test_clusters_are_as_many_as_the_gpu_holds(tmp_path):
    src, exe = tmp_path / "plan.cpp", tmp_path / "plan"
    src.write_text(PLAN)
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "cuvs_b200", "csrc"), "-I",
                    "/usr/local/cuda/include", str(src), "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout == "ok\n"
