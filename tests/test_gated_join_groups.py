"""CPU: the grids of the kernels that add parts of c, over all that a gated layer may have of rows and outputs: more results than 32 bits count."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PROBE = """
#include <cstdio>
#include "dc_linear_route.hpp"
int main() {
  long m, n;
  while (std::scanf("%ld %ld", &m, &n) == 2) {
    const int rows = (int)m, outputs = (int)n;  // (as the argument blocks of the kernels hold them)
    std::printf("%ld\\n", (long)dc::linear_join_groups(rows, outputs));
  }
}
"""


def test_a_workgroup_for_each_256_lanes_up_to_the_most(tmp_path):
    (tmp_path / "probe.cpp").write_text(PROBE)
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(ROOT, "dotcompute_amd", "csrc"),
                    str(tmp_path / "probe.cpp"), "-o", str(tmp_path / "probe")], check=True)
    shapes = [(m, n) for m in (1, 3, 255, 256, 257, 1 << 16, (1 << 20) + 7, 1 << 28, (1 << 30) - 1)
              for n in (1, 8, 9, 16, 17, 4096, 1 << 14, (1 << 22) - 1, 1 << 22)]
    got = subprocess.run([str(tmp_path / "probe")], input="".join(f"{m} {n}\n" for m, n in shapes), capture_output=True, text=True,
                         check=True).stdout.split()
    assert [int(v) for v in got] == [min(-(-m * -(-n // 8) // 256), 1 << 16) for m, n in shapes]
