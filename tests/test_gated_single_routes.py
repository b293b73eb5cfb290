"""CPU: the kernels that the rules of dc_linear_route.hpp pick for a gated layer's gradients asked for by themselves, which are others than those of all of
them at once: for the shapes of tests/gated_single_kernels.py, so that tests of a kernel stay tests of it; and every kernel that they can pick is among them."""
import os
import subprocess

import pytest

from gated_single_kernels import SINGLES

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# The sizes are those of dc_hip_gated_linear_backward, for dense rows.
PROBE = """
#include <cstdio>
#include <string>
#include "dc_linear_route.hpp"
using namespace dc;
static int64_t padded(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
static std::string single(const std::string& which, int64_t m, int64_t n, int64_t k) {
  const int64_t pitch = 2 * padded(k, 8), dz = 4 * padded(n, 64), weights = which == "dws" ? 2 : 1;
  const LinearSize size = which == "dx" ? LinearSize{m, k, dz, dz, pitch} : LinearSize{weights * n, k, 2 * m, 2 * padded(m, 8), pitch};
  const LinearPlan p = linear_plan(size, {true, false}, 256);
  const int64_t groups = linear_tile_groups(p.tile);
  return std::to_string(linear_tile_side(p.tile)) + (groups > 1 ? "x" + std::to_string(groups) : "") + (p.split.parts > 1 ? "/split" : "");
}
int main() {
  char which[16];
  long m, n, k;
  while (std::scanf("%15s %ld %ld %ld", which, &m, &n, &k) == 4) std::puts(single(which, m, n, k).c_str());
}
"""


@pytest.fixture(scope="module")
def picks(tmp_path_factory):
    where = tmp_path_factory.mktemp("routes")
    (where / "probe.cpp").write_text(PROBE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "dotcompute_amd", "csrc"), str(where / "probe.cpp"), "-o",
                    str(where / "probe")], check=True)

    def ask(questions):
        text = "".join(f"{which} {m} {n} {k}\n" for which, m, n, k in questions)
        return subprocess.run([str(where / "probe")], input=text, capture_output=True, text=True, check=True).stdout.split()

    return ask


def test_each_shape_takes_its_kernel(picks):
    got = picks([(which, *shape) for which, _, *shape in SINGLES])
    assert SINGLES == [(which, name, *shape) for name, (which, _, *shape) in zip(got, SINGLES)]


@pytest.mark.parametrize("which", ["dx", "dw", "dws"])
def test_every_kernel_has_a_shape(picks, which):
    """Over a grid of sizes no kernel is picked that has none."""
    sizes = sorted({int(1.5 ** i) for i in range(1, 23)} | {4096, 8192})
    seen = set(picks([(which, m, n, k) for m in sizes for n in sizes for k in sizes]))
    assert seen <= {name for w, name, *_ in SINGLES if w == which}


def test_groups_of_waves_stand_on_both_sides_of_the_weights_border():
    for which, name, _, n, _ in SINGLES:
        if which == "dx" and "x" in name:
            assert -(-n // 64) % int(name.split("x")[1].split("/")[0]), (name, n)
