"""CPU: the kernels that the rules of dc_linear_route.hpp pick for the shapes of tests/gated_kernels.py, so that tests of a kernel stay tests of it; and
every kernel that they can pick is among them."""
import os
import subprocess

import pytest

from gated_kernels import FORWARD, GRADIENTS

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# The order of the choices is that of dc_hip_gated_linear and dc_hip_gated_linear_backward, for dense rows and all gradients.
PROBE = """
#include <cstdio>
#include <cstring>
#include <string>
#include "dc_linear_route.hpp"
using namespace dc;
static int64_t padded(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
static std::string tile(LinearTile t) {
  const int64_t g = linear_tile_groups(t);
  return std::to_string(linear_tile_side(t)) + (g > 1 ? "x" + std::to_string(g) : "");
}
static std::string forward(int64_t m, int64_t n, int64_t k, bool fp8) {
  const int64_t c = k * (fp8 ? 1 : 2), pitch = padded(c, 16);
  if (linear_few_rows(m, n, 256)) return "few" + std::to_string(m > 32 ? 8 : (m + 7) / 8);
  const LinearPlan p = linear_plan({m, 2 * n, c, pitch, pitch}, {false, fp8}, 256);
  return tile(p.tile) + (p.split.parts > 1 ? "/split" : "");
}
static std::string gradients(int64_t m, int64_t n, int64_t k) {
  const int64_t pitch = 2 * padded(k, 8), dz = 4 * padded(n, 64);
  const LinearPair q = linear_plan_of_two({m, k, dz, dz, pitch}, {2 * n, k, 2 * m, 2 * padded(m, 8), pitch}, 256, true);
  return tile(q.tile) + (q.a.parts > 1 ? "/a" : "") + (q.b.parts > 1 ? "/b" : "");
}
int main() {
  char what[16];
  long a, b, c;
  while (std::scanf("%15s %ld %ld %ld", what, &a, &b, &c) == 4)
    std::puts((!std::strcmp(what, "grad") ? gradients(a, b, c) : forward(a, b, c, std::strcmp(what, "bf16") != 0)).c_str());
}
"""


@pytest.fixture(scope="module")
def picks(tmp_path_factory):
    where = tmp_path_factory.mktemp("routes")
    (where / "probe.cpp").write_text(PROBE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "dotcompute_amd", "csrc"), str(where / "probe.cpp"), "-o",
                    str(where / "probe")], check=True)

    def ask(questions):
        text = "".join(f"{what} {a} {b} {c}\n" for what, a, b, c in questions)
        return subprocess.run([str(where / "probe")], input=text, capture_output=True, text=True, check=True).stdout.split()

    return ask


def test_each_shape_takes_its_kernel(picks):
    cases = [(name, (dtype, m, n, k)) for name, m, n, k, dtype in FORWARD] + [(name, ("grad", *shape)) for name, *shape in GRADIENTS]
    got = picks([shape for _, shape in cases])
    assert [(name, *shape) for name, shape in cases] == [(name, *shape) for name, (_, shape) in zip(got, cases)]


def test_every_kernel_has_a_shape(picks):
    """Over a grid of sizes no kernel is picked that has none."""
    sizes = sorted({int(1.5 ** i) for i in range(1, 23)} | {4096, 8192})
    for what, named in (("bf16", {c[0] for c in FORWARD if c[4] == "bf16"}), ("fp8", {c[0] for c in FORWARD if c[4] != "bf16"}),
                        ("grad", {c[0] for c in GRADIENTS})):
        seen = set(picks([(what, m, n, k) for m in sizes for n in sizes for k in sizes]))
        assert seen <= named, (what, seen - named)
