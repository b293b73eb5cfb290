"""CPU: the kernels that dc_linear_route.hpp picks for the shapes of tests/linear_kernels.py, so that tests of a kernel stay tests of it when the
estimate is fitted anew; and every kernel that it can pick is among them."""
import os
import subprocess

import pytest

from linear_kernels import FORWARD, LARGE, PAIRS, SINGLES

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# The order of the choices is that of dc_hip_linear and dc_hip_linear_backward, for dense rows.
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
  if (c % 16 && linear_few_rows_any(m, n, c)) return "any";
  if (linear_few_rows(m, n, 256))
    return (linear_wide_few_rows(m, n, 256) ? "fewwide" : "few") + std::to_string(m > 32 ? 8 : (m + 7) / 8);
  const LinearPlan p = linear_plan({m, n, c, pitch, pitch}, {false, fp8}, 256);
  return tile(p.tile) + (p.split.parts > 1 ? "/split" : "");
}
static std::string pair(int64_t m, int64_t n, int64_t k) {
  const int64_t pitch = 2 * padded(k, 8);
  const LinearPair q = linear_plan_of_two({m, k, 2 * n, 2 * padded(n, 8), pitch}, {n, k, 2 * m, 2 * padded(m, 8), pitch}, 256);
  return tile(q.tile) + (q.a.parts > 1 ? "/a" : "") + (q.b.parts > 1 ? "/b" : "");
}
static std::string single(int64_t m, int64_t c, int64_t k) {
  const LinearPlan p = linear_plan({m, k, 2 * c, 2 * padded(c, 8), 2 * padded(k, 8)}, {true, false}, 256);
  return tile(p.tile) + (p.split.parts > 1 ? "/split" : "");
}
int main() {
  char what[16];
  long a, b, c;
  while (std::scanf("%15s %ld %ld %ld", what, &a, &b, &c) == 4)
    std::puts((!std::strcmp(what, "pair")     ? pair(a, b, c)
               : !std::strcmp(what, "single") ? single(a, b, c)
                                              : forward(a, b, c, !std::strcmp(what, "fp8"))).c_str());
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
    cases = [(name, (dtype, m, n, k)) for name, m, n, k, dtype in FORWARD + LARGE]
    cases += [(name, ("pair", *shape)) for name, *shape in PAIRS] + [(name, ("single", *shape)) for name, *shape in SINGLES]
    got = picks([shape for _, shape in cases])
    assert [(name, *shape) for name, shape in cases] == [(name, *shape) for name, (_, shape) in zip(got, cases)]


def test_every_kernel_has_a_shape(picks):
    """Over a grid of sizes no kernel is picked that has none."""
    sizes = sorted({int(1.5 ** i) for i in range(1, 23)} | {4096, 8192})
    for what, named in (("bf16", {c[0] for c in FORWARD + LARGE if c[4] == "bf16"}), ("fp8", {c[0] for c in FORWARD if c[4] == "fp8"}),
                        ("pair", {c[0] for c in PAIRS}), ("single", {c[0] for c in SINGLES})):
        seen = set(picks([(what, m, n, k) for m in sizes for n in sizes for k in sizes]))
        assert seen <= named, (what, seen - named)
