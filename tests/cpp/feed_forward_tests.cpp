// The feed-forward block of the host layer (FeedForward.hpp): its products, norm, gradients and step run together, against the same
// block in float64 here; and the rules that pick the linear layers' kernels (dc_linear_route.hpp), on the CPU.
#include <cmath>
#include <cstring>
#include <random>

#include "../../dotcompute_amd/csrc/dc_linear_route.hpp"
#include "DotCompute/FeedForward.hpp"
#include "test_framework.hpp"

using namespace DotCompute;
using DotCompute::Algorithms::Activation;
using DotCompute::Algorithms::AdamWOptions;
using DotCompute::Algorithms::FeedForwardBlock;
using DotCompute::Algorithms::Matrix;

namespace {

typedef std::vector<double> Doubles;

std::vector<float> Normal(size_t n, uint32_t seed, float scale = 1.0f, float shift = 0.0f) {
  std::mt19937 gen(seed);
  std::normal_distribution<float> dist(0.0f, 1.0f);
  std::vector<float> v(n);
  for (float& x : v) x = dist(gen) * scale + shift;
  return v;
}

float RoundBf16(float x) {
  uint32_t u;
  std::memcpy(&u, &x, 4);
  u = (u + 0x7fffu + ((u >> 16) & 1u)) & 0xffff0000u;
  std::memcpy(&x, &u, 4);
  return x;
}

// The block in float64 on values that were rounded to bf16, with no rounding between its parts.
struct Reference {
  int d, h, rows = 0;
  Doubles norm, w1, b1, w2, b2, x, unit, normed, z, a, s;

  Doubles Forward(const std::vector<float>& input, int r) {
    rows = r;
    x.assign(input.begin(), input.end());
    for (double& v : x) v = RoundBf16((float)v);
    unit = normed = x;
    s.assign((size_t)r, 0.0);
    z.assign((size_t)r * h, 0.0);
    a = z;
    Doubles y((size_t)r * d);
    for (int i = 0; i < r; ++i) {
      double ss = 0.0;
      for (int c = 0; c < d; ++c) ss += x[i * d + c] * x[i * d + c];
      s[i] = 1.0 / std::sqrt(ss / d + 1e-6);
      for (int c = 0; c < d; ++c) unit[i * d + c] = x[i * d + c] * s[i], normed[i * d + c] = unit[i * d + c] * norm[c];
      for (int j = 0; j < h; ++j) {
        double t = b1[j];
        for (int c = 0; c < d; ++c) t += normed[i * d + c] * w1[j * d + c];
        z[i * h + j] = t;
        a[i * h + j] = t / (1.0 + std::exp(-t));
      }
      for (int c = 0; c < d; ++c) {
        double t = b2[c] + x[i * d + c];
        for (int j = 0; j < h; ++j) t += a[i * h + j] * w2[c * h + j];
        y[i * d + c] = t;
      }
    }
    return y;
  }
  struct Gradients {
    Doubles x, norm, w1, b1, w2, b2;
  };
  Gradients Backward(const std::vector<float>& dy) const {
    Gradients g{Doubles((size_t)rows * d), Doubles(d), Doubles((size_t)h * d), Doubles(h), Doubles((size_t)d * h), Doubles(d)};
    for (int i = 0; i < rows; ++i) {
      Doubles dz(h), dn(d);
      for (int j = 0; j < h; ++j) {
        double da = 0.0;
        for (int c = 0; c < d; ++c) {
          da += dy[i * d + c] * w2[c * h + j];
          g.w2[c * h + j] += dy[i * d + c] * a[i * h + j];
        }
        const double sig = 1.0 / (1.0 + std::exp(-z[i * h + j]));
        dz[j] = da * sig * (1.0 + z[i * h + j] * (1.0 - sig));
        g.b1[j] += dz[j];
        for (int c = 0; c < d; ++c) {
          g.w1[j * d + c] += dz[j] * normed[i * d + c];
          dn[c] += dz[j] * w1[j * d + c];
        }
      }
      double along = 0.0;
      for (int c = 0; c < d; ++c) along += dn[c] * norm[c] * unit[i * d + c] / d;
      for (int c = 0; c < d; ++c) {
        g.b2[c] += dy[i * d + c];
        g.norm[c] += dn[c] * unit[i * d + c];
        g.x[i * d + c] = s[i] * (dn[c] * norm[c] - unit[i * d + c] * along) + dy[i * d + c];
      }
    }
    return g;
  }
};

double Off(const std::vector<float>& got, const Doubles& want) {
  CHECK(got.size() == want.size());
  double d = 0.0, n = 0.0;
  for (size_t i = 0; i < want.size(); ++i) d += (got[i] - want[i]) * (got[i] - want[i]), n += want[i] * want[i];
  return std::sqrt(d / n);
}

std::shared_ptr<Backends::Hip::HipAccelerator> Device() {
  auto acc = Backends::Hip::TryCreateAccelerator();
  CHECK(acc != nullptr);
  return acc;
}

struct Setup {
  int d, h;
  std::vector<float> values[FeedForwardBlock::kParameters];
  Reference ref;
  Setup(int d_, int h_) : d(d_), h(h_) {
    values[0] = Normal((size_t)d, 1, 0.1f, 1.0f);
    values[1] = Normal((size_t)h * d, 2, 1.0f / std::sqrt((float)d));
    values[2] = Normal((size_t)h, 3, 0.1f);
    values[3] = Normal((size_t)d * h, 4, 1.0f / std::sqrt((float)h));
    values[4] = Normal((size_t)d, 5, 0.1f);
    for (auto& v : values)
      for (float& x : v) x = RoundBf16(x);
    Doubles* to[] = {&ref.norm, &ref.w1, &ref.b1, &ref.w2, &ref.b2};
    for (int i = 0; i < FeedForwardBlock::kParameters; ++i) to[i]->assign(values[i].begin(), values[i].end());
    ref.d = d, ref.h = h;
  }
  void Load(FeedForwardBlock& block) const {
    for (int i = 0; i < FeedForwardBlock::kParameters; ++i) block.Set((FeedForwardBlock::Parameter)i, values[i]);
  }
};

}  // namespace

// Tolerances, relative in the 2-norm: a rounding to bf16 is within 2^-8 of each value. Forward rounds the norm's result and the
// activation (the sums carry those errors as they are: at most 2 × 2^-8), Backward the incoming gradient, both layers'
// dz and dx and the saved values: at most 8 × 2^-8. In 8 bits each operand is within 2^-4 of its values or of its row's
// smallest code: four of them, which reach the output through a branch of about its own size: 4 × 2^-4.
TEST_GPU(feed_forward_block_matches_float64) {
  auto acc = Device();
  for (auto [rows, d, h] : {std::array<int, 3>{1, 64, 256}, {5, 33, 70}, {100, 96, 160}}) {
    Setup s(d, h);
    FeedForwardBlock block(d, h, Activation::Silu, *acc);
    s.Load(block);
    const auto input = Normal((size_t)rows * d, 7), seed = Normal((size_t)rows * d, 8);
    std::vector<float> dy(seed);
    for (float& v : dy) v = RoundBf16(v);
    const Doubles y = s.ref.Forward(input, rows);
    CHECK(Off(block.Forward(Matrix(rows, d, input)).Data(), y) <= 2.0 / 256);
    const auto g = s.ref.Backward(dy);
    CHECK(Off(block.Backward(Matrix(rows, d, dy)).Data(), g.x) <= 8.0 / 256);
    const Doubles* want[] = {&g.norm, &g.w1, &g.b1, &g.w2, &g.b2};
    for (int i = 0; i < FeedForwardBlock::kParameters; ++i)
      CHECK(Off(block.Gradient((FeedForwardBlock::Parameter)i), *want[i]) <= 8.0 / 256);
    CHECK(Off(block.ForwardFp8(Matrix(rows, d, input)).Data(), y) <= 4.0 / 16);
  }
}

TEST_GPU(feed_forward_block_learns) {
  auto acc = Device();
  const int rows = 64, d = 48, h = 96;
  Setup s(d, h), goal(d, h);
  goal.values[3] = Normal((size_t)d * h, 40, 1.0f / std::sqrt((float)h));
  goal.ref.w2.assign(goal.values[3].begin(), goal.values[3].end());
  FeedForwardBlock block(d, h, Activation::Silu, *acc);
  s.Load(block);
  const auto input = Normal((size_t)rows * d, 9);
  const Doubles want = goal.ref.Forward(input, rows);
  AdamWOptions options;
  options.LearningRate = 1e-2, options.WeightDecay = 0.0;
  double first = 0.0, last = 0.0;
  for (int t = 0; t < 60; ++t) {
    Matrix y = block.Forward(Matrix(rows, d, input));
    Matrix dy(rows, d);
    last = 0.0;
    for (size_t i = 0; i < want.size(); ++i) {
      const double e = y.Data()[i] - want[i];
      last += e * e;
      dy.Data()[i] = (float)(2.0 * e / rows);
    }
    if (t == 0) first = last;
    block.Backward(dy);
    block.Step(options);
  }
  CHECK(last < first / 20.0);
  // what was learnt serves in 8 bits too: the weights' 8-bit copies follow the steps
  const Matrix y = block.Forward(Matrix(rows, d, input)), q = block.ForwardFp8(Matrix(rows, d, input));
  Doubles now(y.Data().begin(), y.Data().end());
  CHECK(Off(q.Data(), now) <= 4.0 / 16);
}

TEST_GPU(feed_forward_block_refusals) {
  auto acc = Device();
  CHECK_THROWS(ArgumentException, FeedForwardBlock(0, 4, Activation::None, *acc));
  CHECK_THROWS(ArgumentException, FeedForwardBlock(4, 4, Activation::None, *acc, -1.0f));
  FeedForwardBlock block(4, 8, Activation::Gelu, *acc);
  CHECK_THROWS(ArgumentException, block.Set(FeedForwardBlock::W1, std::vector<float>(31)));
  CHECK_THROWS(ArgumentException, block.Forward(Matrix(2, 5)));
  CHECK_THROWS(ArgumentException, block.ForwardFp8(Matrix(2, 3)));
  CHECK_THROWS(InvalidOperationException, block.Backward(Matrix(2, 4)));
  CHECK_THROWS(InvalidOperationException, block.Step(AdamWOptions()));
  CHECK_THROWS(InvalidOperationException, block.Gradient(FeedForwardBlock::B1));
  CHECK(block.Forward(Matrix(0, 4)).Size() == 0);
  const Matrix x(3, 4, Normal(12, 1));
  const Matrix y = block.Forward(x);  // all weights zero: the residual alone
  for (int64_t i = 0; i < 12; ++i) CHECK(y.Data()[(size_t)i] == RoundBf16(x.Data()[(size_t)i]));
  CHECK_THROWS(ArgumentException, block.Backward(Matrix(2, 4)));
}

TEST_CPU(linear_routes) {
  using dc::LinearTile;
  struct Row {
    int64_t m, n, c_bytes;
    bool rows_c, fp8;
    LinearTile want;
    int64_t parts;
  };
  const Row rows[] = {
      {8192, 8192, 16384, false, false, LinearTile::k256, 1},  {8192, 2048, 16384, true, false, LinearTile::k256, 1},
      {8192, 8192, 128, false, false, LinearTile::k256, 1},    {4096, 8192, 4096, false, true, LinearTile::k256, 1},
      {4352, 4096, 2048, false, false, LinearTile::k128, 1},   {2048, 2048, 4096, false, false, LinearTile::k128x2, 1},
      {1537, 2049, 2048, false, false, LinearTile::k64, 1},
      {1500, 1500, 12000, false, false, LinearTile::k128, 3},
  };
  for (const Row& r : rows) {
    const dc::LinearPlan p = dc::linear_plan({r.m, r.n, r.c_bytes, r.c_bytes, r.c_bytes}, {r.rows_c, r.fp8}, 256);
    CHECK(p.tile == r.want && p.split.parts == r.parts);
  }
  // the widest rows stay within the loads' range: small tiles only
  const LinearTile narrow = dc::linear_plan({8192, 8192, 16384, dc::kLinearPitch, dc::kLinearPitch}, {false, false}, 256).tile;
  CHECK(dc::linear_tile_side(narrow) == 64);
  CHECK(dc::linear_plan({8192, 8192, 16384, 16384, dc::kLinearPitch}, {true, false}, 256).tile == LinearTile::k256);
  // splits: every tile along c belongs to exactly one part, and none is empty
  auto whole = [](const dc::LinearSplit& s, LinearTile t, int64_t c) {
    const int64_t step = 128 * dc::linear_tile_groups(t), all = (c + step - 1) / step;
    return s.parts >= 1 && s.parts <= 64 && s.turns >= 1 && s.parts * s.turns >= all && (s.parts - 1) * s.turns < all;
  };
  for (int64_t m : {1, 64, 300, 2515, 8192})
    for (int64_t n : {1, 64, 256, 1000, 8192})
      for (int64_t c : {2, 128, 1000, 2046, 10336, 1 << 24}) {
        const dc::LinearSize a{m, n, c, c, c}, b{n, m, 2 * m, 2 * m, 2 * m};
        const dc::LinearPlan p = dc::linear_plan(a, {false, false}, 256);
        CHECK(whole(p.split, p.tile, c) && p.time > 0.0 && p.time < 1e12);
        const dc::LinearPair q = dc::linear_plan_of_two(a, b, 256);
        CHECK(whole(q.a, q.tile, a.c_bytes) && whole(q.b, q.tile, b.c_bytes));
        const dc::LinearPair r = dc::linear_plan_of_two(b, a, 256);  // (in either order)
        CHECK(a.c_bytes == b.c_bytes || (r.tile == q.tile && r.a.parts == q.b.parts && r.b.parts == q.a.parts));
      }
  // both gradients of an ordinary layer: 128-tiles fill the chip together, as neither's do
  const dc::LinearSize dx{2000, 1000, 6000, 6000, 2000}, dw{3000, 1000, 4000, 4000, 2000};
  CHECK(dc::linear_plan_of_two(dx, dw, 256).tile == LinearTile::k128 && dc::linear_plan(dx, {true, false}, 256).tile != LinearTile::k128);
  CHECK(dc::linear_few_rows(1, 1, 256) && dc::linear_few_rows(32, 100000, 256) && dc::linear_few_rows(64, 4096, 256));
  CHECK(!dc::linear_few_rows(64, 4112, 256) && !dc::linear_few_rows(33, 8192, 256) && dc::linear_few_rows(4096, 64, 256));
  CHECK(dc::linear_wide_few_rows(8, 16384, 256) && !dc::linear_wide_few_rows(8, 8192, 256));
  CHECK(dc::linear_few_rows_any(1, 1000, 666) && dc::linear_few_rows_any(1, 4096, 8190) && !dc::linear_few_rows_any(16, 4096, 8190));
  CHECK(!dc::linear_few_rows_any(33, 16, 2) && !dc::linear_few_rows_any(4, 216, 15954));
}
