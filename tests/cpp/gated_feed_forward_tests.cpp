// The gated feed-forward block of the host layer (FeedForward.hpp): its norm, projections, gradients and step run together, against the same block in
// float64 here; what it keeps between its calls, and which calls it refuses.
#include <array>
#include <cmath>
#include <cstring>
#include <random>

#include "DotCompute/FeedForward.hpp"
#include "test_framework.hpp"

using namespace DotCompute;
using DotCompute::Algorithms::Activation;
using DotCompute::Algorithms::AdamWOptions;
using DotCompute::Algorithms::GatedFeedForwardBlock;
using DotCompute::Algorithms::Matrix;

namespace {

typedef GatedFeedForwardBlock Block;
typedef std::vector<double> Doubles;

std::vector<float> Rounded(size_t n, uint32_t seed, float scale = 1.0f, float shift = 0.0f) {
  std::mt19937 gen(seed);
  std::normal_distribution<float> dist(0.0f, 1.0f);
  std::vector<float> v(n);
  for (float& x : v) {
    x = dist(gen) * scale + shift;
    uint32_t u;
    std::memcpy(&u, &x, 4);
    u = (u + 0x7fffu + ((u >> 16) & 1u)) & 0xffff0000u;  // to bf16
    std::memcpy(&x, &u, 4);
  }
  return v;
}

// The block in float64, with no rounding between its parts.
struct Reference {
  int d, h, rows = 0;
  std::array<Doubles, Block::kParameters> p, grad;
  Doubles x, unit, normed, s, g, u;

  Reference(int d_, int h_) : d(d_), h(h_) {}
  std::vector<std::vector<float>> Fill() {
    const float w = 1.0f / std::sqrt((float)d), w2 = 1.0f / std::sqrt((float)h);
    std::vector<std::vector<float>> v = {Rounded((size_t)d, 1, 0.1f, 1.0f), Rounded((size_t)d, 2, 0.1f),     Rounded((size_t)h * d, 3, w),
                                         Rounded((size_t)h, 4, 0.1f),       Rounded((size_t)h * d, 5, w),    Rounded((size_t)h, 6, 0.1f),
                                         Rounded((size_t)d * h, 7, w2),     Rounded((size_t)d, 8, 0.1f)};
    for (int i = 0; i < Block::kParameters; ++i) p[i].assign(v[i].begin(), v[i].end());
    return v;
  }
  static double Silu(double z) { return z / (1.0 + std::exp(-z)); }
  Doubles Forward(const std::vector<float>& input, int r) {
    rows = r;
    x.assign(input.begin(), input.end());
    unit = normed = x;
    s.assign((size_t)r, 0.0);
    g.assign((size_t)r * h, 0.0);
    u = g;
    Doubles y((size_t)r * d);
    for (int i = 0; i < r; ++i) {
      double mean = 0.0, var = 0.0;
      for (int c = 0; c < d; ++c) mean += x[i * d + c] / d;
      for (int c = 0; c < d; ++c) var += (x[i * d + c] - mean) * (x[i * d + c] - mean) / d;
      s[i] = 1.0 / std::sqrt(var + 1e-5);
      for (int c = 0; c < d; ++c) {
        unit[i * d + c] = (x[i * d + c] - mean) * s[i];
        normed[i * d + c] = unit[i * d + c] * p[Block::NormWeight][c] + p[Block::NormBias][c];
      }
      for (int j = 0; j < h; ++j) {
        double a = p[Block::BGate][j], b = p[Block::BUp][j];
        for (int c = 0; c < d; ++c) {
          a += normed[i * d + c] * p[Block::WGate][j * d + c];
          b += normed[i * d + c] * p[Block::WUp][j * d + c];
        }
        g[i * h + j] = a, u[i * h + j] = b;
      }
      for (int c = 0; c < d; ++c) {
        double t = p[Block::BDown][c] + x[i * d + c];
        for (int j = 0; j < h; ++j) t += Silu(g[i * h + j]) * u[i * h + j] * p[Block::WDown][c * h + j];
        y[i * d + c] = t;
      }
    }
    return y;
  }
  Doubles Backward(const std::vector<float>& dy) {
    for (int i = 0; i < Block::kParameters; ++i) grad[i].assign(p[i].size(), 0.0);
    Doubles dx((size_t)rows * d);
    for (int i = 0; i < rows; ++i) {
      Doubles dn(d);
      for (int j = 0; j < h; ++j) {
        const double a = g[i * h + j], b = u[i * h + j], sig = 1.0 / (1.0 + std::exp(-a));
        double da = 0.0;
        for (int c = 0; c < d; ++c) {
          da += dy[i * d + c] * p[Block::WDown][c * h + j];
          grad[Block::WDown][c * h + j] += dy[i * d + c] * a * sig * b;
        }
        const double dg = da * b * sig * (1.0 + a * (1.0 - sig)), du = da * a * sig;
        grad[Block::BGate][j] += dg, grad[Block::BUp][j] += du;
        for (int c = 0; c < d; ++c) {
          dn[c] += dg * p[Block::WGate][j * d + c] + du * p[Block::WUp][j * d + c];
          grad[Block::WGate][j * d + c] += dg * normed[i * d + c];
          grad[Block::WUp][j * d + c] += du * normed[i * d + c];
        }
      }
      double flat = 0.0, along = 0.0;
      for (int c = 0; c < d; ++c) {
        const double q = dn[c] * p[Block::NormWeight][c];
        flat += q / d, along += q * unit[i * d + c] / d;
        grad[Block::NormWeight][c] += dn[c] * unit[i * d + c];
        grad[Block::NormBias][c] += dn[c];
        grad[Block::BDown][c] += dy[i * d + c];
      }
      for (int c = 0; c < d; ++c)
        dx[i * d + c] = s[i] * (dn[c] * p[Block::NormWeight][c] - flat - unit[i * d + c] * along) + dy[i * d + c];
    }
    return dx;
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

}  // namespace

// Tolerances, relative in the 2-norm: a rounding to bf16 is within 2^-8 of each value. Forward rounds the norm's result, which both factors
// carry, and their product: 3 × 2^-8 and as much again of the activation's slope and the result. Backward rounds dy, the projections' dz and dx, and reads the
// rounded norm, factors and product: at most 12 × 2^-8. In 8 bits each operand is within 2^-4: the norm's result twice, three weights and the product.
TEST_GPU(gated_feed_forward_block_matches_float64) {
  auto acc = Device();
  for (auto [rows, d, h] : {std::array<int, 3>{1, 64, 256}, {5, 33, 70}, {100, 136, 160}}) {
    Reference ref(d, h);
    Block block(d, h, Activation::Silu, *acc);
    const auto values = ref.Fill();
    for (int i = 0; i < Block::kParameters; ++i) {
      block.Set((Block::Parameter)i, values[(size_t)i]);
      CHECK(block.Get((Block::Parameter)i) == values[(size_t)i]);
    }
    const auto input = Rounded((size_t)rows * d, 9), dy = Rounded((size_t)rows * d, 10);
    const Doubles y = ref.Forward(input, rows);
    CHECK(Off(block.Forward(Matrix(rows, d, input)).Data(), y) <= 4.0 / 256);
    const Doubles dx = ref.Backward(dy);
    CHECK(Off(block.Backward(Matrix(rows, d, dy)).Data(), dx) <= 12.0 / 256);
    for (int i = 0; i < Block::kParameters; ++i) CHECK(Off(block.Gradient((Block::Parameter)i), ref.grad[(size_t)i]) <= 12.0 / 256);
    CHECK(Off(block.ForwardFp8(Matrix(rows, d, input)).Data(), y) <= 6.0 / 16);
  }
}

// What a step does reaches the bf16 copies and the 8-bit ones.
TEST_GPU(gated_feed_forward_block_steps) {
  auto acc = Device();
  const int rows = 6, d = 24, h = 40;
  Reference ref(d, h);
  Block block(d, h, Activation::Silu, *acc);
  const auto values = ref.Fill();
  for (int i = 0; i < Block::kParameters; ++i) block.Set((Block::Parameter)i, values[(size_t)i]);
  const Matrix x(rows, d, Rounded((size_t)rows * d, 11));
  const auto before = block.Forward(x).Data(), coded = block.ForwardFp8(x).Data();
  block.Backward(x);
  AdamWOptions options;
  options.LearningRate = 1e-2;
  block.Step(options);
  for (int i = 0; i < Block::kParameters; ++i) CHECK(block.Get((Block::Parameter)i) != values[(size_t)i]);
  const auto after = block.Forward(x).Data();
  CHECK(after != before && block.ForwardFp8(x).Data() != coded);
  // the same as a block that was given the new values
  Block other(d, h, Activation::Silu, *acc);
  for (int i = 0; i < Block::kParameters; ++i) other.Set((Block::Parameter)i, block.Get((Block::Parameter)i));
  CHECK(other.Forward(x).Data() == after && other.ForwardFp8(x).Data() == block.ForwardFp8(x).Data());
}

TEST_GPU(gated_feed_forward_block_refusals) {
  auto acc = Device();
  CHECK_THROWS(ArgumentException, Block(0, 4, Activation::None, *acc));
  CHECK_THROWS(ArgumentException, Block(4, 4, Activation::None, *acc, -1.0f));
  Block block(4, 8, Activation::Gelu, *acc);
  CHECK_THROWS(ArgumentException, block.Set(Block::WUp, std::vector<float>(31)));
  CHECK_THROWS(ArgumentException, block.Forward(Matrix(2, 5)));
  CHECK_THROWS(ArgumentException, block.ForwardFp8(Matrix(2, 3)));
  CHECK_THROWS(InvalidOperationException, block.Backward(Matrix(2, 4)));
  CHECK_THROWS(InvalidOperationException, block.Step(AdamWOptions()));
  CHECK_THROWS(InvalidOperationException, block.Gradient(Block::BGate));
  CHECK(block.Forward(Matrix(0, 4)).Size() == 0 && block.ForwardFp8(Matrix(0, 4)).Size() == 0);
  const Matrix x(3, 4, Rounded(12, 1));
  CHECK(block.Forward(x).Data() == x.Data());  // all weights zero: the residual alone
  CHECK_THROWS(ArgumentException, block.Backward(Matrix(2, 4)));
  block.Backward(x);
  block.Set(Block::BUp, std::vector<float>(8, 1.0f));
  CHECK_THROWS(InvalidOperationException, block.Backward(x));  // (gradients of other parameters)
}

// More than 2^22 outputs are refused by the projections, after the norm has been enqueued.
TEST_GPU(gated_feed_forward_block_keeps_nothing_of_a_forward_that_throws) {
  auto acc = Device();
  Block block(1, (1 << 22) + 1, Activation::Relu, *acc);
  CHECK_THROWS(NotSupportedException, block.Forward(Matrix(2, 1)));
  CHECK_THROWS(InvalidOperationException, block.Backward(Matrix(2, 1)));
}
