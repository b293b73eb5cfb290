// FeedForward.hpp — a pre-norm feed-forward block on the HIP accelerator, trained with AdamW and served in bf16 or 8 bits:
// y = x + W2 act(W1 norm(x) + b1) + b2. It holds its parameters and states on the device and is made of the dc_hip_rms_norm,
// dc_hip_linear, dc_hip_adamw_step entry points and their gradients.
//
// The reference has no counterpart (its dense arithmetic stops at MatrixOperations.MultiplyAsync,
// src/Extensions/DotCompute.Algorithms/LinearAlgebra/Operations/MatrixOperations.cs:28-64); arguments, exceptions and the
// explicit accelerator follow Algorithms.hpp.
#pragma once

#include <array>

#include "Algorithms.hpp"

namespace DotCompute::Algorithms {

enum class Activation { None, Relu, Gelu, GeluTanh, Silu };

struct AdamWOptions {
  double LearningRate = 1e-3, Beta1 = 0.9, Beta2 = 0.999, Epsilon = 1e-8, WeightDecay = 0.01;
};

class FeedForwardBlock {
 public:
  // Which parameter: the norm's weight [width], W1 [hidden][width], b1 [hidden], W2 [width][hidden], b2 [width].
  enum Parameter { NormWeight, W1, B1, W2, B2 };
  static constexpr int kParameters = 5;

  // Weights start as zeros, the norm's as ones. ArgumentException unless both sizes are positive.
  FeedForwardBlock(int32_t width, int32_t hidden, Activation activation, IAccelerator& accelerator, float epsilon = 1e-6f);
  int32_t Width() const { return width_; }
  int32_t Hidden() const { return hidden_; }

  // ArgumentException when the length is not the parameter's.
  void Set(Parameter parameter, const std::vector<float>& values);
  std::vector<float> Get(Parameter parameter) const;
  // The gradient that the last Backward left, before and after a Step. InvalidOperationException before the first.
  std::vector<float> Gradient(Parameter parameter) const;

  // One row of x a token (x.Columns == Width, else ArgumentException). Products of bf16 values, sums in float32; what
  // Backward needs is kept; a Forward that throws past its check of x leaves nothing for a Backward.
  Matrix Forward(const Matrix& x);
  // The gradients of a loss by x (returned) and by the parameters (kept), from its gradient by Forward's result.
  // InvalidOperationException without a Forward since the last Set or Step, whose values were other ones; ArgumentException
  // unless dy has the shape of that Forward's result. A Backward that throws past these checks leaves no gradients.
  Matrix Backward(const Matrix& dy);
  // One AdamW step of all parameters from those gradients. InvalidOperationException without a Backward since the last.
  void Step(const AdamWOptions& options);
  // Forward for serving: products of 8-bit values with a scale per row of each operand. Keeps nothing.
  Matrix ForwardFp8(const Matrix& x);

 private:
  template <typename T>
  using Buffer = std::shared_ptr<IUnifiedMemoryBufferT<T>>;
  struct Tensor {
    int64_t rows = 0, cols = 0;
    Buffer<float> value, m, v;
    Buffer<uint16_t> copy;     // the value in bf16: what the products and the norm read
    Buffer<float> grad_f32;    // of vectors
    Buffer<uint16_t> grad_b16;  // of matrices
    int64_t Size() const { return rows * cols; }
  };
  template <typename T>
  Buffer<T> New(int64_t count) const;
  Buffer<uint16_t> ToBf16(const Matrix& x) const;
  void RequireInput(const Matrix& x) const;

  int32_t width_, hidden_;
  Activation activation_;
  float epsilon_;
  Backends::Hip::HipAccelerator* hip_;
  std::array<Tensor, kParameters> p_;
  int64_t steps_ = 0;
  int32_t rows_ = 0;  // of the last Forward
  bool has_forward_ = false, has_gradient_ = false, stepped_ = false, quantized_ = false;
  Buffer<uint16_t> x_, normed_, pre_, active_;  // kept for Backward
  Buffer<uint8_t> q1_, q2_;                     // W1 and W2 in 8 bits, made from the current values when first asked for
  Buffer<float> s1_, s2_;
};

}  // namespace DotCompute::Algorithms
