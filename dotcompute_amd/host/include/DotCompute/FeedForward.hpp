// FeedForward.hpp — pre-norm feed-forward blocks on the HIP accelerator, trained with AdamW and served in bf16 or 8 bits:
// y = x + W2 act(W1 norm(x) + b1) + b2 (FeedForwardBlock, RMS norm) and y = x + Wd (act(Wg n + bg) * (Wu n + bu)) + bd with n = layer norm(x)
// (GatedFeedForwardBlock). They hold their parameters and states on the device and are made of the dc_hip_rms_norm, dc_hip_layer_norm,
// dc_hip_linear, dc_hip_gated_linear, dc_hip_adamw_step entry points and their like.
//
// The reference has no counterpart (its dense arithmetic stops at MatrixOperations.MultiplyAsync,
// src/Extensions/DotCompute.Algorithms/LinearAlgebra/Operations/MatrixOperations.cs:28-64); arguments, exceptions and the
// explicit accelerator follow Algorithms.hpp.
#pragma once

#include <vector>

#include "Algorithms.hpp"

namespace DotCompute::Algorithms {

enum class Activation { None, Relu, Gelu, GeluTanh, Silu };

struct AdamWOptions {
  double LearningRate = 1e-3, Beta1 = 0.9, Beta2 = 0.999, Epsilon = 1e-8, WeightDecay = 0.01;
};

// What a block keeps on the device: its parameters in float32, their copies in bf16 (what products and norms read), gradients and AdamW states.
class BlockParameters {
 public:
  int32_t Width() const { return width_; }
  int32_t Hidden() const { return hidden_; }
  // One AdamW step of all parameters from the last Backward's gradients. InvalidOperationException without a Backward since the last.
  void Step(const AdamWOptions& options);

 protected:
  template <typename T>
  using Buffer = std::shared_ptr<IUnifiedMemoryBufferT<T>>;
  struct Shape {
    bool matrix;  // (whose gradients are bf16)
    int64_t rows, cols;
    float start;  // what its values start as
  };
  struct Tensor {
    int64_t rows = 0, cols = 0;
    Buffer<float> value, m, v;
    Buffer<uint16_t> copy;
    Buffer<float> grad_f32;
    Buffer<uint16_t> grad_b16;
    int64_t Size() const { return rows * cols; }
  };
  // ArgumentException unless both sizes are positive and epsilon is not negative; NotSupportedException on another accelerator.
  BlockParameters(std::string name, int32_t width, int32_t hidden, IAccelerator& accelerator, float epsilon);
  void Allocate(const std::vector<Shape>& shapes);
  void SetValues(int parameter, const std::vector<float>& values);
  std::vector<float> Values(int parameter) const;
  std::vector<float> GradientOf(int parameter) const;

  template <typename T>
  Buffer<T> New(int64_t count) const;
  Buffer<uint16_t> ToBf16(const Matrix& x) const;
  void RequireInput(const Matrix& x) const;
  void RequireBackward(const Matrix& dy) const;
  Matrix Result(const Buffer<float>& y, int32_t rows) const;     // (waits for it)
  Matrix Result(const Buffer<uint16_t>& y, int32_t rows) const;
  const uint16_t* Copy(int parameter) const { return p_[(size_t)parameter].copy->Data(); }

  std::string name_;
  int32_t width_, hidden_;
  float epsilon_;
  Backends::Hip::HipAccelerator* hip_;
  std::vector<Tensor> p_;
  int64_t steps_ = 0;
  int32_t rows_ = 0;  // of the last Forward
  bool has_forward_ = false, has_gradient_ = false, stepped_ = false, quantized_ = false;
};

class FeedForwardBlock : public BlockParameters {
 public:
  // Which parameter: the norm's weight [width], W1 [hidden][width], b1 [hidden], W2 [width][hidden], b2 [width].
  enum Parameter { NormWeight, W1, B1, W2, B2 };
  static constexpr int kParameters = 5;

  // Weights start as zeros, the norm's as ones. ArgumentException unless both sizes are positive.
  FeedForwardBlock(int32_t width, int32_t hidden, Activation activation, IAccelerator& accelerator, float epsilon = 1e-6f);

  // ArgumentException when the length is not the parameter's.
  void Set(Parameter parameter, const std::vector<float>& values) { SetValues(parameter, values); }
  std::vector<float> Get(Parameter parameter) const { return Values(parameter); }
  // The gradient that the last Backward left, before and after a Step. InvalidOperationException before the first.
  std::vector<float> Gradient(Parameter parameter) const { return GradientOf(parameter); }

  // One row of x a token (x.Columns == Width, else ArgumentException). Products of bf16 values, sums in float32; what
  // Backward needs is kept; a Forward that throws past its check of x leaves nothing for a Backward.
  Matrix Forward(const Matrix& x);
  // The gradients of a loss by x (returned) and by the parameters (kept), from its gradient by Forward's result.
  // InvalidOperationException without a Forward since the last Set or Step, whose values were other ones; ArgumentException
  // unless dy has the shape of that Forward's result. A Backward that throws past these checks leaves no gradients.
  Matrix Backward(const Matrix& dy);
  // Forward for serving: products of 8-bit values with a scale per row of each operand. Keeps nothing.
  Matrix ForwardFp8(const Matrix& x);

 private:
  Activation activation_;
  Buffer<uint16_t> x_, normed_, pre_, active_;  // kept for Backward
  Buffer<uint8_t> q1_, q2_;                     // W1 and W2 in 8 bits, made from the current values when first asked for
  Buffer<float> s1_, s2_;
};

class GatedFeedForwardBlock : public BlockParameters {
 public:
  // Which parameter: the norm's weight and bias [width], Wg [hidden][width], bg [hidden], Wu [hidden][width], bu [hidden], Wd [width][hidden], bd [width].
  enum Parameter { NormWeight, NormBias, WGate, BGate, WUp, BUp, WDown, BDown };
  static constexpr int kParameters = 8;

  // Weights start as zeros, the norm's as ones. ArgumentException unless both sizes are positive.
  GatedFeedForwardBlock(int32_t width, int32_t hidden, Activation activation, IAccelerator& accelerator, float epsilon = 1e-5f);

  // As FeedForwardBlock's.
  void Set(Parameter parameter, const std::vector<float>& values) { SetValues(parameter, values); }
  std::vector<float> Get(Parameter parameter) const { return Values(parameter); }
  std::vector<float> Gradient(Parameter parameter) const { return GradientOf(parameter); }
  Matrix Forward(const Matrix& x);
  Matrix Backward(const Matrix& dy);
  // Forward for serving: products of 8-bit values with a scale for each 128 of a row of each operand. Keeps nothing.
  Matrix ForwardFp8(const Matrix& x);

 private:
  struct Codes {  // rows in 8 bits with block scales
    Buffer<uint8_t> q, scales;
  };
  Codes Quantize(const uint16_t* values, int64_t rows, int64_t cols) const;

  Activation activation_;
  Buffer<uint16_t> x_, normed_, gate_, up_, active_;  // kept for Backward
  Codes wg_, wu_, wd_;                                // made from the current values when first asked for
};

}  // namespace DotCompute::Algorithms
