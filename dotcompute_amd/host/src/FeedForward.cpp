// FeedForward.cpp — FeedForwardBlock on the HIP accelerator.
#include "DotCompute/FeedForward.hpp"

#include <cstring>

namespace DotCompute::Algorithms {

using Backends::Hip::Check;
using Backends::Hip::HipAccelerator;

namespace {
float Widen(uint16_t bits) {
  const uint32_t u = (uint32_t)bits << 16;
  float f;
  std::memcpy(&f, &u, sizeof f);
  return f;
}
std::vector<float> Widen(const std::vector<uint16_t>& bits) {
  std::vector<float> v(bits.size());
  for (size_t i = 0; i < bits.size(); ++i) v[i] = Widen(bits[i]);
  return v;
}
const char* const kShape = "FeedForwardBlock: expected a matrix of ";
std::string Shape(int64_t rows, int64_t cols) { return std::to_string(rows) + "x" + std::to_string(cols); }
}  // namespace

template <typename T>
FeedForwardBlock::Buffer<T> FeedForwardBlock::New(int64_t count) const {
  return hip_->Memory().AllocateAsync<T>((size_t)std::max<int64_t>(count, 1));
}

FeedForwardBlock::FeedForwardBlock(int32_t width, int32_t hidden, Activation activation, IAccelerator& accelerator, float epsilon)
    : width_(width), hidden_(hidden), activation_(activation), epsilon_(epsilon) {
  if (width <= 0 || hidden <= 0) throw ArgumentException("FeedForwardBlock: width and hidden must be positive");
  if (!(epsilon >= 0.0f)) throw ArgumentException("FeedForwardBlock: epsilon must not be negative");
  hip_ = dynamic_cast<HipAccelerator*>(&accelerator);
  if (!hip_)
    throw NotSupportedException("FeedForwardBlock runs on HIP accelerators only (got '" + accelerator.Info().DeviceType + "')");
  const int64_t shapes[kParameters][2] = {{1, width}, {hidden, width}, {1, hidden}, {width, hidden}, {1, width}};
  for (int i = 0; i < kParameters; ++i) {
    Tensor& t = p_[(size_t)i];
    t.rows = shapes[i][0], t.cols = shapes[i][1];
    const int64_t n = t.Size();
    t.value = New<float>(n), t.m = New<float>(n), t.v = New<float>(n), t.copy = New<uint16_t>(n);
    const bool matrix = i == W1 || i == W2;
    if (matrix) t.grad_b16 = New<uint16_t>(n);
    else t.grad_f32 = New<float>(n);
    for (auto* b : {&t.m, &t.v})
      Check(dc_hip_memset_async(hip_->Context(), (*b)->Data(), 0, (size_t)n * sizeof(float)), "FeedForwardBlock: states");
    Set((Parameter)i, std::vector<float>((size_t)n, i == NormWeight ? 1.0f : 0.0f));
  }
}

void FeedForwardBlock::Set(Parameter parameter, const std::vector<float>& values) {
  Tensor& t = p_.at((size_t)parameter);
  if ((int64_t)values.size() != t.Size())
    throw ArgumentException("FeedForwardBlock: a parameter of " + std::to_string(t.Size()) + " values was given " +
                            std::to_string(values.size()));
  has_forward_ = quantized_ = false;  // (both belong to the values before)
  t.value->CopyFromHost(values.data(), values.size() * sizeof(float));
  Check(dc_hip_convert_f32_to_bf16(hip_->Context(), t.value->Data(), t.copy->Data(), t.Size()), "FeedForwardBlock: convert");
}

std::vector<float> FeedForwardBlock::Get(Parameter parameter) const {
  const Tensor& t = p_.at((size_t)parameter);
  std::vector<float> v((size_t)t.Size());
  hip_->Synchronize();
  t.value->CopyToHost(v.data(), v.size() * sizeof(float));
  return v;
}

std::vector<float> FeedForwardBlock::Gradient(Parameter parameter) const {
  if (!has_gradient_) throw InvalidOperationException("FeedForwardBlock: no gradients yet");
  const Tensor& t = p_.at((size_t)parameter);
  hip_->Synchronize();
  if (t.grad_f32) {
    std::vector<float> v((size_t)t.Size());
    t.grad_f32->CopyToHost(v.data(), v.size() * sizeof(float));
    return v;
  }
  std::vector<uint16_t> bits((size_t)t.Size());
  t.grad_b16->CopyToHost(bits.data(), bits.size() * sizeof(uint16_t));
  return Widen(bits);
}

void FeedForwardBlock::RequireInput(const Matrix& x) const {
  if (x.Columns() != width_) throw ArgumentException(kShape + ("rows of " + std::to_string(width_)));
}

FeedForwardBlock::Buffer<uint16_t> FeedForwardBlock::ToBf16(const Matrix& x) const {
  auto wide = New<float>(x.Size());
  auto bits = New<uint16_t>(x.Size());
  if (x.Size() > 0) wide->CopyFromHost(x.Data().data(), (size_t)x.Size() * sizeof(float));
  Check(dc_hip_convert_f32_to_bf16(hip_->Context(), wide->Data(), bits->Data(), x.Size()), "FeedForwardBlock: convert");
  return bits;
}

Matrix FeedForwardBlock::Forward(const Matrix& x) {
  RequireInput(x);
  const int64_t rows = x.Rows(), d = width_, h = hidden_;
  has_forward_ = false;  // (until all of what Backward reads belongs to these rows)
  x_ = ToBf16(x);
  normed_ = New<uint16_t>(rows * d);
  pre_ = New<uint16_t>(rows * h);
  active_ = New<uint16_t>(rows * h);
  auto y = New<float>(rows * d);

  dc_rms_norm norm{};
  norm.rows = rows, norm.cols = d, norm.dtype = norm.y_dtype = DC_DTYPE_BF16, norm.eps = epsilon_;
  norm.x = x_->Data(), norm.weight = p_[NormWeight].copy->Data(), norm.y = normed_->Data();
  norm.x_stride = norm.y_stride = d;
  Check(dc_hip_rms_norm(hip_->Context(), &norm), "dc_hip_rms_norm");

  dc_linear up{};
  up.m = rows, up.n = h, up.k = d, up.dtype = up.y_dtype = DC_DTYPE_BF16, up.activation = (int32_t)activation_;
  up.x = normed_->Data(), up.w = p_[W1].copy->Data(), up.bias = p_[B1].copy->Data();
  up.pre = pre_->Data(), up.y = active_->Data();
  up.x_stride = up.w_stride = d, up.pre_stride = up.y_stride = h;
  Check(dc_hip_linear(hip_->Context(), &up), "dc_hip_linear");

  dc_linear down{};
  down.m = rows, down.n = d, down.k = h, down.dtype = DC_DTYPE_BF16, down.y_dtype = DC_DTYPE_F32;
  down.x = active_->Data(), down.w = p_[W2].copy->Data(), down.bias = p_[B2].copy->Data();
  down.residual = x_->Data(), down.y = y->Data();
  down.x_stride = down.w_stride = h, down.residual_stride = down.y_stride = d;
  Check(dc_hip_linear(hip_->Context(), &down), "dc_hip_linear");

  Matrix out(x.Rows(), width_);
  hip_->Synchronize();
  if (out.Size() > 0) y->CopyToHost(out.Data().data(), (size_t)out.Size() * sizeof(float));
  rows_ = x.Rows();
  has_forward_ = true;
  return out;
}

Matrix FeedForwardBlock::Backward(const Matrix& dy) {
  if (!has_forward_) throw InvalidOperationException("FeedForwardBlock: Backward follows a Forward with the current parameters");
  if (dy.Rows() != rows_ || dy.Columns() != width_) throw ArgumentException(kShape + Shape(rows_, width_));
  const int64_t rows = rows_, d = width_, h = hidden_;
  has_gradient_ = false;  // (until all of them are of this dy)
  auto g = ToBf16(dy);
  auto dactive = New<uint16_t>(rows * h);
  auto dnormed = New<uint16_t>(rows * d);
  auto dx = New<uint16_t>(rows * d);

  dc_linear_grad down{};
  down.m = rows, down.n = d, down.k = h;
  down.dy = g->Data(), down.x = active_->Data(), down.w = p_[W2].copy->Data();
  down.dx = dactive->Data(), down.dw = p_[W2].grad_b16->Data(), down.dbias = p_[B2].grad_f32->Data();
  down.dy_stride = d, down.x_stride = down.w_stride = down.dx_stride = down.dw_stride = h;
  Check(dc_hip_linear_backward(hip_->Context(), &down), "dc_hip_linear_backward");

  dc_linear_grad up{};
  up.m = rows, up.n = h, up.k = d, up.activation = (int32_t)activation_;
  up.dy = dactive->Data(), up.x = normed_->Data(), up.w = p_[W1].copy->Data(), up.pre = pre_->Data();
  up.dx = dnormed->Data(), up.dw = p_[W1].grad_b16->Data(), up.dbias = p_[B1].grad_f32->Data();
  up.dy_stride = up.pre_stride = h, up.x_stride = up.w_stride = up.dx_stride = up.dw_stride = d;
  Check(dc_hip_linear_backward(hip_->Context(), &up), "dc_hip_linear_backward");

  dc_rms_norm_grad norm{};
  norm.rows = rows, norm.cols = d, norm.dtype = DC_DTYPE_BF16, norm.eps = epsilon_;
  norm.dy = dnormed->Data(), norm.h = x_->Data(), norm.weight = p_[NormWeight].copy->Data();
  norm.dh = g->Data();  // what reaches x past the block
  norm.dx = dx->Data(), norm.dweight = p_[NormWeight].grad_f32->Data();
  norm.dy_stride = norm.h_stride = norm.dh_stride = norm.dx_stride = d;
  Check(dc_hip_rms_norm_backward(hip_->Context(), &norm), "dc_hip_rms_norm_backward");
  has_gradient_ = true;
  stepped_ = false;

  std::vector<uint16_t> bits((size_t)(rows * d));
  hip_->Synchronize();
  if (!bits.empty()) dx->CopyToHost(bits.data(), bits.size() * sizeof(uint16_t));
  return Matrix(rows_, width_, Widen(bits));
}

void FeedForwardBlock::Step(const AdamWOptions& options) {
  if (!has_gradient_ || stepped_) throw InvalidOperationException("FeedForwardBlock: Step follows Backward");
  dc_adamw args{};
  args.lr = options.LearningRate, args.beta1 = options.Beta1, args.beta2 = options.Beta2, args.eps = options.Epsilon;
  args.weight_decay = options.WeightDecay, args.grad_scale = 1.0, args.step = steps_ + 1, args.state_dtype = DC_DTYPE_F32;
  dc_adamw_tensor tensors[kParameters] = {};
  for (int i = 0; i < kParameters; ++i) {
    Tensor& t = p_[(size_t)i];
    dc_adamw_tensor& a = tensors[i];
    a.param = t.value->Data(), a.m = t.m->Data(), a.v = t.v->Data(), a.copy = t.copy->Data(), a.n = t.Size();
    a.grad = t.grad_f32 ? static_cast<const void*>(t.grad_f32->Data()) : t.grad_b16->Data();
    a.grad_dtype = t.grad_f32 ? DC_DTYPE_F32 : DC_DTYPE_BF16;
  }
  Check(dc_hip_adamw_step(hip_->Context(), &args, tensors, kParameters), "dc_hip_adamw_step");
  ++steps_;
  has_forward_ = quantized_ = false;
  stepped_ = true;
}

Matrix FeedForwardBlock::ForwardFp8(const Matrix& x) {
  RequireInput(x);
  const int64_t rows = x.Rows(), d = width_, h = hidden_;
  auto quantize = [&](Buffer<uint16_t>& from, int64_t r, int64_t c, Buffer<uint8_t>& q, Buffer<float>& s) {
    q = New<uint8_t>(r * c), s = New<float>(r);
    Check(dc_hip_quantize_fp8(hip_->Context(), from->Data(), DC_DTYPE_BF16, c, q->Data(), c, s->Data(), r, c), "dc_hip_quantize_fp8");
  };
  if (!quantized_) {
    quantize(p_[W1].copy, h, d, q1_, s1_);
    quantize(p_[W2].copy, d, h, q2_, s2_);
    quantized_ = true;
  }
  auto bits = ToBf16(x);
  auto q = New<uint8_t>(rows * d);
  auto scales = New<float>(rows);
  auto active = New<uint16_t>(rows * h);
  auto y = New<float>(rows * d);

  dc_rms_norm norm{};
  norm.rows = rows, norm.cols = d, norm.dtype = DC_DTYPE_BF16, norm.y_dtype = DC_DTYPE_FP8, norm.eps = epsilon_;
  norm.x = bits->Data(), norm.weight = p_[NormWeight].copy->Data(), norm.y = q->Data(), norm.scales = scales->Data();
  norm.x_stride = norm.y_stride = d;
  Check(dc_hip_rms_norm(hip_->Context(), &norm), "dc_hip_rms_norm");

  dc_linear up{};
  up.m = rows, up.n = h, up.k = d, up.dtype = DC_DTYPE_FP8, up.y_dtype = DC_DTYPE_BF16, up.activation = (int32_t)activation_;
  up.x = q->Data(), up.w = q1_->Data(), up.x_scales = scales->Data(), up.w_scales = s1_->Data();
  up.bias = p_[B1].copy->Data(), up.y = active->Data();
  up.x_stride = up.w_stride = d, up.y_stride = h;
  Check(dc_hip_linear(hip_->Context(), &up), "dc_hip_linear");

  Buffer<uint8_t> aq;
  Buffer<float> as;
  quantize(active, rows, h, aq, as);
  dc_linear down{};
  down.m = rows, down.n = d, down.k = h, down.dtype = DC_DTYPE_FP8, down.y_dtype = DC_DTYPE_F32;
  down.x = aq->Data(), down.w = q2_->Data(), down.x_scales = as->Data(), down.w_scales = s2_->Data();
  down.bias = p_[B2].copy->Data(), down.residual = bits->Data(), down.y = y->Data();
  down.x_stride = down.w_stride = h, down.residual_stride = down.y_stride = d;
  Check(dc_hip_linear(hip_->Context(), &down), "dc_hip_linear");

  Matrix out(x.Rows(), width_);
  hip_->Synchronize();
  if (out.Size() > 0) y->CopyToHost(out.Data().data(), (size_t)out.Size() * sizeof(float));
  return out;
}

}  // namespace DotCompute::Algorithms
