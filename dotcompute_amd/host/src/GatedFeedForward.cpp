// GatedFeedForward.cpp — GatedFeedForwardBlock on the HIP accelerator.
#include "DotCompute/FeedForward.hpp"

namespace DotCompute::Algorithms {

using Backends::Hip::Check;

GatedFeedForwardBlock::GatedFeedForwardBlock(int32_t width, int32_t hidden, Activation activation, IAccelerator& accelerator, float epsilon)
    : BlockParameters("GatedFeedForwardBlock", width, hidden, accelerator, epsilon), activation_(activation) {
  Allocate({{false, 1, width, 1.0f},
            {false, 1, width, 0.0f},
            {true, hidden, width, 0.0f},
            {false, 1, hidden, 0.0f},
            {true, hidden, width, 0.0f},
            {false, 1, hidden, 0.0f},
            {true, width, hidden, 0.0f},
            {false, 1, width, 0.0f}});
}

Matrix GatedFeedForwardBlock::Forward(const Matrix& x) {
  RequireInput(x);
  const int64_t rows = x.Rows(), d = width_, h = hidden_;
  has_forward_ = false;  // (until all of what Backward reads belongs to these rows)
  x_ = ToBf16(x);
  normed_ = New<uint16_t>(rows * d);
  gate_ = New<uint16_t>(rows * h);
  up_ = New<uint16_t>(rows * h);
  active_ = New<uint16_t>(rows * h);
  auto y = New<float>(rows * d);

  dc_layer_norm norm{};
  norm.rows = rows, norm.cols = d, norm.dtype = norm.y_dtype = DC_DTYPE_BF16, norm.eps = epsilon_;
  norm.x = x_->Data(), norm.weight = Copy(NormWeight), norm.bias = Copy(NormBias), norm.y = normed_->Data();
  norm.x_stride = norm.y_stride = d;
  Check(dc_hip_layer_norm(hip_->Context(), &norm), "dc_hip_layer_norm");

  dc_gated_linear both{};
  both.m = rows, both.n = h, both.k = d, both.dtype = both.y_dtype = DC_DTYPE_BF16, both.activation = (int32_t)activation_;
  both.x = normed_->Data(), both.w_gate = Copy(WGate), both.w_up = Copy(WUp), both.bias_gate = Copy(BGate), both.bias_up = Copy(BUp);
  both.pre_gate = gate_->Data(), both.pre_up = up_->Data(), both.y = active_->Data();
  both.x_stride = both.w_gate_stride = both.w_up_stride = d, both.pre_gate_stride = both.pre_up_stride = both.y_stride = h;
  Check(dc_hip_gated_linear(hip_->Context(), &both), "dc_hip_gated_linear");

  dc_linear down{};
  down.m = rows, down.n = d, down.k = h, down.dtype = DC_DTYPE_BF16, down.y_dtype = DC_DTYPE_F32;
  down.x = active_->Data(), down.w = Copy(WDown), down.bias = Copy(BDown), down.residual = x_->Data(), down.y = y->Data();
  down.x_stride = down.w_stride = h, down.residual_stride = down.y_stride = d;
  Check(dc_hip_linear(hip_->Context(), &down), "dc_hip_linear");

  Matrix out = Result(y, x.Rows());
  rows_ = x.Rows();
  has_forward_ = true;
  return out;
}

Matrix GatedFeedForwardBlock::Backward(const Matrix& dy) {
  RequireBackward(dy);
  const int64_t rows = rows_, d = width_, h = hidden_;
  has_gradient_ = false;  // (until all of them are of this dy)
  auto g = ToBf16(dy);
  auto dactive = New<uint16_t>(rows * h);
  auto dnormed = New<uint16_t>(rows * d);
  auto dx = New<uint16_t>(rows * d);
  auto b16 = [&](Parameter p) { return p_[p].grad_b16->Data(); };
  auto f32 = [&](Parameter p) { return p_[p].grad_f32->Data(); };

  dc_linear_grad down{};
  down.m = rows, down.n = d, down.k = h;
  down.dy = g->Data(), down.x = active_->Data(), down.w = Copy(WDown);
  down.dx = dactive->Data(), down.dw = b16(WDown), down.dbias = f32(BDown);
  down.dy_stride = d, down.x_stride = down.w_stride = down.dx_stride = down.dw_stride = h;
  Check(dc_hip_linear_backward(hip_->Context(), &down), "dc_hip_linear_backward");

  dc_gated_linear_grad both{};
  both.m = rows, both.n = h, both.k = d, both.activation = (int32_t)activation_;
  both.dy = dactive->Data(), both.x = normed_->Data(), both.w_gate = Copy(WGate), both.w_up = Copy(WUp);
  both.pre_gate = gate_->Data(), both.pre_up = up_->Data();
  both.dx = dnormed->Data(), both.dw_gate = b16(WGate), both.dw_up = b16(WUp), both.dbias_gate = f32(BGate), both.dbias_up = f32(BUp);
  both.dy_stride = both.pre_gate_stride = both.pre_up_stride = h;
  both.x_stride = both.w_gate_stride = both.w_up_stride = both.dx_stride = both.dw_gate_stride = both.dw_up_stride = d;
  Check(dc_hip_gated_linear_backward(hip_->Context(), &both), "dc_hip_gated_linear_backward");

  dc_layer_norm_grad norm{};
  norm.rows = rows, norm.cols = d, norm.dtype = DC_DTYPE_BF16, norm.eps = epsilon_;
  norm.dy = dnormed->Data(), norm.h = x_->Data(), norm.weight = Copy(NormWeight);
  norm.dh = g->Data();  // what reaches x past the block
  norm.dx = dx->Data(), norm.dweight = f32(NormWeight), norm.dbias = f32(NormBias);
  norm.dy_stride = norm.h_stride = norm.dh_stride = norm.dx_stride = d;
  Check(dc_hip_layer_norm_backward(hip_->Context(), &norm), "dc_hip_layer_norm_backward");
  has_gradient_ = true;
  stepped_ = false;
  return Result(dx, rows_);
}

GatedFeedForwardBlock::Codes GatedFeedForwardBlock::Quantize(const uint16_t* values, int64_t rows, int64_t cols) const {
  const int64_t blocks = (cols + DC_SCALE_BLOCK - 1) / DC_SCALE_BLOCK;
  Codes c{New<uint8_t>(rows * cols), New<uint8_t>(rows * blocks)};
  Check(dc_hip_quantize_fp8_blocks(hip_->Context(), values, DC_DTYPE_BF16, cols, c.q->Data(), cols, c.scales->Data(), rows, rows, cols),
        "dc_hip_quantize_fp8_blocks");
  return c;
}

Matrix GatedFeedForwardBlock::ForwardFp8(const Matrix& x) {
  RequireInput(x);
  const int64_t rows = x.Rows(), d = width_, h = hidden_;
  if (!quantized_) {
    wg_ = Quantize(Copy(WGate), h, d);
    wu_ = Quantize(Copy(WUp), h, d);
    wd_ = Quantize(Copy(WDown), d, h);
    quantized_ = true;
  }
  auto bits = ToBf16(x);
  const int64_t blocks = (d + DC_SCALE_BLOCK - 1) / DC_SCALE_BLOCK;
  const Codes normed{New<uint8_t>(rows * d), New<uint8_t>(rows * blocks)};
  auto active = New<uint16_t>(rows * h);
  auto y = New<float>(rows * d);

  dc_layer_norm norm{};
  norm.rows = rows, norm.cols = d, norm.dtype = DC_DTYPE_BF16, norm.y_dtype = DC_DTYPE_FP8, norm.eps = epsilon_, norm.scale_block = DC_SCALE_BLOCK;
  norm.x = bits->Data(), norm.weight = Copy(NormWeight), norm.bias = Copy(NormBias), norm.y = normed.q->Data(), norm.scales = normed.scales->Data();
  norm.x_stride = norm.y_stride = d, norm.scales_stride = rows;
  Check(dc_hip_layer_norm(hip_->Context(), &norm), "dc_hip_layer_norm");

  dc_gated_linear both{};
  both.m = rows, both.n = h, both.k = d, both.dtype = DC_DTYPE_FP8, both.y_dtype = DC_DTYPE_BF16, both.activation = (int32_t)activation_;
  both.scale_block = DC_SCALE_BLOCK;
  both.x = normed.q->Data(), both.w_gate = wg_.q->Data(), both.w_up = wu_.q->Data();
  both.x_scales = normed.scales->Data(), both.gate_scales = wg_.scales->Data(), both.up_scales = wu_.scales->Data();
  both.bias_gate = Copy(BGate), both.bias_up = Copy(BUp), both.y = active->Data();
  both.x_stride = both.w_gate_stride = both.w_up_stride = d, both.y_stride = h;
  both.x_scales_stride = rows, both.gate_scales_stride = both.up_scales_stride = h;
  Check(dc_hip_gated_linear(hip_->Context(), &both), "dc_hip_gated_linear");

  const Codes a = Quantize(active->Data(), rows, h);
  dc_linear_blocks down{};
  down.m = rows, down.n = d, down.k = h, down.y_dtype = DC_DTYPE_F32;
  down.x = a.q->Data(), down.w = wd_.q->Data(), down.x_scales = a.scales->Data(), down.w_scales = wd_.scales->Data();
  down.bias = Copy(BDown), down.residual = bits->Data(), down.y = y->Data();
  down.x_stride = down.w_stride = h, down.x_scales_stride = rows, down.w_scales_stride = d, down.residual_stride = down.y_stride = d;
  Check(dc_hip_linear_blocks(hip_->Context(), &down), "dc_hip_linear_blocks");
  return Result(y, x.Rows());
}

}  // namespace DotCompute::Algorithms
