// dc_linear_blocks.hip — matrix products of e4m3 values with a scale for each 128 of a row, for both operands: y = act(x w^T + bias) + residual.
//
// The scales are powers of two held as exponents, which v_mfma_scale_f32_*_f8f6f4 takes beside the codes, a byte for each row and 32 of c: a tile's turn
// is 128 bytes of c, one block, so that the scales cost a byte's load a row and turn, and no arithmetic. (A float32 scale would be a product and an
// addition for each sum and block, beside the matrix cores: 128 of them a lane and turn in the largest tiles, whose sums take half of the registers.)
// Everything else is a linear layer's (dc_linear.hip), what the 8-bit instructions cut products at (2^-13 of the largest that they add at once) among it: results in
// bf16 differ from those of float32 products by 0.0002 of themselves, in the mean, beside their rounding's 0.0017.
#include "dc_linear_device.hpp"

namespace {

typedef ProductOf<MoreOperands, Epilogue> BlocksProduct;

template <int TM, int TN, int WM, int WN, int KS>
int32_t launch_blocks(dc_hip_ctx* ctx, const BlocksProduct& p) {
  typename ProductTypes<false, false, true>::Jobs jobs{};
  auto& j = jobs.job[0];
  j.o = p.o, j.ep = p.ep;
  j.tiles_m = (p.o.m + TM - 1) / TM, j.tiles_n = (p.o.n + TN - 1) / TN;
  j.parts = (int32_t)p.plan.split.parts, j.turns = (int32_t)p.plan.split.turns;
  if (j.parts > 1) {  // the sums alone
    j.ep = Epilogue{};
    j.ep.y = p.parts(ctx), j.ep.y_stride = p.pitch(), j.ep.y_f32 = 1, j.ep.part_stride = p.o.m * p.pitch();
  }
  const int64_t total = (int64_t)j.tiles_m * j.tiles_n * j.parts;
  if (total > INT32_MAX / 2) return DC_ERR_UNSUPPORTED;
  jobs.ends[0] = (int32_t)total;
  return launch_jobs<TM, TN, WM, WN, KS, true, false, false, true>(ctx, jobs, total);
}

int32_t product(dc_hip_ctx* ctx, const BlocksProduct& p) {
  using dc::LinearTile;
  int32_t status = DC_ERR_INVALID_ARGUMENT;
  switch (p.plan.tile) {
    case LinearTile::k256: status = launch_blocks<256, 256, 2, 4, 1>(ctx, p); break;
    case LinearTile::k128: status = launch_blocks<128, 128, 2, 2, 1>(ctx, p); break;
    case LinearTile::k128x2: status = launch_blocks<128, 128, 2, 2, 2>(ctx, p); break;
    case LinearTile::k64: status = launch_blocks<64, 64, 2, 2, 1>(ctx, p); break;
    case LinearTile::k64x2: status = launch_blocks<64, 64, 2, 2, 2>(ctx, p); break;
    case LinearTile::k64x4: status = launch_blocks<64, 64, 2, 2, 4>(ctx, p); break;
  }
  if (status != DC_OK) return status;
  const Product sums{p.o, p.ep, p.plan};
  const Product* const one[] = {&sums};
  return join(ctx, one, 1);
}

// NB blocks of 16 outputs and XB blocks of 8 rows of x, W waves, and as many stages as fit in `kLds` KiB of LDS.
template <int XB, int NB, int W, int kLds>
int32_t launch_few_rows(dc_hip_ctx* ctx, const MoreOperands& o, const Epilogue& ep) {
  constexpr int kFit = kLds / W / (2 * NB + XB), kStages = kFit < 4 ? kFit : 4;
  const dim3 grid((unsigned)((o.n + 16 * NB - 1) / (16 * NB)), (unsigned)((o.m + 8 * XB - 1) / (8 * XB)));
  few_rows_kernel<true, XB, NB, W, kStages, false, true><<<grid, 64 * W, 0, ctx->stream>>>(o, ep);
  return dc::last_launch_status();
}

// 32 outputs to a workgroup where that leaves a workgroup for every other CU at least, so that x comes half as often with w through a CU's loads to LDS;
// with nine rows or more, eight waves of them in a CU's whole LDS, or, where there is more than one workgroup for a CU, four in half of it. us for 16 outputs / 32
// with eight waves / 32 with four: 1×4096×4096 6.33 / 5.93 / 6.44, 1×8192×4096 10.1 / 8.5 / 8.9; 17×4096×4096 6.85 / 6.37 / 7.15, 17×8192×4096 10.6 / 9.1 / 9.9,
// 17×16384×2048 9.9 / 10.1 / 8.5, 17×2048×8192 6.9 / 8.6 / 10.1; 32×8192×4096 11.2 / 9.7 / 10.1, 32×16384×2048 10.7 / 10.2 / 8.5. Past 32 rows eight waves of 16
// outputs: 64×4096×4096 8.4, four 9.1, 256×512×2048 4.8, 5.5.
template <int XB>
int32_t few_rows_of(dc_hip_ctx* ctx, const MoreOperands& o, const Epilogue& ep) {
  const int64_t cus = std::max(1, ctx->cu_count);
  if ((o.n + 15) / 16 < cus) return launch_few_rows<XB, 1, XB < 4 ? 8 : 4, 80>(ctx, o, ep);
  if constexpr (XB > 1)
    return (o.n + 31) / 32 > cus ? launch_few_rows<XB, 2, 4, 80>(ctx, o, ep) : launch_few_rows<XB, 2, 8, 160>(ctx, o, ep);
  else
    return launch_few_rows<XB, 2, 8, 80>(ctx, o, ep);
}
int32_t few_rows(dc_hip_ctx* ctx, const MoreOperands& o, const Epilogue& ep) {
  if (o.m <= 8) return few_rows_of<1>(ctx, o, ep);
  if (o.m <= 16) return few_rows_of<2>(ctx, o, ep);
  if (o.m <= 24) return few_rows_of<3>(ctx, o, ep);
  if (o.m <= 32) return few_rows_of<4>(ctx, o, ep);
  return launch_few_rows<8, 1, 8, 160>(ctx, o, ep);
}

}  // namespace

extern "C" {

DC_HIP_API int32_t dc_hip_linear_blocks(dc_hip_ctx* ctx, const dc_linear_blocks* args) {
  if (!args) return DC_ERR_INVALID_ARGUMENT;
  const dc_linear_blocks& p = *args;
  DC_RETURN_IF(check_dims(p.m, p.n, p.k, p.activation));
  const bool y_f32 = p.y_dtype == DC_DTYPE_F32;
  if (!y_f32 && p.y_dtype != DC_DTYPE_BF16) return DC_ERR_INVALID_ARGUMENT;
  if (p.m > 0 && p.n > 0) {
    if (p.k > 0) {
      DC_RETURN_IF(check_rows(p.x, 1, p.x_stride, p.m, p.k));
      DC_RETURN_IF(check_rows(p.w, 1, p.w_stride, p.n, p.k));
      DC_RETURN_IF(check_codes(p.x_scales, p.x_scales_stride, p.m, p.k));
      DC_RETURN_IF(check_codes(p.w_scales, p.w_scales_stride, p.n, p.k));
    }
    DC_RETURN_IF(check_rows(p.y, y_f32 ? 4 : 2, p.y_stride, p.m, p.n));
    if (p.residual) DC_RETURN_IF(check_rows(p.residual, 2, p.residual_stride, p.m, p.n));
    if (!aligned_to(p.bias, 2)) return DC_ERR_MISALIGNED;
  }
  DC_CTX_ENTER(ctx);
  if (p.m == 0 || p.n == 0) return DC_OK;
  Epilogue ep{};
  ep.bias = reinterpret_cast<const bf16*>(p.bias), ep.residual = reinterpret_cast<const bf16*>(p.residual), ep.residual_stride = p.residual_stride;
  ep.y = p.y, ep.y_stride = p.y_stride, ep.act = p.activation, ep.y_f32 = y_f32;
  MoreOperands o{};
  o.m = (int32_t)p.m, o.n = (int32_t)p.n, o.c_bytes = (int32_t)p.k;
  if (p.k == 0) {  // (bias, activation and residual alone)
    few_rows_any_kernel<true, 4, 2, 8, 2><<<dim3((unsigned)((o.n + 15) / 16), (unsigned)std::min((o.m + 31) / 32, 32768)), 512, 0, ctx->stream>>>(o, ep);
    return dc::last_launch_status();
  }
  o.a_codes = p.x_scales, o.a_codes_pitch = p.x_scales_stride, o.b_codes = p.w_scales, o.b_codes_pitch = p.w_scales_stride;
  Scratch scratch;
  Rows x{static_cast<const unsigned char*>(p.x), pitch_of(p.x_stride, p.m, p.k, 1), p.m, o.c_bytes};
  Rows w{static_cast<const unsigned char*>(p.w), pitch_of(p.w_stride, p.n, p.k, 1), p.n, o.c_bytes};
  x.plan(scratch);
  w.plan(scratch);
  const int64_t cus = std::max(1, ctx->cu_count);
  const bool few = dc::linear_few_rows(p.m, p.n, cus);
  const dc::LinearSize shape{p.m, p.n, o.c_bytes, x.width(), w.width()};
  const dc::LinearPlan best = few ? dc::LinearPlan{dc::LinearTile::k64, {1, 1}, 0.0} : dc::linear_plan(shape, {false, true}, cus);
  const ProductPlan plan(scratch, shape, best.tile, best.split);
  if (scratch.bytes) DC_RETURN_IF(dc::ensure_partials(ctx, scratch.bytes));
  DC_RETURN_IF(copy_rows(ctx, lay_out(ctx, &x, &w)));
  o.a = x.p, o.b = w.p, o.a_pitch = x.pitch, o.b_pitch = w.pitch;
  o.c_bytes = (int32_t)padded(o.c_bytes, 16);  // (ragged rows have been copied, with zeros there)
  return few ? few_rows(ctx, o, ep) : product(ctx, BlocksProduct{o, ep, plan});
}

}  // extern "C"
