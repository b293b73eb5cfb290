// dc_gated.hip — both projections of a gated feed-forward block and their gate: y = act(x wg^T + bg) (x wu^T + bu), in one kernel.
//
// The products are those of the linear layers (dc_linear_device.hpp), with B's rows in LDS 32 of wg and 32 of wu in turn: a wave's neighbouring 32×32
// blocks are the two sums of the same outputs, and the epilogue's rows come back from LDS with both factors in one lane. So x is read once for both,
// and neither factor goes through memory unless the backward pass is to have it (`pre_gate`, `pre_up`).
//
// What is rounded: y, pre_gate and pre_up to their type once; y is formed from the unrounded factors. Sums are float32; of 8-bit operands as
// dc_linear.hip says. Block scales are powers of two, which the matrix instructions apply as they add.
#include "dc_linear_device.hpp"

namespace {

// Both factors from the sums over `count` parts of c (0: no sums at all), and the results: a lane takes eight neighbouring outputs.
struct GatedJoin {
  const float* parts;  // [count][m][2][pitch]
  int64_t m, n, pitch;
  int32_t count;
  GatedEpilogue ep;
};
__global__ __launch_bounds__(256) void gated_join_kernel(GatedJoin a) {
  const int64_t across = (a.n + 7) / 8, total = a.m * across, step = (int64_t)gridDim.x * 256;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += step) {
    const int64_t i = total <= UINT32_MAX ? (int64_t)((uint32_t)t / (uint32_t)across) : t / across, j = 8 * (t - i * across);
    GatedColumns<8> cols;
    cols.read(a.ep, j, a.n);
    f32x4 v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int32_t c = 0; c < a.count; ++c) {
      const float* from = a.parts + (c * a.m + i) * 2 * a.pitch + j;
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] += *reinterpret_cast<const f32x4*>(from + (q >> 1) * a.pitch + 4 * (q & 1));
    }
    float g[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
    float u[8] = {v[2].x, v[2].y, v[2].z, v[2].w, v[3].x, v[3].y, v[3].z, v[3].w};
    gated_finish(a.ep, cols, i, a.ep.a_scales ? a.ep.a_scales[i] : 1.0f, g, u);
  }
}

int32_t join_gated(dc_hip_ctx* ctx, const float* parts, const MoreOperands& o, int64_t pitch, int64_t count, const GatedEpilogue& ep) {
  const GatedJoin a{parts, o.m, o.n, pitch, (int32_t)count, ep};
  gated_join_kernel<<<(unsigned)dc::linear_join_groups(o.m, o.n), 256, 0, ctx->stream>>>(a);
  return dc::last_launch_status();
}

struct GatedProduct {
  MoreOperands o;
  GatedEpilogue ep;
  dc::LinearTile tile;
  dc::LinearSplit split;
  float* parts;
  int64_t pitch() const { return padded(o.n, 8); }
};

template <int TM, int TN, int WM, int WN, int KS, bool kFp8, bool kBlocks>
int32_t launch_gated(dc_hip_ctx* ctx, const GatedProduct& p) {
  typename ProductTypes<false, true, kBlocks>::Jobs jobs{};
  auto& j = jobs.job[0];
  j.o = p.o, j.ep = p.ep;
  j.tiles_m = (p.o.m + TM - 1) / TM, j.tiles_n = (p.o.n + TN / 2 - 1) / (TN / 2);
  j.parts = (int32_t)p.split.parts, j.turns = (int32_t)p.split.turns;
  if (j.parts > 1) {  // the sums alone
    j.ep = GatedEpilogue{};
    j.ep.y = p.parts, j.ep.y_stride = 2 * p.pitch(), j.ep.part_up = p.pitch(), j.ep.part_stride = p.o.m * 2 * p.pitch();
  }
  const int64_t total = (int64_t)j.tiles_m * j.tiles_n * j.parts;
  if (total > INT32_MAX / 2) return DC_ERR_UNSUPPORTED;
  jobs.ends[0] = (int32_t)total;
  return launch_jobs<TM, TN, WM, WN, KS, kFp8, false, true, kBlocks>(ctx, jobs, total);
}

// A wave has both sums of its outputs: at least 64 rows of B, so that the smallest tiles have two waves.
template <bool kFp8, bool kBlocks>
int32_t product(dc_hip_ctx* ctx, const GatedProduct& p) {
  using dc::LinearTile;
  int32_t status = DC_ERR_INVALID_ARGUMENT;
  switch (p.tile) {
    case LinearTile::k256: status = launch_gated<256, 256, 2, 4, 1, kFp8, kBlocks>(ctx, p); break;
    case LinearTile::k128: status = launch_gated<128, 128, 2, 2, 1, kFp8, kBlocks>(ctx, p); break;
    case LinearTile::k128x2: status = launch_gated<128, 128, 2, 2, 2, kFp8, kBlocks>(ctx, p); break;
    case LinearTile::k64: status = launch_gated<64, 64, 2, 1, 1, kFp8, kBlocks>(ctx, p); break;
    case LinearTile::k64x2: status = launch_gated<64, 64, 2, 1, 2, kFp8, kBlocks>(ctx, p); break;
    case LinearTile::k64x4: status = launch_gated<64, 64, 2, 1, 4, kFp8, kBlocks>(ctx, p); break;
  }
  if (status != DC_OK || p.split.parts == 1) return status;
  return join_gated(ctx, p.parts, p.o, p.pitch(), p.split.parts, p.ep);
}

// NB blocks of 16 rows of both weights together and XB blocks of 8 rows of x, W waves, and as many stages as fit in `kLds` KiB of LDS.
template <bool kFp8, bool kBlocks, int XB, int NB, int W, int kLds>
int32_t launch_few_rows(dc_hip_ctx* ctx, const MoreOperands& o, const GatedEpilogue& ep) {
  constexpr int kFit = kLds / W / (2 * NB + XB), kStages = kFit < 4 ? kFit : 4;
  static_assert(kStages >= 2, "a step in flight beside the one that is read");
  const dim3 grid((unsigned)((o.n + 8 * NB - 1) / (8 * NB)), (unsigned)((o.m + 8 * XB - 1) / (8 * XB)));
  // (us, the weights' bytes kept by the caches / not, each call over one of three sets in turn: bf16 1×8192×4096 25.6 / 23.7, 8×8192×4096 25.9 / 23.2,
  // 1×14336×4096 41.3 / 38.8; of 67 MB 1×8192×2048 11.8–12.7 / 12.7. Where more than one row of workgroups reads them, they are kept.)
  const bool once = grid.y == 1 && dc::read_once(o.n, o.c_bytes, 2);
  auto* kernel = once ? few_rows_kernel<kFp8, XB, NB, W, kStages, true, kBlocks, true> : few_rows_kernel<kFp8, XB, NB, W, kStages, true, kBlocks, false>;
  kernel<<<grid, 64 * W, 0, ctx->stream>>>(o, ep);
  return dc::last_launch_status();
}

template <bool kFp8, bool kBlocks>
int32_t few_rows(dc_hip_ctx* ctx, const MoreOperands& o, const GatedEpilogue& ep) {
  if (o.m <= 8) return launch_few_rows<kFp8, kBlocks, 1, 2, 8, 80>(ctx, o, ep);
  if (o.m <= 16) return launch_few_rows<kFp8, kBlocks, 2, 2, 4, 80>(ctx, o, ep);
  if (o.m <= 24) return launch_few_rows<kFp8, kBlocks, 3, 2, 4, 80>(ctx, o, ep);
  if (o.m <= 32) return launch_few_rows<kFp8, kBlocks, 4, 2, 4, 80>(ctx, o, ep);
  return launch_few_rows<kFp8, kBlocks, 8, 2, 4, 160>(ctx, o, ep);
}

}  // namespace

extern "C" {

DC_HIP_API int32_t dc_hip_gated_linear(dc_hip_ctx* ctx, const dc_gated_linear* args) {
  if (!args) return DC_ERR_INVALID_ARGUMENT;
  const dc_gated_linear& p = *args;
  DC_RETURN_IF(check_dims(p.m, p.n, p.k, p.activation));
  if (p.n > dc::kGatedWidth) return DC_ERR_UNSUPPORTED;
  const bool fp8 = p.dtype == DC_DTYPE_FP8, y_f32 = p.y_dtype == DC_DTYPE_F32, blocks = p.scale_block == DC_SCALE_BLOCK;
  if ((!fp8 && p.dtype != DC_DTYPE_BF16) || (!y_f32 && p.y_dtype != DC_DTYPE_BF16)) return DC_ERR_INVALID_ARGUMENT;
  if (p.scale_block != 0 && !(fp8 && blocks)) return DC_ERR_INVALID_ARGUMENT;
  for (const void* scales : {p.x_scales, p.gate_scales, p.up_scales})
    if (fp8 ? !scales && !(blocks && p.k == 0) : scales != nullptr) return DC_ERR_INVALID_ARGUMENT;
  const int64_t size = fp8 ? 1 : 2;
  if (p.m > 0 && p.n > 0) {
    if (p.k > 0) {
      DC_RETURN_IF(check_rows(p.x, size, p.x_stride, p.m, p.k));
      DC_RETURN_IF(check_rows(p.w_gate, size, p.w_gate_stride, p.n, p.k));
      DC_RETURN_IF(check_rows(p.w_up, size, p.w_up_stride, p.n, p.k));
      if (blocks) {
        DC_RETURN_IF(check_codes(p.x_scales, p.x_scales_stride, p.m, p.k));
        DC_RETURN_IF(check_codes(p.gate_scales, p.gate_scales_stride, p.n, p.k));
        DC_RETURN_IF(check_codes(p.up_scales, p.up_scales_stride, p.n, p.k));
      }
    }
    DC_RETURN_IF(check_rows(p.y, y_f32 ? 4 : 2, p.y_stride, p.m, p.n));
    if (p.pre_gate) DC_RETURN_IF(check_rows(p.pre_gate, 2, p.pre_gate_stride, p.m, p.n));
    if (p.pre_up) DC_RETURN_IF(check_rows(p.pre_up, 2, p.pre_up_stride, p.m, p.n));
    if (!aligned_to(p.bias_gate, 2) || !aligned_to(p.bias_up, 2)) return DC_ERR_MISALIGNED;
    if (!blocks && (!aligned_to(p.x_scales, 4) || !aligned_to(p.gate_scales, 4) || !aligned_to(p.up_scales, 4))) return DC_ERR_MISALIGNED;
  }
  DC_CTX_ENTER(ctx);
  if (p.m == 0 || p.n == 0) return DC_OK;
  GatedEpilogue ep{};
  if (!blocks) {
    ep.a_scales = static_cast<const float*>(p.x_scales);
    ep.b_scales = static_cast<const float*>(p.gate_scales);
    ep.b2_scales = static_cast<const float*>(p.up_scales);
  }
  ep.bias = reinterpret_cast<const bf16*>(p.bias_gate), ep.bias2 = reinterpret_cast<const bf16*>(p.bias_up);
  ep.pre = reinterpret_cast<bf16*>(p.pre_gate), ep.pre2 = reinterpret_cast<bf16*>(p.pre_up);
  ep.pre_stride = p.pre_gate_stride, ep.pre2_stride = p.pre_up_stride;
  ep.y = p.y, ep.y_stride = p.y_stride, ep.act = p.activation, ep.y_f32 = y_f32;
  MoreOperands o{};
  o.m = (int32_t)p.m, o.n = (int32_t)p.n, o.c_bytes = (int32_t)(p.k * size);
  if (blocks) {
    o.a_codes = static_cast<const uint8_t*>(p.x_scales), o.a_codes_pitch = p.x_scales_stride;
    o.b_codes = static_cast<const uint8_t*>(p.gate_scales), o.b_codes_pitch = p.gate_scales_stride;
    o.b2_codes = static_cast<const uint8_t*>(p.up_scales), o.b2_codes_pitch = p.up_scales_stride;
  }
  if (p.k == 0) return join_gated(ctx, nullptr, o, 0, 0, ep);
  Scratch scratch;
  Rows x{static_cast<const unsigned char*>(p.x), pitch_of(p.x_stride, p.m, p.k, size), p.m, o.c_bytes};
  Rows gate{static_cast<const unsigned char*>(p.w_gate), pitch_of(p.w_gate_stride, p.n, p.k, size), p.n, o.c_bytes};
  Rows up{static_cast<const unsigned char*>(p.w_up), pitch_of(p.w_up_stride, p.n, p.k, size), p.n, o.c_bytes};
  for (Rows* r : {&x, &gate, &up}) r->plan(scratch);
  const int64_t cus = std::max(1, ctx->cu_count);
  // (A workgroup of that kernel has 16 outputs here too. Against the tiles, 45 shapes of 33 to 1024 rows: up to a workgroup for each CU 0.66 to 0.99 of their time,
  // but 1.19 of 565×224×6448; beyond that 1.15 to 1.53.)
  const bool few = dc::linear_few_rows(p.m, p.n, cus);
  GatedProduct all{o, ep, dc::LinearTile::k64, {1, 1}, nullptr};
  size_t at_parts = 0;
  if (!few) {
    const dc::LinearSize shape{p.m, 2 * p.n, o.c_bytes, x.width(), std::max(gate.width(), up.width())};
    const dc::LinearPlan best = dc::linear_plan(shape, {false, fp8}, cus);
    all.tile = best.tile, all.split = best.split;
    if (best.split.parts > 1) at_parts = scratch.take(best.split.parts * p.m * 2 * all.pitch() * (int64_t)sizeof(float));
  }
  if (scratch.bytes) DC_RETURN_IF(dc::ensure_partials(ctx, scratch.bytes));
  DC_RETURN_IF(copy_rows(ctx, lay_out(ctx, &x, &gate, &up)));
  o.a = x.p, o.b = gate.p, o.b2 = up.p, o.a_pitch = x.pitch, o.b_pitch = gate.pitch, o.b2_pitch = up.pitch;
  o.c_bytes = (int32_t)padded(o.c_bytes, 16);  // (ragged rows have been copied, with zeros there)
  if (few) return !fp8 ? few_rows<false, false>(ctx, o, ep) : blocks ? few_rows<true, true>(ctx, o, ep) : few_rows<true, false>(ctx, o, ep);
  all.o = o;
  all.parts = reinterpret_cast<float*>(static_cast<unsigned char*>(ctx->partials) + at_parts);
  return !fp8 ? product<false, false>(ctx, all) : blocks ? product<true, true>(ctx, all) : product<true, false>(ctx, all);
}

}  // extern "C"
