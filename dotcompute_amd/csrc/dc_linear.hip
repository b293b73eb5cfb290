// dc_linear.hip — matrix products with bias, activation and residual in their epilogue, and their gradients.
//
// Forward: z = x w^T (x_scales w_scales) + bias, y = act(z) + residual, with x [m][k] and w [n][k] in bf16 or e4m3 and
// sums in fp32. Backward: dz = dy act'(pre); dx = dz w, dw = dz^T x, dbias = column sums of dz.
//
// Kernels:
//   - product_kernel: D[i][j] = sum_c A(i, c) B(j, c) in tiles on the matrix cores. A's rows run along c. B's do too
//     (forward), or are the rows c of a row-major [c][j] matrix (the gradients, both in one launch).
//   - join_kernel: the results from the sums over parts of c, where few tiles have long sums.
//   - few_rows_kernel, few_rows_any_kernel: forward with few rows of x, or so few results that 64 rows and 16 outputs of them to a
//     workgroup leave no CU two.
//   - slope_kernel: dz and its transpose in bf16 (what the two gradients' products run along), and dbias's parts.
//   - pack_kernel: rows that the direct-to-LDS loads cannot take (not 16-byte aligned, or no whole number of
//     16 bytes) copied to ones padded with zeros.
//
// What is rounded: results to their type once, from float32 sums; `pre` to bf16 from the z that the activation also takes
// unrounded; dz to bf16, as the matrix cores take no float32 at a useful rate (dbias adds it unrounded). The 8-bit matrix instructions
// add 64 or 128 products at a time and cut each at 2^-13 of the largest of a lane's share of them (measured with pairs of powers of
// two; sums of whole numbers are exact): far less than the 2^-4 by which rounding to e4m3 may have moved each operand, so
// their full rate is taken. Their sums are float32 from there on.
#include "dc_linear_device.hpp"

namespace {

// ---- what the gradients' products run along ---------------------------------------------------------------
// dz = dy act'(pre) over 64×64 pieces: dz itself (pitch dz_pitch, columns from n to there zero), its transpose (pitch
// t_pitch, columns from m to there zero) through LDS, and the piece's column sums, unrounded. A thread holds two
// neighbouring rows of 8 columns, so the transpose's LDS words are pairs of rows. Bound by memory: 8192×8192 with silu, dz, its
// transpose and parts 98-103 us (537 MB, 5.2-5.5 TB/s); 2000×3000 with gelu 13.6, half of it the slope's arithmetic. (All four
// loads in flight at once, by addresses that need no branch: 13.2 for 12.2 without the writes, 2000×3000.)
struct SlopeArgs {
  const bf16 *dy, *pre;
  bf16 *dz, *dzt;  // either may be NULL
  float* parts;    // [pieces of rows][n], or NULL
  int64_t m, n, dy_stride, pre_stride, dz_pitch, t_pitch;
  int32_t act;
};
// (The workgroups with blockIdx.y > 0 copy the operands that have to be, beside it.)
__global__ __launch_bounds__(256) void slope_kernel(SlopeArgs a, PackArgs copies) {
  __shared__ uint32_t turned[64][33];
  __shared__ float sums[32][65];
  if (blockIdx.y > 0) return pack_rows(copies.job[blockIdx.y - 1], blockIdx.x, gridDim.x);
  const int t = threadIdx.x, c8 = t & 7, pair = t >> 3;
  const int64_t across = (a.n + 63) / 64, total = across * ((a.m + 63) / 64);
  for (int64_t at = blockIdx.x; at < total; at += gridDim.x) {
    const int64_t down = total <= UINT32_MAX ? (int64_t)((uint32_t)at / (uint32_t)across) : at / across;
    const int64_t m0 = down * 64, n0 = (at - down * across) * 64;
    const int64_t j = n0 + 8 * c8;
    float dz[2][8];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int64_t i = m0 + 2 * pair + q;
      if (i < a.m && j < a.n) {
        dc::load_some(a.dy + i * a.dy_stride + j, a.n - j, dz[q]);
        if (a.act != DC_ACT_NONE) {
          float z[8];
          dc::load_some(a.pre + i * a.pre_stride + j, a.n - j, z);  // (zeros past the last: their dz stays zero)
          apply_slope(a.act, z, dz[q]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) dz[q][e] = 0.0f;
      }
      if (a.dz && i < a.m && j < a.dz_pitch) dc::store_chunk(a.dz + i * a.dz_pitch + j, dz[q]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      turned[8 * c8 + e][pair] = dc::pack_bf16(dz[0][e], dz[1][e]);
      sums[pair][8 * c8 + e] = dz[0][e] + dz[1][e];
    }
    __syncthreads();
    if (a.dzt) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {  // 64 rows of 8 16-byte chunks
        const int row = (t >> 3) + 32 * q, chunk = t & 7;
        const int64_t c = m0 + 8 * chunk;
        if (n0 + row < a.n && c < a.t_pitch) {
          const dc::u32x4 w = {turned[row][4 * chunk], turned[row][4 * chunk + 1], turned[row][4 * chunk + 2],
                               turned[row][4 * chunk + 3]};
          *reinterpret_cast<dc::u32x4*>(a.dzt + (n0 + row) * a.t_pitch + c) = w;
        }
      }
    }
    if (a.parts && t < 64 && n0 + t < a.n) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < 32; ++i) s += sums[i][t];
      a.parts[m0 / 64 * a.n + n0 + t] = s;
    }
    __syncthreads();
  }
}

// ---- host ------------------------------------------------------------------------------------------------
template <bool kRowsC>
constexpr int kJobs = ProductTypes<kRowsC, false, false>::kJobs;

template <int TM, int TN, int WM, int WN, int KS, bool kFp8, bool kRowsC>
int32_t launch_products(dc_hip_ctx* ctx, const Product* const (&p)[kJobs<kRowsC>], const ColumnParts& columns) {
  typename ProductTypes<kRowsC, false, false>::Jobs jobs{};
  int64_t total = 0;
  for (int i = 0; i < kJobs<kRowsC>; ++i) {
    jobs.ends[i] = (int32_t)total;
    if (!p[i]) continue;
    auto& j = jobs.job[i];
    j.o = p[i]->o, j.ep = p[i]->ep;
    j.tiles_m = (j.o.m + TM - 1) / TM, j.tiles_n = (j.o.n + TN - 1) / TN;
    j.parts = (int32_t)p[i]->plan.split.parts, j.turns = (int32_t)p[i]->plan.split.turns;
    if (j.parts > 1) {  // the sums alone
      j.ep = Epilogue{};
      j.ep.y = p[i]->parts(ctx), j.ep.y_stride = p[i]->pitch(), j.ep.y_f32 = 1, j.ep.part_stride = j.o.m * p[i]->pitch();
    }
    total += (int64_t)j.tiles_m * j.tiles_n * j.parts;
    if (total > INT32_MAX / 2) return DC_ERR_UNSUPPORTED;
    jobs.ends[i] = (int32_t)total;
  }
  jobs.columns = columns;
  return launch_jobs<TM, TN, WM, WN, KS, kFp8, kRowsC, false, false>(ctx, jobs, total);
}

// Products of one tile.
template <bool kFp8, bool kRowsC>
int32_t products(dc_hip_ctx* ctx, const Product* const (&p)[kJobs<kRowsC>], const ColumnParts& columns = {}) {
  using dc::LinearTile;
  int32_t status = DC_ERR_INVALID_ARGUMENT;
  switch (p[0]->plan.tile) {
    case LinearTile::k256: status = launch_products<256, 256, 2, 4, 1, kFp8, kRowsC>(ctx, p, columns); break;
    case LinearTile::k128: status = launch_products<128, 128, 2, 2, 1, kFp8, kRowsC>(ctx, p, columns); break;
    case LinearTile::k128x2: status = launch_products<128, 128, 2, 2, 2, kFp8, kRowsC>(ctx, p, columns); break;
    case LinearTile::k64: status = launch_products<64, 64, 2, 2, 1, kFp8, kRowsC>(ctx, p, columns); break;
    case LinearTile::k64x2: status = launch_products<64, 64, 2, 2, 2, kFp8, kRowsC>(ctx, p, columns); break;
    case LinearTile::k64x4: status = launch_products<64, 64, 2, 2, 4, kFp8, kRowsC>(ctx, p, columns); break;
  }
  return status == DC_OK ? join(ctx, p, kJobs<kRowsC>) : status;
}

// NB blocks of 16 outputs and XB blocks of 8 rows of x, W waves, and as many stages as fit in `kLds` KiB of LDS.
template <bool kFp8, int XB, int NB, int W, int kLds>
int32_t launch_few_rows(dc_hip_ctx* ctx, const Operands& o, const Epilogue& ep) {
  constexpr int kFit = kLds / W / (2 * NB + XB), kStages = kFit < 4 ? kFit : 4;
  const dim3 grid((unsigned)((o.n + 16 * NB - 1) / (16 * NB)), (unsigned)((o.m + 8 * XB - 1) / (8 * XB)));
  few_rows_kernel<kFp8, XB, NB, W, kStages, false, false><<<grid, 64 * W, 0, ctx->stream>>>(o, ep);
  return dc::last_launch_status();
}

template <bool kFp8>
int32_t few_rows(dc_hip_ctx* ctx, const Operands& o, const Epilogue& ep) {
  const bool wide = dc::linear_wide_few_rows(o.m, o.n, std::max(1, ctx->cu_count));
  if (o.m <= 8) return wide ? launch_few_rows<kFp8, 1, 4, 4, 80>(ctx, o, ep) : launch_few_rows<kFp8, 1, 1, 8, 80>(ctx, o, ep);
  if (o.m <= 16) return wide ? launch_few_rows<kFp8, 2, 4, 4, 80>(ctx, o, ep) : launch_few_rows<kFp8, 2, 1, 8, 80>(ctx, o, ep);
  if (o.m <= 24) return wide ? launch_few_rows<kFp8, 3, 4, 4, 160>(ctx, o, ep) : launch_few_rows<kFp8, 3, 1, 8, 80>(ctx, o, ep);
  if (o.m <= 32) return wide ? launch_few_rows<kFp8, 4, 4, 4, 160>(ctx, o, ep) : launch_few_rows<kFp8, 4, 1, 4, 80>(ctx, o, ep);
  return launch_few_rows<kFp8, 8, 1, 4, 80>(ctx, o, ep);
}

template <bool kFp8, int MT>
int32_t launch_few_rows_any(dc_hip_ctx* ctx, const Operands& o, const Epilogue& ep) {
  const dim3 grid((unsigned)((o.n + 15) / 16), (unsigned)std::min((o.m + 8 * MT - 1) / (8 * MT), 32768));
  few_rows_any_kernel<kFp8, MT, 2, 8, 2><<<grid, 512, 0, ctx->stream>>>(o, ep);
  return dc::last_launch_status();
}

template <bool kFp8>
int32_t few_rows_any(dc_hip_ctx* ctx, const Operands& o, const Epilogue& ep) {
  if (o.m <= 8) return launch_few_rows_any<kFp8, 1>(ctx, o, ep);
  if (o.m <= 16) return launch_few_rows_any<kFp8, 2>(ctx, o, ep);
  return launch_few_rows_any<kFp8, 4>(ctx, o, ep);
}

}  // namespace

extern "C" {

DC_HIP_API int32_t dc_hip_linear(dc_hip_ctx* ctx, const dc_linear* args) {
  if (!args) return DC_ERR_INVALID_ARGUMENT;
  const dc_linear& p = *args;
  DC_RETURN_IF(check_dims(p.m, p.n, p.k, p.activation));
  const bool fp8 = p.dtype == DC_DTYPE_FP8, y_f32 = p.y_dtype == DC_DTYPE_F32;
  if ((!fp8 && p.dtype != DC_DTYPE_BF16) || (!y_f32 && p.y_dtype != DC_DTYPE_BF16) || p.reserved != 0)
    return DC_ERR_INVALID_ARGUMENT;
  if (fp8 != (p.x_scales != nullptr) || fp8 != (p.w_scales != nullptr)) return DC_ERR_INVALID_ARGUMENT;
  const int64_t size = fp8 ? 1 : 2;
  if (p.m > 0 && p.n > 0) {
    if (p.k > 0) {
      DC_RETURN_IF(check_rows(p.x, size, p.x_stride, p.m, p.k));
      DC_RETURN_IF(check_rows(p.w, size, p.w_stride, p.n, p.k));
    }
    DC_RETURN_IF(check_rows(p.y, y_f32 ? 4 : 2, p.y_stride, p.m, p.n));
    if (p.residual) DC_RETURN_IF(check_rows(p.residual, 2, p.residual_stride, p.m, p.n));
    if (p.pre) DC_RETURN_IF(check_rows(p.pre, 2, p.pre_stride, p.m, p.n));
    if (!aligned_to(p.bias, 2) || !aligned_to(p.x_scales, 4) || !aligned_to(p.w_scales, 4)) return DC_ERR_MISALIGNED;
  }
  DC_CTX_ENTER(ctx);
  if (p.m == 0 || p.n == 0) return DC_OK;
  const Epilogue ep{p.x_scales,
                    p.w_scales,
                    reinterpret_cast<const bf16*>(p.bias),
                    reinterpret_cast<const bf16*>(p.residual),
                    reinterpret_cast<bf16*>(p.pre),
                    p.y,
                    p.residual_stride,
                    p.pre_stride,
                    p.y_stride,
                    p.activation,
                    y_f32};
  Operands o{static_cast<const unsigned char*>(p.x),
             static_cast<const unsigned char*>(p.w),
             pitch_of(p.x_stride, p.m, p.k, size),
             pitch_of(p.w_stride, p.n, p.k, size),
             (int32_t)p.m,
             (int32_t)p.n,
             (int32_t)(p.k * size),
             0};
  Scratch scratch;
  Rows x{o.a, o.a_pitch, p.m, o.c_bytes}, w{o.b, o.b_pitch, p.n, o.c_bytes};
  x.plan(scratch);
  w.plan(scratch);
  if (p.k == 0 || ((x.copied || w.copied) && dc::linear_few_rows_any(p.m, p.n, o.c_bytes)))
    return fp8 ? few_rows_any<true>(ctx, o, ep) : few_rows_any<false>(ctx, o, ep);
  auto lay_out_all = [&]() -> int32_t {
    if (scratch.bytes) DC_RETURN_IF(dc::ensure_partials(ctx, scratch.bytes));
    DC_RETURN_IF(copy_rows(ctx, lay_out(ctx, &x, &w)));
    o.a = x.p, o.b = w.p, o.a_pitch = x.pitch, o.b_pitch = w.pitch;
    o.c_bytes = (int32_t)padded(o.c_bytes, 16);  // (ragged rows have been copied, with zeros there)
    return DC_OK;
  };
  if (dc::linear_few_rows(p.m, p.n, std::max(1, ctx->cu_count))) {
    DC_RETURN_IF(lay_out_all());
    return fp8 ? few_rows<true>(ctx, o, ep) : few_rows<false>(ctx, o, ep);
  }
  const dc::LinearSize shape{p.m, p.n, o.c_bytes, x.width(), w.width()};
  const dc::LinearPlan best = dc::linear_plan(shape, {false, fp8}, std::max(1, ctx->cu_count));
  const ProductPlan plan(scratch, shape, best.tile, best.split);
  DC_RETURN_IF(lay_out_all());
  const Product all{o, ep, plan};
  return fp8 ? products<true, false>(ctx, {&all}) : products<false, false>(ctx, {&all});
}

DC_HIP_API int32_t dc_hip_linear_backward(dc_hip_ctx* ctx, const dc_linear_grad* args) {
  if (!args) return DC_ERR_INVALID_ARGUMENT;
  const dc_linear_grad& p = *args;
  DC_RETURN_IF(check_dims(p.m, p.n, p.k, p.activation));
  if (p.reserved != 0) return DC_ERR_INVALID_ARGUMENT;
  const bool act = p.activation != DC_ACT_NONE;
  const bool dx = p.dx && p.m > 0 && p.k > 0, dw = p.dw && p.n > 0 && p.k > 0, dbias = p.dbias && p.n > 0;
  if (dw && p.m > dc::kLinearWidth) return DC_ERR_UNSUPPORTED;  // (dw's sums run along m)
  const bool inputs = p.m > 0 && p.n > 0 && (dx || dw || dbias);
  if (inputs) {
    DC_RETURN_IF(check_rows(p.dy, 2, p.dy_stride, p.m, p.n));
    if (act) DC_RETURN_IF(check_rows(p.pre, 2, p.pre_stride, p.m, p.n));
    if (dx) DC_RETURN_IF(check_rows(p.w, 2, p.w_stride, p.n, p.k));
    if (dw) DC_RETURN_IF(check_rows(p.x, 2, p.x_stride, p.m, p.k));
  }
  if (dx) DC_RETURN_IF(check_rows(p.dx, 2, p.dx_stride, p.m, p.k));
  if (dw) DC_RETURN_IF(check_rows(p.dw, 2, p.dw_stride, p.n, p.k));
  if (!aligned_to(p.dbias, 4)) return DC_ERR_MISALIGNED;
  DC_CTX_ENTER(ctx);
  if (!dx && !dw && !dbias) return DC_OK;
  // dz runs along n in dx and along m in dw: a copy of each, padded to whole 16-byte pieces, in scratch; dy itself where
  // it serves as dz.
  Scratch scratch;
  Rows dz{reinterpret_cast<const unsigned char*>(p.dy), pitch_of(p.dy_stride, p.m, p.n, 2), p.m, 2 * p.n};
  Rows w{reinterpret_cast<const unsigned char*>(p.w), pitch_of(p.w_stride, p.n, p.k, 2), p.n, 2 * p.k};
  Rows x{reinterpret_cast<const unsigned char*>(p.x), pitch_of(p.x_stride, p.m, p.k, 2), p.m, 2 * p.k};
  SlopeArgs s{reinterpret_cast<const bf16*>(p.dy), reinterpret_cast<const bf16*>(p.pre), nullptr, nullptr, nullptr, p.m, p.n,
              p.dy_stride, p.pre_stride, padded(p.n, 8), padded(p.m, 8), p.activation};
  size_t at_dzt = 0, at_parts = 0;
  const int64_t pieces = (p.m + 63) / 64;
  if (!inputs) {  // (no rows, or columns, of dz: the sums are empty, which few_rows_any writes as such)
    auto zeros = [&](uint16_t* out, int64_t rows, int64_t stride) -> int32_t {
      Epilogue ep{};
      ep.y = out, ep.y_stride = stride;
      return few_rows_any<false>(ctx, Operands{nullptr, nullptr, 0, 0, (int32_t)rows, (int32_t)p.k, 0, 0, 0}, ep);
    };
    if (dx) DC_RETURN_IF(zeros(p.dx, p.m, p.dx_stride));
    if (dw) DC_RETURN_IF(zeros(p.dw, p.n, p.dw_stride));
    return dbias ? dc::zero_async(ctx, p.dbias, (size_t)p.n * sizeof(float)) : DC_OK;
  }
  if (dx) {
    dz.plan(scratch);
    if (act && !dz.copied) dz.at = scratch.take(p.m * 2 * s.dz_pitch);
    w.plan(scratch);
  }
  const bool own_dz = dx && (act || dz.copied);
  if (dw) {
    at_dzt = scratch.take(p.n * 2 * s.t_pitch);
    x.plan(scratch);
  }
  if (dbias && pieces > 1) at_parts = scratch.take(pieces * p.n * (int64_t)sizeof(float));
  const int64_t dz_pitch = own_dz ? 2 * s.dz_pitch : dz.pitch;
  const dc::LinearSize dx_size{p.m, p.k, 2 * p.n, dz_pitch, w.width()}, dw_size{p.n, p.k, 2 * p.m, 2 * s.t_pitch, x.width()};
  const int64_t cus = std::max(1, ctx->cu_count);
  const bool together = dx && dw;
  dc::LinearPlan dx_best{dc::LinearTile::k64, {1, 1}, 0.0}, dw_best = dx_best;
  if (together) {
    const dc::LinearPair pair = dc::linear_plan_of_two(dx_size, dw_size, cus);
    dx_best = {pair.tile, pair.a, pair.time}, dw_best = {pair.tile, pair.b, pair.time};
  } else if (dx) {
    dx_best = dc::linear_plan(dx_size, {true, false}, cus);
  } else if (dw) {
    dw_best = dc::linear_plan(dw_size, {true, false}, cus);
  }
  const ProductPlan dx_plan(scratch, dx_size, dx_best.tile, dx_best.split), dw_plan(scratch, dw_size, dw_best.tile, dw_best.split);
  if (scratch.bytes) DC_RETURN_IF(dc::ensure_partials(ctx, scratch.bytes));
  unsigned char* base = static_cast<unsigned char*>(ctx->partials);
  if (own_dz) s.dz = reinterpret_cast<bf16*>(base + dz.at);
  if (dw) s.dzt = reinterpret_cast<bf16*>(base + at_dzt);
  if (dbias) s.parts = pieces > 1 ? reinterpret_cast<float*>(base + at_parts) : p.dbias;
  const Copies copies = lay_out(ctx, dx ? &w : nullptr, dw ? &x : nullptr);
  if (s.dz || s.dzt || s.parts) {
    const int64_t grid = std::max(copies.groups, std::min<int64_t>((p.n + 63) / 64 * pieces, 1 << 20));
    slope_kernel<<<dim3((unsigned)grid, (unsigned)(1 + copies.jobs)), 256, 0, ctx->stream>>>(s, copies.args);
    DC_RETURN_IF(dc::last_launch_status());
  } else {
    DC_RETURN_IF(copy_rows(ctx, copies));
  }
  // One gradient: the product of `rows` (m of them, along c) and `b` (c rows of k).
  auto gradient = [&](const void* rows, int64_t pitch, int64_t m, int64_t c, const Rows& b, void* out, int64_t stride,
                      const ProductPlan& plan) {
    Epilogue ep{};
    ep.y = out, ep.y_stride = stride;
    return Product{Operands{static_cast<const unsigned char*>(rows), b.p, pitch, b.pitch, (int32_t)m, (int32_t)p.k, (int32_t)(2 * c),
                            (int32_t)c, (int32_t)padded(p.k, 8)},
                   ep, plan};
  };
  const Product of_x = gradient(own_dz ? static_cast<const void*>(s.dz) : p.dy, dz_pitch, p.m, p.n, w, p.dx, p.dx_stride, dx_plan);
  const Product of_w = gradient(s.dzt, 2 * s.t_pitch, p.n, p.m, x, p.dw, p.dw_stride, dw_plan);
  ColumnParts columns{};
  if (dbias && pieces > 1) columns = {s.parts, p.dbias, (int32_t)pieces, (int32_t)p.n};
  auto run = [&](const Product* first, const Product* second) { return products<false, true>(ctx, {first, second}, columns); };
  if (together) return p.n >= p.m ? run(&of_x, &of_w) : run(&of_w, &of_x);  // (the longer sums first)
  if (dx || dw) return run(dx ? &of_x : &of_w, nullptr);
  return columns.n > 0 ? dc::launch_column_sums(ctx, s.parts, p.dbias, pieces, p.n) : DC_OK;
}

}  // extern "C"
