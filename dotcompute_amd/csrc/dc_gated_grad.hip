// dc_gated_grad.hip — gradients of y = act(g) u with g = x wg^T + bg and u = x wu^T + bu, from dy and the g and u that the forward pass left:
// dg = dy u act'(g), du = dy act(g); dx = dg wg + du wu, dwg = dg^T x, dwu = du^T x, dbg and dbu the column sums of dg and du.
//
// As a linear layer's gradients (dc_linear.hip): one pass forms dg and du beside each other in rows, and their transposes, in bf16, and the column sums'
// parts; one launch runs all three products. dx is one sum along both halves of a row: its B's rows are wg's, then wu's, each half padded with zeros to
// whole tiles along c, so that a tile is of one weight.
//
// What is rounded: dg and du to bf16, as a linear layer's dz: the matrix cores take float32 at a 16th of the rate, and a second bf16 for what is
// left of each would double the products (890 of 1066 us at 8192×8192×2048). It leaves the gradients 0.0023 of themselves off, in the mean, where
// rounding them alone leaves 0.0017. The biases' gradients add dg and du unrounded. Sums are float32, results rounded once.
#include "dc_linear_device.hpp"

namespace {

struct GatedSlopeArgs {
  const bf16 *dy, *gate, *up;
  bf16* dz;                   // [m][2 half]: dg, then du, zeros from n to half; or NULL
  bf16 *gate_t, *up_t;        // their transposes (pitch t_pitch, columns from m to there zero), or NULL
  float *gate_parts, *up_parts;  // [pieces of rows][part_pitch] sums of columns, or NULL
  int64_t m, n, half, dy_stride, gate_stride, up_stride, t_pitch, part_pitch;
  int32_t act;
};

template <bool kOnce>
__device__ inline void load_part(const bf16* p, int64_t left, float (&v)[8]) {
  if (kOnce && left >= 8) dc::unpack(dc::load_raw_once(p), v);
  else dc::load_some(p, left, v);
}
// 64×64 pieces, as slope_kernel's: a thread holds two neighbouring rows of 8 columns; the transposes and the column sums through LDS, dg's before du's.
// (The workgroups with blockIdx.y > 0 copy the operands that have to be, beside it.) HBM: 6 bytes in and 8 out for each element: 8192×8192 169 us, 5.6 TB/s.
template <bool kOnce>
__global__ __launch_bounds__(256) void gated_slope_kernel(GatedSlopeArgs a, PackArgs copies) {
  __shared__ uint32_t turned[64][33];
  __shared__ float sums[32][65];
  if (blockIdx.y > 0) return pack_rows(copies.job[blockIdx.y - 1], blockIdx.x, gridDim.x);
  const int t = threadIdx.x, c8 = t & 7, pair = t >> 3;
  const int64_t across = (a.n + 63) / 64, total = across * ((a.m + 63) / 64);
  for (int64_t at = blockIdx.x; at < total; at += gridDim.x) {
    const int64_t down = total <= UINT32_MAX ? (int64_t)((uint32_t)at / (uint32_t)across) : at / across;
    const int64_t m0 = down * 64, n0 = (at - down * across) * 64;
    const int64_t j = n0 + 8 * c8;
    float dz[2][2][8];  // of the gate, and of the other factor; of two rows
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int64_t i = m0 + 2 * pair + q;
      float g[8], u[8], dy[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) dz[0][q][e] = dz[1][q][e] = 0.0f;
      if (i < a.m && j < a.n) {
        load_part<kOnce>(a.dy + i * a.dy_stride + j, a.n - j, dy);
        load_part<kOnce>(a.gate + i * a.gate_stride + j, a.n - j, g);
        load_part<kOnce>(a.up + i * a.up_stride + j, a.n - j, u);  // (zeros past the last: their dy is zero)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          dz[0][q][e] = dy[e] * u[e];
          dz[1][q][e] = g[e];
        }
        apply_slope(a.act, g, dz[0][q]);
        activate(a.act, dz[1][q]);
#pragma unroll
        for (int e = 0; e < 8; ++e) dz[1][q][e] *= dy[e];
      }
      if (a.dz && i < a.m) {
        bf16* to = a.dz + i * 2 * a.half + j;
        dc::store_chunk(to, dz[0][q]);
        dc::store_chunk(to + a.half, dz[1][q]);
      }
    }
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      bf16* to = f ? a.up_t : a.gate_t;
      float* parts = f ? a.up_parts : a.gate_parts;
      if (!to && !parts) continue;  // (uniform)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        turned[8 * c8 + e][pair] = dc::pack_bf16(dz[f][0][e], dz[f][1][e]);
        sums[pair][8 * c8 + e] = dz[f][0][e] + dz[f][1][e];
      }
      __syncthreads();
      if (to) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {  // 64 rows of 8 16-byte chunks
          const int row = (t >> 3) + 32 * q, chunk = t & 7;
          const int64_t c = m0 + 8 * chunk;
          if (n0 + row < a.n && c < a.t_pitch) {
            const dc::u32x4 w = {turned[row][4 * chunk], turned[row][4 * chunk + 1], turned[row][4 * chunk + 2],
                                 turned[row][4 * chunk + 3]};
            *reinterpret_cast<dc::u32x4*>(to + (n0 + row) * a.t_pitch + c) = w;
          }
        }
      }
      if (parts && t < 64 && n0 + t < a.n) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < 32; ++i) s += sums[i][t];
        parts[m0 / 64 * a.part_pitch + n0 + t] = s;
      }
      __syncthreads();
    }
  }
}

// One of the gradients' products.
struct GradProduct {
  MoreOperands o;
  Epilogue ep;
  ProductPlan plan;
};

template <int TM, int TN, int WM, int WN, int KS>
int32_t launch_gradients(dc_hip_ctx* ctx, const GradProduct* const* p, int count, const ColumnPartsOfTwo& columns) {
  typedef ProductTypes<true, true, false> Types;
  typename Types::Jobs jobs{};
  int64_t total = 0;
  for (int i = 0; i < Types::kJobs; ++i) {
    if (i < count) {
      auto& j = jobs.job[i];
      const Product sums{p[i]->o, p[i]->ep, p[i]->plan};
      j.o = p[i]->o, j.ep = p[i]->ep;
      j.tiles_m = (j.o.m + TM - 1) / TM, j.tiles_n = (j.o.n + TN - 1) / TN;
      j.parts = (int32_t)sums.plan.split.parts, j.turns = (int32_t)sums.plan.split.turns;
      if (j.parts > 1) {  // the sums alone
        j.ep = Epilogue{};
        j.ep.y = sums.parts(ctx), j.ep.y_stride = sums.pitch(), j.ep.y_f32 = 1, j.ep.part_stride = j.o.m * sums.pitch();
      }
      total += (int64_t)j.tiles_m * j.tiles_n * j.parts;
      if (total > INT32_MAX / 2) return DC_ERR_UNSUPPORTED;
    }
    jobs.ends[i] = (int32_t)total;
  }
  jobs.columns = columns;
  return launch_jobs<TM, TN, WM, WN, KS, false, true, true, false>(ctx, jobs, total);
}

int32_t gradients(dc_hip_ctx* ctx, const GradProduct* const* p, int count, const ColumnPartsOfTwo& columns) {
  using dc::LinearTile;
  int32_t status = DC_ERR_INVALID_ARGUMENT;
  switch (p[0]->plan.tile) {
    case LinearTile::k256: status = launch_gradients<256, 256, 2, 4, 1>(ctx, p, count, columns); break;
    case LinearTile::k128: status = launch_gradients<128, 128, 2, 2, 1>(ctx, p, count, columns); break;
    case LinearTile::k128x2: status = launch_gradients<128, 128, 2, 2, 2>(ctx, p, count, columns); break;
    case LinearTile::k64: status = launch_gradients<64, 64, 2, 2, 1>(ctx, p, count, columns); break;
    case LinearTile::k64x2: status = launch_gradients<64, 64, 2, 2, 2>(ctx, p, count, columns); break;
    case LinearTile::k64x4: status = launch_gradients<64, 64, 2, 2, 4>(ctx, p, count, columns); break;
  }
  if (status != DC_OK) return status;
  JoinArgs args{};
  int jobs = 0;
  int64_t most = 0;
  for (int i = 0; i < count; ++i) {
    const Product sums{p[i]->o, p[i]->ep, p[i]->plan};
    if (sums.plan.split.parts == 1) continue;
    args.job[jobs++] = JoinJob{sums.parts(ctx), sums.o.m, sums.o.n, sums.pitch(), (int32_t)sums.plan.split.parts, sums.ep};
    most = std::max(most, (sums.o.m * (sums.pitch() / 8) + 255) / 256);
  }
  if (jobs == 0) return DC_OK;
  join_kernel<<<dim3((unsigned)std::min<int64_t>(most, 1 << 16), (unsigned)jobs), 256, 0, ctx->stream>>>(args);
  return dc::last_launch_status();
}

}  // namespace

extern "C" {

DC_HIP_API int32_t dc_hip_gated_linear_backward(dc_hip_ctx* ctx, const dc_gated_linear_grad* args) {
  if (!args) return DC_ERR_INVALID_ARGUMENT;
  const dc_gated_linear_grad& p = *args;
  DC_RETURN_IF(check_dims(p.m, p.n, p.k, p.activation));
  if (p.n > dc::kGatedWidth) return DC_ERR_UNSUPPORTED;
  if (p.reserved != 0) return DC_ERR_INVALID_ARGUMENT;
  const bool dx = p.dx && p.m > 0 && p.k > 0, dw_gate = p.dw_gate && p.n > 0 && p.k > 0, dw_up = p.dw_up && p.n > 0 && p.k > 0;
  const bool db_gate = p.dbias_gate && p.n > 0, db_up = p.dbias_up && p.n > 0, dw = dw_gate || dw_up, db = db_gate || db_up;
  if (dw && p.m > dc::kLinearWidth) return DC_ERR_UNSUPPORTED;  // (their sums run along m)
  const bool inputs = p.m > 0 && p.n > 0 && (dx || dw || db);
  if (inputs) {
    DC_RETURN_IF(check_rows(p.dy, 2, p.dy_stride, p.m, p.n));
    DC_RETURN_IF(check_rows(p.pre_gate, 2, p.pre_gate_stride, p.m, p.n));
    DC_RETURN_IF(check_rows(p.pre_up, 2, p.pre_up_stride, p.m, p.n));
    if (dx) DC_RETURN_IF(check_rows(p.w_gate, 2, p.w_gate_stride, p.n, p.k));
    if (dx) DC_RETURN_IF(check_rows(p.w_up, 2, p.w_up_stride, p.n, p.k));
    if (dw) DC_RETURN_IF(check_rows(p.x, 2, p.x_stride, p.m, p.k));
  }
  if (dx) DC_RETURN_IF(check_rows(p.dx, 2, p.dx_stride, p.m, p.k));
  if (dw_gate) DC_RETURN_IF(check_rows(p.dw_gate, 2, p.dw_gate_stride, p.n, p.k));
  if (dw_up) DC_RETURN_IF(check_rows(p.dw_up, 2, p.dw_up_stride, p.n, p.k));
  if (!aligned_to(p.dbias_gate, 4) || !aligned_to(p.dbias_up, 4)) return DC_ERR_MISALIGNED;
  DC_CTX_ENTER(ctx);
  if (!dx && !dw && !db) return DC_OK;
  if (!inputs) {  // (no rows, or no outputs: the sums are empty, which the adding kernel writes as such)
    auto zeros = [&](uint16_t* out, int64_t rows, int64_t stride) -> int32_t {
      Epilogue ep{};
      ep.y = out, ep.y_stride = stride;
      few_rows_any_kernel<false, 4, 2, 8, 2><<<dim3((unsigned)((p.k + 15) / 16), (unsigned)std::min<int64_t>((rows + 31) / 32, 32768)), 512, 0,
                                               ctx->stream>>>(Operands{nullptr, nullptr, 0, 0, (int32_t)rows, (int32_t)p.k, 0, 0, 0}, ep);
      return dc::last_launch_status();
    };
    if (dx) DC_RETURN_IF(zeros(p.dx, p.m, p.dx_stride));
    if (dw_gate) DC_RETURN_IF(zeros(p.dw_gate, p.n, p.dw_gate_stride));
    if (dw_up) DC_RETURN_IF(zeros(p.dw_up, p.n, p.dw_up_stride));
    if (db_gate) DC_RETURN_IF(dc::zero_async(ctx, p.dbias_gate, (size_t)p.n * sizeof(float)));
    return db_up ? dc::zero_async(ctx, p.dbias_up, (size_t)p.n * sizeof(float)) : DC_OK;
  }
  constexpr int64_t kTileRows = kTileBytes / 2;  // of c
  Scratch scratch;
  Rows gate{reinterpret_cast<const unsigned char*>(p.w_gate), pitch_of(p.w_gate_stride, p.n, p.k, 2), p.n, 2 * p.k};
  Rows up{reinterpret_cast<const unsigned char*>(p.w_up), pitch_of(p.w_up_stride, p.n, p.k, 2), p.n, 2 * p.k};
  Rows x{reinterpret_cast<const unsigned char*>(p.x), pitch_of(p.x_stride, p.m, p.k, 2), p.m, 2 * p.k};
  GatedSlopeArgs s{};
  s.dy = reinterpret_cast<const bf16*>(p.dy), s.gate = reinterpret_cast<const bf16*>(p.pre_gate), s.up = reinterpret_cast<const bf16*>(p.pre_up);
  s.m = p.m, s.n = p.n, s.half = padded(p.n, kTileRows), s.t_pitch = padded(p.m, 8), s.act = p.activation;
  s.dy_stride = p.dy_stride, s.gate_stride = p.pre_gate_stride, s.up_stride = p.pre_up_stride;
  const int64_t pieces = (p.m + 63) / 64, dz_pitch = 4 * s.half;
  size_t at_dz = 0, at_gate_t = 0, at_up_t = 0, at_parts = 0;
  if (dx) {
    at_dz = scratch.take(p.m * dz_pitch);
    gate.plan(scratch);
    up.plan(scratch);
  }
  if (dw_gate) at_gate_t = scratch.take(p.n * 2 * s.t_pitch);
  if (dw_up) at_up_t = scratch.take(p.n * 2 * s.t_pitch);
  if (dw) x.plan(scratch);
  if (db && pieces > 1) at_parts = scratch.take(pieces * 2 * p.n * (int64_t)sizeof(float));
  const int64_t dws = (dw_gate ? 1 : 0) + (dw_up ? 1 : 0), cus = std::max(1, ctx->cu_count);
  const dc::LinearSize dx_size{p.m, p.k, dz_pitch, dz_pitch, std::max(gate.width(), up.width())};
  const dc::LinearSize dw_size{p.n, p.k, 2 * p.m, 2 * s.t_pitch, x.width()}, dws_size{dws * p.n, p.k, 2 * p.m, 2 * s.t_pitch, x.width()};
  dc::LinearPlan dx_best{dc::LinearTile::k64, {1, 1}, 0.0}, dw_best = dx_best;
  if (dx && dw) {
    const dc::LinearPair pair = dc::linear_plan_of_two(dx_size, dws_size, cus, true);
    dx_best = {pair.tile, pair.a, pair.time}, dw_best = {pair.tile, pair.b, pair.time};
  } else if (dx) {
    dx_best = dc::linear_plan(dx_size, {true, false}, cus);
  } else if (dw) {
    dw_best = dc::linear_plan(dws_size, {true, false}, cus);
  }
  const dc::LinearSplit one{1, 1};
  const ProductPlan dx_plan(scratch, dx_size, dx_best.tile, dx ? dx_best.split : one);
  const ProductPlan gate_plan(scratch, dw_size, dw_best.tile, dw_gate ? dw_best.split : one);
  const ProductPlan up_plan(scratch, dw_size, dw_best.tile, dw_up ? dw_best.split : one);
  if (scratch.bytes) DC_RETURN_IF(dc::ensure_partials(ctx, scratch.bytes));
  unsigned char* base = static_cast<unsigned char*>(ctx->partials);
  if (dx) s.dz = reinterpret_cast<bf16*>(base + at_dz);
  if (dw_gate) s.gate_t = reinterpret_cast<bf16*>(base + at_gate_t);
  if (dw_up) s.up_t = reinterpret_cast<bf16*>(base + at_up_t);
  float* parts = reinterpret_cast<float*>(base + at_parts);
  s.part_pitch = pieces > 1 ? 2 * p.n : p.n;
  if (db_gate) s.gate_parts = pieces > 1 ? parts : p.dbias_gate;
  if (db_up) s.up_parts = pieces > 1 ? parts + p.n : p.dbias_up;
  const Copies copies = lay_out(ctx, dx ? &gate : nullptr, dx ? &up : nullptr, dw ? &x : nullptr);
  const int64_t grid = std::max(copies.groups, std::min<int64_t>((p.n + 63) / 64 * pieces, 1 << 20));
  auto* slopes = dc::read_once(p.m, p.n, 14) ? gated_slope_kernel<true> : gated_slope_kernel<false>;
  slopes<<<dim3((unsigned)grid, (unsigned)(1 + copies.jobs)), 256, 0, ctx->stream>>>(s, copies.args);
  DC_RETURN_IF(dc::last_launch_status());
  ColumnPartsOfTwo columns{};
  if (db && pieces > 1) {
    columns.parts = parts, columns.count = (int32_t)pieces, columns.n = (int32_t)(2 * p.n), columns.half = (int32_t)p.n;
    columns.out = db_gate ? p.dbias_gate : nullptr, columns.out2 = db_up ? p.dbias_up : nullptr;
  }
  // One gradient: the product of `rows` (m of them, along c) and `b` (its rows along c, then `b2`'s).
  auto gradient = [&](const bf16* rows, int64_t pitch, int64_t m, int64_t c_bytes, int64_t c_rows, const Rows& b, const Rows* b2, void* out,
                      int64_t stride, const ProductPlan& plan) {
    MoreOperands o{};
    o.a = reinterpret_cast<const unsigned char*>(rows), o.a_pitch = pitch, o.b = b.p, o.b_pitch = b.pitch;
    o.m = (int32_t)m, o.n = (int32_t)p.k, o.c_bytes = (int32_t)c_bytes, o.c_rows = (int32_t)c_rows, o.b_cols = (int32_t)padded(p.k, 8);
    o.c_half = b2 ? (int32_t)s.half : INT32_MAX;
    if (b2) o.b2 = b2->p, o.b2_pitch = b2->pitch;
    Epilogue ep{};
    ep.y = out, ep.y_stride = stride;
    return GradProduct{o, ep, plan};
  };
  const GradProduct of_x = gradient(s.dz, dz_pitch, p.m, dz_pitch, p.n, gate, &up, p.dx, p.dx_stride, dx_plan);
  const GradProduct of_gate = gradient(s.gate_t, 2 * s.t_pitch, p.n, 2 * p.m, p.m, x, nullptr, p.dw_gate, p.dw_gate_stride, gate_plan);
  const GradProduct of_up = gradient(s.up_t, 2 * s.t_pitch, p.n, 2 * p.m, p.m, x, nullptr, p.dw_up, p.dw_up_stride, up_plan);
  const GradProduct* list[3];
  int count = 0;
  const bool dx_first = 2 * p.n >= p.m;  // (the longer sums first)
  if (dx && dx_first) list[count++] = &of_x;
  if (dw_gate) list[count++] = &of_gate;
  if (dw_up) list[count++] = &of_up;
  if (dx && !dx_first) list[count++] = &of_x;
  if (count > 0) return gradients(ctx, list, count, columns);
  if (columns.n == 0) return DC_OK;
  float* first = db_gate ? p.dbias_gate : p.dbias_up;
  return dc::launch_column_sums_of(ctx, db_gate ? parts : parts + p.n, 2 * p.n, p.n, first, db_gate && db_up ? p.dbias_up : nullptr, pieces, p.n);
}

}  // extern "C"
