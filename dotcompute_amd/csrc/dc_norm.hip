// dc_norm.hip — RMS norm with the residual's addition, its gradients, and rows in 8 bits with scales.
//
// Forward, a row at a time: h = x + r, s = 1 / sqrt(mean(h^2) + eps), y = h w s. Memory-bound: 8 bytes an element in
// bf16 (x, r in; h, y out), 7 with y in 8 bits. A row stays in registers between its one read and its write, so nothing
// is read twice: W waves hold it in C 16-byte chunks a lane (W = 1: no barrier, the wave sums by DPP; W = 4 or 16:
// the waves' sums meet in LDS). Rows too long for 16 waves are read again from the caches for each pass (C = 0).
//
// Backward: g = dy w, dx = s (g - h s mean(g h s)) + dh, dw = sum over rows of dy h s. Also one read of each operand; a
// workgroup walks over rows and keeps its part of dw in registers, the parts are added in a fixed order by a
// second kernel (no atomics: the same bits from call to call).
#include <algorithm>

#include "dc_internal.hpp"
#include "dc_numeric.hpp"

namespace {

using dc::bf16;
using dc::kElems;

struct NormArgs {
  const void *x, *residual, *weight;
  void *sum, *y;
  float* scales;
  int64_t rows, x_stride, residual_stride, sum_stride, y_stride;
  int32_t cols;
  float eps;
};

// Sum (or unsigned maximum) over the W waves that share a row, in every lane. `scratch`: W words, which nobody writes
// again before the caller's next barrier.
template <int W>
__device__ inline float row_sum(float v, float* scratch, int wave) {
  v = dc::wave_sum_f32(v);
  if constexpr (W > 1) {
    if ((threadIdx.x & 63) == 0) scratch[wave] = v;
    __syncthreads();
    v = scratch[0];
#pragma unroll
    for (int i = 1; i < W; ++i) v += scratch[i];
  }
  return v;
}
template <int W>
__device__ inline uint32_t row_max(uint32_t v, float* scratch, int wave) {
  v = dc::wave_max_u32(v);
  if constexpr (W > 1) {
    uint32_t* s = reinterpret_cast<uint32_t*>(scratch);
    if ((threadIdx.x & 63) == 0) s[wave] = v;
    __syncthreads();
    v = s[0];
#pragma unroll
    for (int i = 1; i < W; ++i) v = max(v, s[i]);
  }
  return v;
}

// Workgroups of W waves take a row each, or, for W = 1, of four waves with a row each.
template <int W>
constexpr int kNormThreads = W == 1 ? 256 : 64 * W;
template <int W>
constexpr int kNormRows = W == 1 ? 4 : 1;

// y = x itself (a conversion to 8 bits): no norm, no weight.
template <typename T, typename Y, int W, int C, bool kNorm>
__global__ __launch_bounds__(kNormThreads<W>) void rms_norm_kernel(NormArgs a) {
  constexpr int E = kElems<T>;
  constexpr bool kFp8 = sizeof(Y) == 1;
  __shared__ float scratch[3][W == 1 ? 1 : W];
  const int lane = threadIdx.x & 63, wave = W == 1 ? 0 : threadIdx.x >> 6;
  const int64_t cols = a.cols;
  const T* weight = static_cast<const T*>(a.weight);
  const int64_t step = (int64_t)gridDim.x * kNormRows<W>;
  for (int64_t row = (int64_t)blockIdx.x * kNormRows<W> + (W == 1 ? threadIdx.x >> 6 : 0); row < a.rows; row += step) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* r = a.residual ? static_cast<const T*>(a.residual) + row * a.residual_stride : nullptr;
    T* sum = a.sum ? static_cast<T*>(a.sum) + row * a.sum_stride : nullptr;
    Y* y = static_cast<Y*>(a.y) + row * a.y_stride;
    auto read = [&](int64_t c, float (&v)[E]) __attribute__((always_inline)) {
      dc::load_some(x + c, cols - c, v);
      if (r) {
        float u[E];
        dc::load_some(r + c, cols - c, u);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] += u[e];
      }
    };
    if constexpr (C > 0) {
      float h[C][E];
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const int64_t c = (int64_t)((i * W + wave) * 64 + lane) * E;
        if (c < cols) {
          read(c, h[i]);
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e) h[i][e] = 0.0f;
        }
      }
      if constexpr (kNorm) {
#pragma unroll
        for (int i = 0; i < C; ++i)
#pragma unroll
          for (int e = 0; e < E; ++e) ss += h[i][e] * h[i][e];
        const float s = 1.0f / sqrtf(row_sum<W>(ss, scratch[0], wave) / (float)a.cols + a.eps);
#pragma unroll
        for (int i = 0; i < C; ++i) {
          const int64_t c = (int64_t)((i * W + wave) * 64 + lane) * E;
          if (c < cols) {
            if (sum) dc::store_some(sum + c, cols - c, h[i]);
            float w[E];
            dc::load_some(weight + c, cols - c, w);
#pragma unroll
            for (int e = 0; e < E; ++e) h[i][e] = h[i][e] * s * w[e];
          }
        }
      }
      float factor = 1.0f;
      if constexpr (kFp8) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < C; ++i)
#pragma unroll
          for (int e = 0; e < E; ++e) top = max(top, dc::magnitude(h[i][e]));
        const float t = __builtin_bit_cast(float, row_max<W>(top, scratch[1], wave));
        factor = dc::fp8_factor(t);
        if (lane == 0 && wave == 0) a.scales[row] = t / dc::kFp8Top;
      }
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const int64_t c = (int64_t)((i * W + wave) * 64 + lane) * E;
        if (c < cols) {
          if constexpr (kFp8)
#pragma unroll
            for (int e = 0; e < E; ++e) h[i][e] *= factor;
          dc::store_some(y + c, cols - c, h[i]);
        }
      }
    } else {
      const int64_t first = (int64_t)threadIdx.x * E;
      constexpr int64_t kStep = 64 * W * E;
      float s = 1.0f;
      if constexpr (kNorm) {
        float ss = 0.0f;
        for (int64_t c = first; c < cols; c += kStep) {
          float v[E];
          read(c, v);
#pragma unroll
          for (int e = 0; e < E; ++e) ss += v[e] * v[e];
        }
        s = 1.0f / sqrtf(row_sum<W>(ss, scratch[0], wave) / (float)a.cols + a.eps);
      }
      auto normed = [&](int64_t c, float (&v)[E]) __attribute__((always_inline)) {
        if constexpr (kNorm) {
          float w[E];
          dc::load_some(weight + c, cols - c, w);
#pragma unroll
          for (int e = 0; e < E; ++e) v[e] = v[e] * s * w[e];
        }
      };
      float factor = 1.0f;
      if constexpr (kFp8) {
        uint32_t top = 0;
        for (int64_t c = first; c < cols; c += kStep) {
          float v[E];
          read(c, v);
          normed(c, v);
#pragma unroll
          for (int e = 0; e < E; ++e) top = max(top, dc::magnitude(v[e]));
        }
        const float t = __builtin_bit_cast(float, row_max<W>(top, scratch[1], wave));
        factor = dc::fp8_factor(t);
        if (lane == 0 && wave == 0) a.scales[row] = t / dc::kFp8Top;
      }
      for (int64_t c = first; c < cols; c += kStep) {  // (a lane writes only what it alone has read)
        float v[E];
        read(c, v);
        if (sum) dc::store_some(sum + c, cols - c, v);
        normed(c, v);
        if constexpr (kFp8)
#pragma unroll
          for (int e = 0; e < E; ++e) v[e] *= factor;
        dc::store_some(y + c, cols - c, v);
      }
    }
    if constexpr (W > 1) __syncthreads();  // the next row writes the scratch words again
  }
}

struct NormGradArgs {
  const void *dy, *h, *weight, *dh;
  void* dx;
  float* parts;  // [gridDim.x][cols] of dweight, or NULL
  int64_t rows, dy_stride, h_stride, dh_stride, dx_stride;
  int32_t cols;
  float eps;
};

template <typename T, int W, int C>
__global__ __launch_bounds__(64 * W) void rms_norm_grad_kernel(NormGradArgs a) {
  constexpr int E = kElems<T>;
  constexpr int kC = C > 0 ? C : 1;
  __shared__ float scratch[4][W];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t cols = a.cols;
  const T* weight = static_cast<const T*>(a.weight);
  float* part = a.parts ? a.parts + (int64_t)blockIdx.x * cols : nullptr;
  float acc[kC][E];
#pragma unroll
  for (int i = 0; i < kC; ++i)
#pragma unroll
    for (int e = 0; e < E; ++e) acc[i][e] = 0.0f;
  if (C == 0 && part)
    for (int64_t c = threadIdx.x; c < cols; c += 64 * W) part[c] = 0.0f;
  if constexpr (C == 0) __syncthreads();
  int flip = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* dy = static_cast<const T*>(a.dy) + row * a.dy_stride;
    const T* h = static_cast<const T*>(a.h) + row * a.h_stride;
    const T* dh = a.dh ? static_cast<const T*>(a.dh) + row * a.dh_stride : nullptr;
    T* dx = a.dx ? static_cast<T*>(a.dx) + row * a.dx_stride : nullptr;
    float hh = 0.0f, gh = 0.0f;
    float hv[kC][E], dv[kC][E], wv[kC][E];
    auto read = [&](int64_t c, float (&hr)[E], float (&dr)[E], float (&wr)[E]) __attribute__((always_inline)) {
      dc::load_some(h + c, cols - c, hr);
      dc::load_some(dy + c, cols - c, dr);
      dc::load_some(weight + c, cols - c, wr);
    };
    auto add = [&](const float (&hr)[E], const float (&dr)[E], const float (&wr)[E]) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        hh += hr[e] * hr[e];
        gh += dr[e] * wr[e] * hr[e];
      }
    };
    if constexpr (C > 0) {
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const int64_t c = (int64_t)((i * W + wave) * 64 + lane) * E;
        if (c < cols) {
          read(c, hv[i], dv[i], wv[i]);
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e) hv[i][e] = dv[i][e] = wv[i][e] = 0.0f;
        }
      }
#pragma unroll
      for (int i = 0; i < C; ++i) add(hv[i], dv[i], wv[i]);
    } else {
      for (int64_t c = (int64_t)threadIdx.x * E; c < cols; c += 64 * W * E) {
        read(c, hv[0], dv[0], wv[0]);
        add(hv[0], dv[0], wv[0]);
      }
    }
    // (two sets of words in turn: a wave writes a set again only past the barrier of the row between)
    hh = dc::wave_sum_f32(hh);
    gh = dc::wave_sum_f32(gh);
    if constexpr (W > 1) {
      float *s0 = scratch[2 * flip], *s1 = scratch[2 * flip + 1];
      flip ^= 1;
      if (lane == 0) {
        s0[wave] = hh;
        s1[wave] = gh;
      }
      __syncthreads();
      hh = s0[0];
      gh = s1[0];
#pragma unroll
      for (int i = 1; i < W; ++i) {
        hh += s0[i];
        gh += s1[i];
      }
    }
    const float s = 1.0f / sqrtf(hh / (float)a.cols + a.eps);
    const float mean = s * s * (gh / (float)a.cols);  // mean(g h s) s
    auto finish = [&](int64_t c, const float (&hr)[E], const float (&dr)[E], const float (&wr)[E], float (&ac)[E])
        __attribute__((always_inline)) {
      if (dx) {
        float o[E], u[E];
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = s * (dr[e] * wr[e] - hr[e] * mean);
        if (dh) {
          dc::load_some(dh + c, cols - c, u);
#pragma unroll
          for (int e = 0; e < E; ++e) o[e] += u[e];
        }
        dc::store_some(dx + c, cols - c, o);
      }
#pragma unroll
      for (int e = 0; e < E; ++e) ac[e] += dr[e] * (hr[e] * s);
    };
    if constexpr (C > 0) {
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const int64_t c = (int64_t)((i * W + wave) * 64 + lane) * E;
        if (c < cols) finish(c, hv[i], dv[i], wv[i], acc[i]);
      }
    } else {
      for (int64_t c = (int64_t)threadIdx.x * E; c < cols; c += 64 * W * E) {
        read(c, hv[0], dv[0], wv[0]);
        float ac[E];
#pragma unroll
        for (int e = 0; e < E; ++e) ac[e] = part && c + e < cols ? part[c + e] : 0.0f;
        finish(c, hv[0], dv[0], wv[0], ac);
        if (part)
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (c + e < cols) part[c + e] = ac[e];
      }
    }
  }
  if (C > 0 && part)
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int64_t c = (int64_t)((i * W + wave) * 64 + lane) * E;
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (c + e < cols) part[c + e] = acc[i][e];
    }
}

// out[c] = parts[0][c] + ... + parts[count - 1][c]: 64 columns a workgroup, 16 threads a column that each add every
// 16th part, then those 16 sums in order.
constexpr int kSumGroups = 16;
__global__ __launch_bounds__(64 * kSumGroups) void column_sums_kernel(const float* __restrict__ parts, float* __restrict__ out,
                                                                      int64_t count, int64_t cols) {
  __shared__ float sums[kSumGroups][64];
  const int lane = threadIdx.x & 63, g = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane;
  float v = 0.0f;
  if (c < cols)
#pragma unroll 8
    for (int64_t i = g; i < count; i += kSumGroups) v += parts[i * cols + c];
  sums[g][lane] = v;
  __syncthreads();
  if (g == 0 && c < cols) {
#pragma unroll
    for (int i = 1; i < kSumGroups; ++i) v += sums[i][lane];
    out[c] = v;
  }
}

constexpr int64_t kMaxCols = int64_t(1) << 27;
constexpr int64_t kMaxGrid = 1 << 20;  // rows beyond are walked over by the same workgroups

template <typename T, typename Y, int W, int C, bool kNorm>
int32_t launch_norm(dc_hip_ctx* ctx, const NormArgs& a) {
  const int64_t groups = (a.rows + kNormRows<W> - 1) / kNormRows<W>;
  rms_norm_kernel<T, Y, W, C, kNorm>
      <<<(unsigned)std::min<int64_t>(groups, kMaxGrid), kNormThreads<W>, 0, ctx->stream>>>(a);
  return dc::last_launch_status();
}

template <typename T, typename Y, bool kNorm>
int32_t norm_by_shape(dc_hip_ctx* ctx, const NormArgs& a) {
  const int64_t chunks = (a.cols + kElems<T> - 1) / kElems<T>;
  if (chunks <= 512 && a.rows >= 8 * (int64_t)ctx->cu_count) {
    if (chunks <= 64) return launch_norm<T, Y, 1, 1, kNorm>(ctx, a);
    if (chunks <= 128) return launch_norm<T, Y, 1, 2, kNorm>(ctx, a);
    if (chunks <= 256) return launch_norm<T, Y, 1, 4, kNorm>(ctx, a);
    return launch_norm<T, Y, 1, 8, kNorm>(ctx, a);
  }
  if (chunks <= 256) return launch_norm<T, Y, 4, 1, kNorm>(ctx, a);
  if (chunks <= 512) return launch_norm<T, Y, 4, 2, kNorm>(ctx, a);
  if (chunks <= 1024) return launch_norm<T, Y, 4, 4, kNorm>(ctx, a);
  if (chunks <= 2048) return launch_norm<T, Y, 4, 8, kNorm>(ctx, a);
  if (chunks <= 4096) return launch_norm<T, Y, 16, 4, kNorm>(ctx, a);
  if (chunks <= 8192) return launch_norm<T, Y, 16, 8, kNorm>(ctx, a);
  return launch_norm<T, Y, 16, 0, kNorm>(ctx, a);
}

template <typename T>
int32_t norm_grad_by_shape(dc_hip_ctx* ctx, const NormGradArgs& a, int64_t grid) {
  const int64_t chunks = (a.cols + kElems<T> - 1) / kElems<T>;
  const unsigned g = (unsigned)grid;
  if (chunks <= 64) rms_norm_grad_kernel<T, 1, 1><<<g, 64, 0, ctx->stream>>>(a);
  else if (chunks <= 256) rms_norm_grad_kernel<T, 4, 1><<<g, 256, 0, ctx->stream>>>(a);
  else if (chunks <= 512) rms_norm_grad_kernel<T, 4, 2><<<g, 256, 0, ctx->stream>>>(a);
  else if (chunks <= 1024) rms_norm_grad_kernel<T, 4, 4><<<g, 256, 0, ctx->stream>>>(a);
  else if (chunks <= 4096) rms_norm_grad_kernel<T, 16, 4><<<g, 1024, 0, ctx->stream>>>(a);
  else rms_norm_grad_kernel<T, 16, 0><<<g, 1024, 0, ctx->stream>>>(a);
  return dc::last_launch_status();
}

bool float_dtype(int32_t t) { return t == DC_DTYPE_F32 || t == DC_DTYPE_BF16; }
int64_t size_of(int32_t t) { return t == DC_DTYPE_F32 ? 4 : t == DC_DTYPE_BF16 ? 2 : 1; }
bool aligned_to(const void* p, int64_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }

// One row, or several with a stride of at least a row's length.
int32_t check_rows(const void* p, int32_t dtype, int64_t stride, int64_t rows, int64_t cols) {
  if (!aligned_to(p, size_of(dtype))) return DC_ERR_MISALIGNED;
  return rows > 1 && stride < cols ? DC_ERR_DIMENSION : DC_OK;
}

int32_t check_shape(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 0) return DC_ERR_INVALID_ARGUMENT;
  return cols > kMaxCols ? DC_ERR_UNSUPPORTED : DC_OK;
}

}  // namespace

namespace dc {

int32_t launch_column_sums(dc_hip_ctx* ctx, const float* parts, float* out, int64_t count, int64_t cols) {
  // (1024 work items for 64 columns, at most kMaxCols of them: within the 2^32 of a launch)
  column_sums_kernel<<<(unsigned)((cols + 63) / 64), 64 * kSumGroups, 0, ctx->stream>>>(parts, out, count, cols);
  return last_launch_status();
}

}  // namespace dc

extern "C" {

DC_HIP_API int32_t dc_hip_rms_norm(dc_hip_ctx* ctx, const dc_rms_norm* args) {
  if (!args) return DC_ERR_INVALID_ARGUMENT;
  const dc_rms_norm& p = *args;
  DC_RETURN_IF(check_shape(p.rows, p.cols));
  const bool fp8 = p.y_dtype == DC_DTYPE_FP8;
  if (!float_dtype(p.dtype) || (!fp8 && p.y_dtype != p.dtype) || p.reserved != 0) return DC_ERR_INVALID_ARGUMENT;
  if (!(p.eps >= 0.0f) || fp8 != (p.scales != nullptr)) return DC_ERR_INVALID_ARGUMENT;
  if (p.rows > 0 && p.cols > 0) {
    if (!p.x || !p.weight || !p.y) return DC_ERR_INVALID_ARGUMENT;
    DC_RETURN_IF(check_rows(p.x, p.dtype, p.x_stride, p.rows, p.cols));
    DC_RETURN_IF(check_rows(p.y, p.y_dtype, p.y_stride, p.rows, p.cols));
    DC_RETURN_IF(check_rows(p.weight, p.dtype, p.cols, 1, p.cols));
    if (p.residual) DC_RETURN_IF(check_rows(p.residual, p.dtype, p.residual_stride, p.rows, p.cols));
    if (p.sum) DC_RETURN_IF(check_rows(p.sum, p.dtype, p.sum_stride, p.rows, p.cols));
    if (!aligned_to(p.scales, 4)) return DC_ERR_MISALIGNED;
  }
  DC_CTX_ENTER(ctx);
  if (p.rows == 0 || p.cols == 0) return DC_OK;
  const NormArgs a{p.x,    p.residual,        p.weight,     p.sum,      p.y,              p.scales, p.rows,
                   p.x_stride, p.residual_stride, p.sum_stride, p.y_stride, (int32_t)p.cols, p.eps};
  if (p.dtype == DC_DTYPE_F32)
    return fp8 ? norm_by_shape<float, uint8_t, true>(ctx, a) : norm_by_shape<float, float, true>(ctx, a);
  return fp8 ? norm_by_shape<bf16, uint8_t, true>(ctx, a) : norm_by_shape<bf16, bf16, true>(ctx, a);
}

DC_HIP_API int32_t dc_hip_rms_norm_backward(dc_hip_ctx* ctx, const dc_rms_norm_grad* args) {
  if (!args) return DC_ERR_INVALID_ARGUMENT;
  const dc_rms_norm_grad& p = *args;
  DC_RETURN_IF(check_shape(p.rows, p.cols));
  if (!float_dtype(p.dtype) || !(p.eps >= 0.0f)) return DC_ERR_INVALID_ARGUMENT;
  if (p.rows > 0 && p.cols > 0) {
    if (!p.dy || !p.h || !p.weight) return DC_ERR_INVALID_ARGUMENT;
    DC_RETURN_IF(check_rows(p.dy, p.dtype, p.dy_stride, p.rows, p.cols));
    DC_RETURN_IF(check_rows(p.h, p.dtype, p.h_stride, p.rows, p.cols));
    DC_RETURN_IF(check_rows(p.weight, p.dtype, p.cols, 1, p.cols));
    if (p.dh) DC_RETURN_IF(check_rows(p.dh, p.dtype, p.dh_stride, p.rows, p.cols));
    if (p.dx) DC_RETURN_IF(check_rows(p.dx, p.dtype, p.dx_stride, p.rows, p.cols));
  }
  if (!aligned_to(p.dweight, 4)) return DC_ERR_MISALIGNED;
  DC_CTX_ENTER(ctx);
  if (p.cols == 0 || (!p.dx && !p.dweight)) return DC_OK;
  if (p.rows == 0) return p.dweight ? dc::zero_async(ctx, p.dweight, (size_t)p.cols * sizeof(float)) : DC_OK;
  const int64_t grid = std::min<int64_t>(p.rows, 4 * (int64_t)std::max(1, ctx->cu_count));
  float* parts = nullptr;
  if (p.dweight) {
    DC_RETURN_IF(dc::ensure_partials(ctx, (size_t)(grid * p.cols) * sizeof(float)));
    parts = static_cast<float*>(ctx->partials);
  }
  const NormGradArgs a{p.dy,   p.h,         p.weight,   p.dh,        p.dx,        parts,
                       p.rows, p.dy_stride, p.h_stride, p.dh_stride, p.dx_stride, (int32_t)p.cols, p.eps};
  DC_RETURN_IF(p.dtype == DC_DTYPE_F32 ? norm_grad_by_shape<float>(ctx, a, grid) : norm_grad_by_shape<bf16>(ctx, a, grid));
  return p.dweight ? dc::launch_column_sums(ctx, parts, p.dweight, grid, p.cols) : DC_OK;
}

DC_HIP_API int32_t dc_hip_quantize_fp8(dc_hip_ctx* ctx, const void* x, int32_t dtype, int64_t x_stride, uint8_t* q,
                                       int64_t q_stride, float* scales, int64_t rows, int64_t cols) {
  DC_RETURN_IF(check_shape(rows, cols));
  if (!float_dtype(dtype)) return DC_ERR_INVALID_ARGUMENT;
  if (rows > 0 && cols > 0) {
    if (!x || !q || !scales) return DC_ERR_INVALID_ARGUMENT;
    DC_RETURN_IF(check_rows(x, dtype, x_stride, rows, cols));
    DC_RETURN_IF(check_rows(q, DC_DTYPE_FP8, q_stride, rows, cols));
    if (!aligned_to(scales, 4)) return DC_ERR_MISALIGNED;
  }
  DC_CTX_ENTER(ctx);
  if (rows == 0 || cols == 0) return DC_OK;
  const NormArgs a{x, nullptr, nullptr, nullptr, q, scales, rows, x_stride, 0, 0, q_stride, (int32_t)cols, 0.0f};
  return dtype == DC_DTYPE_F32 ? norm_by_shape<float, uint8_t, false>(ctx, a) : norm_by_shape<bf16, uint8_t, false>(ctx, a);
}

}  // extern "C"
