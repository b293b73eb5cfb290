// dc_layer_norm.hip — layer norm with the residual's addition, its gradients, and rows in 8 bits with a scale for each 128 elements.
//
// Forward, a row at a time: h = x + r, y = (h - mean) s w + b with s = 1 / sqrt(var + eps). Memory-bound: 8 bytes an element in bf16 (x, r
// in; h, y out), 7 with y in 8 bits. A row stays in registers between its one read and its write, as an RMS norm's.
//
// Backward: u = (h - mean) s, g = dy w: dx = s (g - mean(g) - u mean(g u)) + dh, dw = the sum over rows of dy u, db of dy. One read of each
// operand; the statistics are formed again from h, which is read anyway. A workgroup walks over rows and keeps its parts of dw
// and db in registers; a second kernel adds the parts in a fixed order (no atomics: the same bits from call to call).
//
// Statistics. The difference of mean(h^2) and mean(h)^2 loses the variance's digits where the mean is large, and a second sum over a row that
// several waves share would be a second barrier. So each wave takes a value k near its own part's mean, the mean of the first 32 elements (of 256 or
// 512, or up to four times as many), and the sums of d = h - k and d^2, in registers; the waves' triples meet in LDS once, and every wave joins them: M is
// the rounded mean, e what is left, and sum((h - M)^2) = the sum over waves of sum(d^2) + 2 c sum(d) + n c^2, c = k - M. Elements
// are taken as (h - M) - e, exact next to the mean. (However a wave's values lie, (k - mean)^2 is at most n / 32 times their variance, so
// that at worst 4 to 6 bits of its 24 are lost there, where one value stands out by itself among the first 32; none for others.)
#include <algorithm>

#include "dc_internal.hpp"
#include "dc_norm_row.hpp"
#include "dc_numeric.hpp"

namespace {

using namespace dc;

struct LayerNormArgs {
  const void *x, *residual, *weight, *bias;
  void *sum, *y, *scales;
  int64_t rows, x_stride, residual_stride, sum_stride, y_stride, scales_stride;
  int32_t cols;
  float eps;
};

// Elements of a row that a wave holds (Row's chunks).
template <int E, int C>
__device__ inline float wave_count(int64_t cols, int waves, int wave) {
  int64_t n = 0;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int64_t left = cols - (int64_t)(i * waves + wave) * 64 * E;
    n += left < 0 ? 0 : left > 64 * E ? 64 * E : left;
  }
  return (float)n;
}
// Whether all elements of a wave's chunk i are in the row (uniform).
template <typename T, int C>
__device__ inline bool whole_chunk(const Row<T, C>& R, int i) {
  return (int64_t)((i * R.waves + R.wave) * 64 + 64) * kElems<T> <= R.cols;
}

// A value near the mean of a wave's elements, and the sums of what is left over it and of that squared (elements past the row's end are zeros in h).
struct Moments {
  float near, left, squares;
};
// 1 / the number of elements that `near` is the mean of.
template <int E>
__device__ inline float near_weight(int64_t cols, int wave) {
  const int64_t left = cols - (int64_t)wave * 64 * E;
  return 1.0f / (float)(left < 4 * E ? left : 4 * E);
}
template <typename T, int C>
__device__ inline float value_near(const float (&h)[C][kElems<T>], float weight) {
  constexpr int E = kElems<T>;
  float v = 0.0f;
#pragma unroll
  for (int e = 0; e < E; e += 4) v += (h[0][e] + h[0][e + 1]) + (h[0][e + 2] + h[0][e + 3]);
  v += __builtin_bit_cast(float, dpp_u32<0xB1, 0xF>(__builtin_bit_cast(uint32_t, v)));
  v += __builtin_bit_cast(float, dpp_u32<0x4E, 0xF>(__builtin_bit_cast(uint32_t, v)));
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v))) * weight;
}
// The lane's part of the sums.
template <typename T, int C>
__device__ inline Moments lane_moments(const Row<T, C>& R, const float (&h)[C][kElems<T>], float near) {
  constexpr int E = kElems<T>;
  Moments m{near, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const bool whole = whole_chunk(R, i);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float d = h[i][e] - near;
      if (!whole) d = R.at(i) + e < R.cols ? d : 0.0f;
      m.left += d;
      m.squares += d * d;
    }
  }
  return m;
}

// A row's mean in two parts, and 1 / sqrt(var + eps).
struct RowStats {
  float mean, rest, s;
};
// The waves' moments, one in each of 16 lanes (`n`: of how many elements, 0 where there is no wave), joined; `off`: what the lane's wave's value
// is away from the row's mean. `per`: 1 / cols.
__device__ inline RowStats join_moments(const Moments& m, float n, float per, float eps, float* off) {
  RowStats r;
  r.mean = row16_sum_f32(__builtin_fmaf(n, m.near, m.left)) * per;
  *off = m.near - r.mean;
  const float rest = row16_sum_f32(__builtin_fmaf(n, *off, m.left));
  const float squares = row16_sum_f32(m.squares + *off * __builtin_fmaf(n, *off, 2.0f * m.left));
  r.rest = rest * per;
  r.s = 1.0f / sqrtf((squares - rest * r.rest) * per + eps);
  return r;
}
// Of a row that one wave holds.
__device__ inline RowStats own_stats(const Moments& m, float per, float eps) {
  RowStats r;
  r.mean = m.near;
  r.rest = m.left * per;
  r.s = 1.0f / sqrtf((m.squares - m.left * r.rest) * per + eps);
  return r;
}

typedef float f32x4_lds __attribute__((ext_vector_type(4)));

// A row a workgroup; or, where a wave holds a row, one for each of its four waves. 8 bits: a scale a row, or (kBlocks) one for each 128.
template <typename T, typename Y, int C, bool kBlocks>
__global__ __launch_bounds__(C == 4 ? 1024 : 512) void layer_norm_kernel(LayerNormArgs a, int waves) {
  constexpr int E = kElems<T>;
  constexpr bool kFp8 = sizeof(Y) == 1;
  __shared__ __align__(16) f32x4_lds words[kWaves];
  __shared__ __align__(16) float scratch[1][kWaves];
  const int lane = threadIdx.x & 63, group = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = waves == 1 ? 0 : group;
  const int64_t cols = a.cols;
  const Row<T, C> R{cols, waves, wave, lane};
  const int other = lane & (kWaves - 1);  // whose moments this lane joins
  const float weight = near_weight<E>(cols, wave), n_other = other < waves ? wave_count<E, C>(cols, waves, other) : 0.0f;
  const float per_col = 1.0f / (float)a.cols;
  clear_words(scratch, 1, waves);
  const int per = waves == 1 ? 4 : 1;
  const int64_t step = (int64_t)gridDim.x * per;
  for (int64_t row = (int64_t)blockIdx.x * per + (waves == 1 ? group : 0); row < a.rows; row += step) {
    T* sum = a.sum ? static_cast<T*>(a.sum) + row * a.sum_stride : nullptr;
    Y* y = static_cast<Y*>(a.y) + row * a.y_stride;
    u32x4 xr[C], rr[C], wr[C], br[C];
    R.load(static_cast<const T*>(a.x) + row * a.x_stride, xr);
    if (a.residual) R.load(static_cast<const T*>(a.residual) + row * a.residual_stride, rr);
    R.load(static_cast<const T*>(a.weight), wr);
    if (a.bias) R.load(static_cast<const T*>(a.bias), br);
    R.cut(xr);
    if (a.residual) R.cut(rr);
    float h[C][E];
#pragma unroll
    for (int i = 0; i < C; ++i) unpack(xr[i], h[i]);
    if (a.residual)
#pragma unroll
      for (int i = 0; i < C; ++i) {
        float u[E];
        unpack(rr[i], u);
#pragma unroll
        for (int e = 0; e < E; ++e) h[i][e] += u[e];
      }
    if (sum)
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const int64_t c = R.at(i);
        if (c < cols) store_some(sum + c, cols - c, h[i]);
      }
    Moments m = lane_moments(R, h, value_near<T, C>(h, weight));
    m.left = wave_sum_f32(m.left);
    m.squares = wave_sum_f32(m.squares);
    RowStats r;
    if (waves == 1) {
      r = own_stats(m, per_col, a.eps);
    } else {
      if (lane == 0) words[wave] = f32x4_lds{m.near, m.left, m.squares, 0.0f};
      __syncthreads();
      Moments q{0.0f, 0.0f, 0.0f};
      if (other < waves) {
        const f32x4_lds v = words[other];
        q = Moments{v.x, v.y, v.z};
      }
      float off;
      r = join_moments(q, n_other, per_col, a.eps, &off);
    }
    R.cut(wr);
    if (a.bias) R.cut(br);
#pragma unroll
    for (int i = 0; i < C; ++i) {
      float w[E], b[E];
      unpack(wr[i], w);
      if (a.bias) unpack(br[i], b);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        h[i][e] = ((h[i][e] - r.mean) - r.rest) * r.s;
        h[i][e] = a.bias ? __builtin_fmaf(h[i][e], w[e], b[e]) : h[i][e] * w[e];
      }
    }
    if constexpr (kFp8) {
      uint32_t top[C];
#pragma unroll
      for (int i = 0; i < C; ++i) {
        top[i] = 0;
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (R.at(i) + e < cols) top[i] = max(top[i], magnitude(h[i][e]));
      }
      if constexpr (kBlocks) {
#pragma unroll
        for (int i = 0; i < C; ++i) {
          const uint32_t scale = block_scale(block_max_u32<E>(top[i]));
          const float factor = block_factor(scale);
          const int64_t c = R.at(i);
          if (c % kScaleBlock == 0 && c < cols) static_cast<uint8_t*>(a.scales)[c / kScaleBlock * a.scales_stride + row] = (uint8_t)scale;
#pragma unroll
          for (int e = 0; e < E; ++e) h[i][e] *= factor;
        }
      } else {
#pragma unroll
        for (int i = 1; i < C; ++i) top[0] = max(top[0], top[i]);
        const float t = __builtin_bit_cast(float, row_max(top[0], scratch[0], wave, waves));
        const float factor = fp8_factor(t);
        if (lane == 0 && wave == 0) static_cast<float*>(a.scales)[row] = fp8_scale(t);
#pragma unroll
        for (int i = 0; i < C; ++i)
#pragma unroll
          for (int e = 0; e < E; ++e) h[i][e] *= factor;
      }
    }
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int64_t c = R.at(i);
      if (c < cols) store_some(y + c, cols - c, h[i]);
    }
    if (waves > 1) __syncthreads();  // the next row writes the words again
  }
}

// The same for rows that 16 waves cannot hold: read again, from the caches where they last, for each pass.
template <typename T, typename Y, bool kBlocks>
__global__ __launch_bounds__(1024) void layer_norm_long_kernel(LayerNormArgs a) {
  constexpr int E = kElems<T>;
  constexpr bool kFp8 = sizeof(Y) == 1;
  constexpr int64_t kStep = 64 * kWaves * E;
  __shared__ __align__(16) float scratch[4][kWaves];
  const int wave = threadIdx.x >> 6;
  const int64_t cols = a.cols, first = (int64_t)threadIdx.x * E;
  const T *weight = static_cast<const T*>(a.weight), *bias = static_cast<const T*>(a.bias);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* r = a.residual ? static_cast<const T*>(a.residual) + row * a.residual_stride : nullptr;
    T* sum = a.sum ? static_cast<T*>(a.sum) + row * a.sum_stride : nullptr;
    Y* y = static_cast<Y*>(a.y) + row * a.y_stride;
    auto read = [&](int64_t c, float (&v)[E]) __attribute__((always_inline)) {
      load_some(x + c, cols - c, v);
      if (r) {
        float u[E];
        load_some(r + c, cols - c, u);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] += u[e];
      }
    };
    float total = 0.0f;
    for (int64_t c = first; c < cols; c += kStep) {
      float v[E];
      read(c, v);
#pragma unroll
      for (int e = 0; e < E; ++e) total += v[e];
    }
    const float mean = row_sum(total, scratch[0], wave, kWaves) / (float)a.cols;
    float left = 0.0f, squares = 0.0f;
    for (int64_t c = first; c < cols; c += kStep) {
      float v[E];
      read(c, v);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float d = c + e < cols ? v[e] - mean : 0.0f;
        left += d;
        squares += d * d;
      }
    }
    left = row_sum(left, scratch[1], wave, kWaves);
    squares = row_sum(squares, scratch[2], wave, kWaves);
    const float rest = left / (float)a.cols, s = 1.0f / sqrtf((squares - left * rest) / (float)a.cols + a.eps);
    auto normed = [&](int64_t c, float (&v)[E]) __attribute__((always_inline)) {
      float w[E], b[E];
      load_some(weight + c, cols - c, w);
      if (bias) load_some(bias + c, cols - c, b);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        v[e] = ((v[e] - mean) - rest) * s;
        v[e] = bias ? __builtin_fmaf(v[e], w[e], b[e]) : v[e] * w[e];
      }
    };
    float factor = 1.0f;
    if constexpr (kFp8 && !kBlocks) {
      uint32_t top = 0;
      for (int64_t c = first; c < cols; c += kStep) {
        float v[E];
        read(c, v);
        normed(c, v);
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (c + e < cols) top = max(top, magnitude(v[e]));
      }
      const float t = __builtin_bit_cast(float, row_max(top, scratch[3], wave, kWaves));
      factor = fp8_factor(t);
      if (threadIdx.x == 0) static_cast<float*>(a.scales)[row] = fp8_scale(t);
    }
    // (a lane writes only what it alone has read; all lanes of a wave walk together, for the blocks' maxima)
    for (int64_t c0 = (int64_t)wave * 64 * E; c0 < cols; c0 += kStep) {
      const int64_t c = c0 + (int64_t)(threadIdx.x & 63) * E;
      float v[E];
      read(c, v);
      if (sum && c < cols) store_some(sum + c, cols - c, v);
      normed(c, v);
      if constexpr (kBlocks) {
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (c + e < cols) top = max(top, magnitude(v[e]));
        const uint32_t scale = block_scale(block_max_u32<E>(top));
        factor = block_factor(scale);
        if (c % kScaleBlock == 0 && c < cols) static_cast<uint8_t*>(a.scales)[c / kScaleBlock * a.scales_stride + row] = (uint8_t)scale;
      }
      if constexpr (kFp8)
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] *= factor;
      if (c < cols) store_some(y + c, cols - c, v);
    }
    __syncthreads();
  }
}

struct LayerNormGradArgs {
  const void *dy, *h, *weight, *dh;
  void* dx;
  float *weight_parts, *bias_parts;  // [gridDim.x][part_pitch] of dweight and of dbias, or NULL
  int64_t rows, dy_stride, h_stride, dh_stride, dx_stride, part_pitch;
  int32_t cols;
  float eps;
};

// A workgroup's rows are blockIdx.x, + gridDim.x, ...; with kAhead the next row's operands are asked for before this one's sums.
template <typename T, int C, bool kAhead>
__global__ __launch_bounds__(1024) void layer_norm_grad_kernel(LayerNormGradArgs a, int waves) {
  constexpr int E = kElems<T>;
  __shared__ __align__(16) f32x4_lds words[2][kWaves];
  __shared__ float more[2][kWaves];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t cols = a.cols;
  const Row<T, C> R{cols, waves, wave, lane};
  const int other = lane & (kWaves - 1);
  const float weight = near_weight<E>(cols, wave), n_other = other < waves ? wave_count<E, C>(cols, waves, other) : 0.0f;
  const float per_col = 1.0f / (float)a.cols;
  float dw[C][E], db[C][E];
#pragma unroll
  for (int i = 0; i < C; ++i)
#pragma unroll
    for (int e = 0; e < E; ++e) dw[i][e] = db[i][e] = 0.0f;
  u32x4 wr[C], hr[C], dr[C], ur[C];
  auto load = [&](int64_t row) __attribute__((always_inline)) {
    R.load(static_cast<const T*>(a.h) + row * a.h_stride, hr);
    R.load(static_cast<const T*>(a.dy) + row * a.dy_stride, dr);
    if (a.dh && a.dx) R.load(static_cast<const T*>(a.dh) + row * a.dh_stride, ur);
  };
  R.load(static_cast<const T*>(a.weight), wr);
  if constexpr (kAhead) load(blockIdx.x);
  R.cut(wr);
  int flip = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    if constexpr (!kAhead) load(row);
    R.cut(hr);
    R.cut(dr);
    float h[C][E], dy[C][E];
    u32x4 uv[C];
#pragma unroll
    for (int i = 0; i < C; ++i) {
      unpack(hr[i], h[i]);
      unpack(dr[i], dy[i]);
      uv[i] = ur[i];
    }
    if constexpr (kAhead)
      if (row + gridDim.x < a.rows) load(row + gridDim.x);
    Moments m = lane_moments(R, h, value_near<T, C>(h, weight));
    float g_sum = 0.0f, gd_sum = 0.0f;  // of g and of g d (dy is zero past the end)
#pragma unroll
    for (int i = 0; i < C; ++i) {
      float w[E];
      unpack(wr[i], w);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float g = dy[i][e] * w[e];
        g_sum += g;
        gd_sum += g * (h[i][e] - m.near);
      }
    }
    m.left = wave_sum_f32(m.left);
    m.squares = wave_sum_f32(m.squares);
    g_sum = wave_sum_f32(g_sum);
    gd_sum = wave_sum_f32(gd_sum);
    RowStats r;
    if (waves == 1) {
      r = own_stats(m, per_col, a.eps);
      gd_sum -= r.rest * g_sum;
    } else {
      if (lane == 0) {
        words[flip][wave] = f32x4_lds{m.near, m.left, m.squares, g_sum};
        more[flip][wave] = gd_sum;
      }
      __syncthreads();  // (two sets in turn: a wave writes a set again only past the barrier of the row between)
      f32x4_lds v = {0.0f, 0.0f, 0.0f, 0.0f};
      float gd = 0.0f, off;
      if (other < waves) {
        v = words[flip][other];
        gd = more[flip][other];
      }
      flip ^= 1;
      r = join_moments(Moments{v.x, v.y, v.z}, n_other, per_col, a.eps, &off);
      g_sum = row16_sum_f32(v.w);
      gd_sum = row16_sum_f32(__builtin_fmaf(off, v.w, gd)) - r.rest * g_sum;
    }
    const float g_mean = g_sum * per_col;
    const float along = r.s * (r.s * (gd_sum * per_col));  // mean(g u) s (s^2 alone may be no float where eps is 0)
    T* dx = a.dx ? static_cast<T*>(a.dx) + row * a.dx_stride : nullptr;
    if (dx && a.dh) R.cut(uv);
#pragma unroll
    for (int i = 0; i < C; ++i) {
      float o[E], w[E];
      unpack(wr[i], w);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float d = (h[i][e] - r.mean) - r.rest;
        dw[i][e] += dy[i][e] * (d * r.s);
        db[i][e] += dy[i][e];
        o[e] = r.s * (dy[i][e] * w[e] - g_mean - d * along);
      }
      if (dx) {
        if (a.dh) {
          float u[E];
          unpack(uv[i], u);
#pragma unroll
          for (int e = 0; e < E; ++e) o[e] += u[e];
        }
        const int64_t c = R.at(i);
        if (c < cols) store_some(dx + c, cols - c, o);
      }
    }
  }
  auto leave = [&](float* parts, const float (&v)[C][E]) __attribute__((always_inline)) {
    float* part = parts + (int64_t)blockIdx.x * a.part_pitch;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int64_t c = R.at(i);
#pragma unroll
      for (int e = 0; e < E; e += 4)
        if (c + e < cols) store_some(part + c + e, cols - c - e, *reinterpret_cast<const float (*)[4]>(v[i] + e));
    }
  };
  if (a.weight_parts) leave(a.weight_parts, dw);
  if (a.bias_parts) leave(a.bias_parts, db);
}

// The same for rows that a workgroup cannot hold: read three times, and the parts kept in memory.
template <typename T>
__global__ __launch_bounds__(1024) void layer_norm_grad_long_kernel(LayerNormGradArgs a) {
  constexpr int E = kElems<T>;
  constexpr int64_t kStep = 64 * kWaves * E;
  __shared__ __align__(16) float scratch[5][kWaves];
  const int wave = threadIdx.x >> 6;
  const int64_t cols = a.cols, first = (int64_t)threadIdx.x * E;
  const T* weight = static_cast<const T*>(a.weight);
  float* weight_part = a.weight_parts ? a.weight_parts + (int64_t)blockIdx.x * a.part_pitch : nullptr;
  float* bias_part = a.bias_parts ? a.bias_parts + (int64_t)blockIdx.x * a.part_pitch : nullptr;
  bool fresh = true;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* dy = static_cast<const T*>(a.dy) + row * a.dy_stride;
    const T* h = static_cast<const T*>(a.h) + row * a.h_stride;
    const T* dh = a.dh ? static_cast<const T*>(a.dh) + row * a.dh_stride : nullptr;
    T* dx = a.dx ? static_cast<T*>(a.dx) + row * a.dx_stride : nullptr;
    float hv[E], dv[E], wv[E];
    float total = 0.0f;
    for (int64_t c = first; c < cols; c += kStep) {
      load_some(h + c, cols - c, hv);
#pragma unroll
      for (int e = 0; e < E; ++e) total += hv[e];
    }
    const float mean = row_sum(total, scratch[0], wave, kWaves) / (float)a.cols;
    auto read = [&](int64_t c) __attribute__((always_inline)) {
      load_some(h + c, cols - c, hv);
      load_some(dy + c, cols - c, dv);
      load_some(weight + c, cols - c, wv);
    };
    float left = 0.0f, squares = 0.0f, g_sum = 0.0f, gd_sum = 0.0f;
    for (int64_t c = first; c < cols; c += kStep) {
      read(c);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float d = c + e < cols ? hv[e] - mean : 0.0f, g = dv[e] * wv[e];
        left += d;
        squares += d * d;
        g_sum += g;
        gd_sum += g * d;
      }
    }
    left = row_sum(left, scratch[1], wave, kWaves);
    squares = row_sum(squares, scratch[2], wave, kWaves);
    g_sum = row_sum(g_sum, scratch[3], wave, kWaves);
    gd_sum = row_sum(gd_sum, scratch[4], wave, kWaves);
    const float n = (float)a.cols, rest = left / n, s = 1.0f / sqrtf((squares - left * rest) / n + a.eps);
    const float g_mean = g_sum / n, along = s * (s * ((gd_sum - rest * g_sum) / n));
    for (int64_t c = first; c < cols; c += kStep) {
      read(c);
      float o[E], d[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        d[e] = (hv[e] - mean) - rest;
        o[e] = s * (dv[e] * wv[e] - g_mean - d[e] * along);
      }
      if (weight_part)  // (a thread's own columns)
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (c + e < cols) weight_part[c + e] = (fresh ? 0.0f : weight_part[c + e]) + dv[e] * (d[e] * s);
      if (bias_part)
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (c + e < cols) bias_part[c + e] = (fresh ? 0.0f : bias_part[c + e]) + dv[e];
      if (dx) {
        if (dh) {
          float u[E];
          load_some(dh + c, cols - c, u);
#pragma unroll
          for (int e = 0; e < E; ++e) o[e] += u[e];
        }
        store_some(dx + c, cols - c, o);
      }
    }
    fresh = false;
    __syncthreads();  // the next row writes the scratch words again
  }
}

// ---- rows in 8 bits with a scale for each 128 elements -----------------------------------------------------
// Memory-bound: 3 bytes an element of bf16, 5 of float32. A wave takes 64 chunks of 16 bytes of a row (512 elements of bf16, 256 of float32), whose blocks'
// maxima are found among 16 or 32 lanes, without LDS; its workgroup's 16 such pieces lie below each other, so that the scales, which run
// along the rows, are written 16 neighbouring bytes at a time.
struct QuantizeArgs {
  const void* x;
  uint8_t *q, *scales;
  int64_t rows, cols, x_stride, q_stride, scales_stride, across;  // across: pieces to a row
};
constexpr int kPieceRows = 16;
template <typename T>
__global__ __launch_bounds__(256) void quantize_blocks_kernel(QuantizeArgs a) {
  constexpr int E = kElems<T>, kBlocks = 64 * E / kScaleBlock, kEach = kPieceRows / 4;
  __shared__ uint8_t codes[kBlocks][kPieceRows];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t total = a.across * ((a.rows + kPieceRows - 1) / kPieceRows);
  for (int64_t t = blockIdx.x; t < total; t += gridDim.x) {
    const int64_t down = total <= UINT32_MAX ? (int64_t)((uint32_t)t / (uint32_t)a.across) : t / a.across;
    const int64_t row0 = down * kPieceRows, c0 = (t - down * a.across) * 64 * E, c = c0 + (int64_t)lane * E;
    float v[kEach][E];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int64_t row = row0 + wave * kEach + i;
      load_some(static_cast<const T*>(a.x) + row * a.x_stride + c, row < a.rows ? a.cols - c : 0, v[i]);
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int64_t row = row0 + wave * kEach + i;
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) top = max(top, magnitude(v[i][e]));  // (zeros past the end)
      const uint32_t scale = block_scale(block_max_u32<E>(top));
      const float factor = block_factor(scale);
#pragma unroll
      for (int e = 0; e < E; ++e) v[i][e] *= factor;
      if (row < a.rows && c < a.cols) store_some(a.q + row * a.q_stride + c, a.cols - c, v[i]);
      if (lane % (kScaleBlock / E) == 0) codes[lane / (kScaleBlock / E)][wave * kEach + i] = (uint8_t)scale;
    }
    __syncthreads();
    if (threadIdx.x < kBlocks * kPieceRows) {
      const int b = threadIdx.x / kPieceRows, i = threadIdx.x % kPieceRows;
      if (row0 + i < a.rows && c0 + b * kScaleBlock < a.cols) a.scales[(c0 / kScaleBlock + b) * a.scales_stride + row0 + i] = codes[b][i];
    }
    __syncthreads();
  }
}

// ---- host --------------------------------------------------------------------------------------------------
template <typename T, typename Y, int C, bool kBlocks>
int32_t launch_norm(dc_hip_ctx* ctx, const LayerNormArgs& a, int64_t chunks) {
  const int waves = waves_for(chunks, C);
  const int64_t groups = waves == 1 ? (a.rows + 3) / 4 : a.rows;
  layer_norm_kernel<T, Y, C, kBlocks>
      <<<(unsigned)std::min(groups, kMaxGrid), waves == 1 ? 256 : 64 * waves, 0, ctx->stream>>>(a, waves);
  return last_launch_status();
}

template <typename T, typename Y, bool kBlocks>
int32_t norm_by_shape(dc_hip_ctx* ctx, const LayerNormArgs& a) {
  const int64_t chunks = (a.cols + kElems<T> - 1) / kElems<T>;
  const bool wave = chunks > 64 && chunks <= 128 && (sizeof(T) == 2 || sizeof(Y) == 1);
  if (chunks <= 256 && !wave) return launch_norm<T, Y, 1, kBlocks>(ctx, a, chunks);
  if (chunks <= 1024) return launch_norm<T, Y, 2, kBlocks>(ctx, a, chunks);
  if (chunks <= 64 * 4 * kWaves) return launch_norm<T, Y, 4, kBlocks>(ctx, a, chunks);
  layer_norm_long_kernel<T, Y, kBlocks><<<(unsigned)std::min(a.rows, kMaxGrid), 64 * kWaves, 0, ctx->stream>>>(a);
  return last_launch_status();
}

template <typename T>
int32_t norm_by_output(dc_hip_ctx* ctx, const LayerNormArgs& a, bool fp8, bool blocks) {
  if (!fp8) return norm_by_shape<T, T, false>(ctx, a);
  return blocks ? norm_by_shape<T, uint8_t, true>(ctx, a) : norm_by_shape<T, uint8_t, false>(ctx, a);
}

template <typename T>
int32_t norm_grad_by_shape(dc_hip_ctx* ctx, const LayerNormGradArgs& a, int64_t grid, int c, int waves) {
  const unsigned g = (unsigned)grid;
  if (c == 1) layer_norm_grad_kernel<T, 1, true><<<g, 64 * waves, 0, ctx->stream>>>(a, waves);
  else if (c == 2) layer_norm_grad_kernel<T, 2, false><<<g, 64 * waves, 0, ctx->stream>>>(a, waves);
  else layer_norm_grad_long_kernel<T><<<g, 64 * kWaves, 0, ctx->stream>>>(a);
  return last_launch_status();
}

// 16-byte chunks of a row that a lane of the gradient's kernel holds (0: the long kernel).
int norm_grad_chunks(int64_t chunks) { return chunks <= 64 * kWaves ? 1 : chunks <= 128 * kWaves ? 2 : 0; }

}  // namespace

extern "C" {

DC_HIP_API int32_t dc_hip_layer_norm(dc_hip_ctx* ctx, const dc_layer_norm* args) {
  if (!args) return DC_ERR_INVALID_ARGUMENT;
  const dc_layer_norm& p = *args;
  DC_RETURN_IF(check_shape(p.rows, p.cols));
  const bool fp8 = p.y_dtype == DC_DTYPE_FP8, blocks = p.scale_block == kScaleBlock;
  if (!float_dtype(p.dtype) || (!fp8 && p.y_dtype != p.dtype)) return DC_ERR_INVALID_ARGUMENT;
  if (p.scale_block != 0 && !(fp8 && blocks)) return DC_ERR_INVALID_ARGUMENT;
  if (!(p.eps >= 0.0f) || (!fp8 && p.scales)) return DC_ERR_INVALID_ARGUMENT;
  if (fp8 && !p.scales && p.rows > 0 && !(blocks && p.cols == 0)) return DC_ERR_INVALID_ARGUMENT;
  if (p.rows > 0 && p.cols > 0) {
    if (!p.x || !p.weight || !p.y) return DC_ERR_INVALID_ARGUMENT;
    DC_RETURN_IF(check_rows(p.x, p.dtype, p.x_stride, p.rows, p.cols));
    DC_RETURN_IF(check_rows(p.y, p.y_dtype, p.y_stride, p.rows, p.cols));
    DC_RETURN_IF(check_rows(p.weight, p.dtype, p.cols, 1, p.cols));
    if (p.bias) DC_RETURN_IF(check_rows(p.bias, p.dtype, p.cols, 1, p.cols));
    if (p.residual) DC_RETURN_IF(check_rows(p.residual, p.dtype, p.residual_stride, p.rows, p.cols));
    if (p.sum) DC_RETURN_IF(check_rows(p.sum, p.dtype, p.sum_stride, p.rows, p.cols));
    if (blocks && p.cols > kScaleBlock && p.scales_stride < p.rows) return DC_ERR_DIMENSION;
  }
  if (!blocks && !aligned_to(p.scales, 4)) return DC_ERR_MISALIGNED;
  DC_CTX_ENTER(ctx);
  if (p.rows == 0 || p.cols == 0) return blocks ? DC_OK : empty_scales(ctx, static_cast<float*>(p.scales), p.rows);
  const LayerNormArgs a{p.x,        p.residual,        p.weight,     p.bias,     p.sum,           p.y,             p.scales, p.rows,
                        p.x_stride, p.residual_stride, p.sum_stride, p.y_stride, p.scales_stride, (int32_t)p.cols, p.eps};
  return p.dtype == DC_DTYPE_F32 ? norm_by_output<float>(ctx, a, fp8, blocks) : norm_by_output<bf16>(ctx, a, fp8, blocks);
}

DC_HIP_API int32_t dc_hip_layer_norm_backward(dc_hip_ctx* ctx, const dc_layer_norm_grad* args) {
  if (!args) return DC_ERR_INVALID_ARGUMENT;
  const dc_layer_norm_grad& p = *args;
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
  if (!aligned_to(p.dweight, 4) || !aligned_to(p.dbias, 4)) return DC_ERR_MISALIGNED;
  DC_CTX_ENTER(ctx);
  if (p.cols == 0 || (!p.dx && !p.dweight && !p.dbias)) return DC_OK;
  if (p.rows == 0) {
    for (float* out : {p.dweight, p.dbias})
      if (out) DC_RETURN_IF(zero_async(ctx, out, (size_t)p.cols * sizeof(float)));
    return DC_OK;
  }
  const int64_t elems = 16 / size_of(p.dtype), chunks = (p.cols + elems - 1) / elems;
  const int c = norm_grad_chunks(chunks), waves = c ? waves_for(chunks, c) : kWaves;
  const int per_cu = waves <= 2 ? 8 / waves : c > 1 ? 1 : std::max(1, 15 / waves);
  const int64_t held = per_cu * (int64_t)std::max(1, ctx->cu_count);  // workgroups
  const int64_t each = (p.rows + held - 1) / held, grid = each <= 4 ? (p.rows + each - 1) / each : held;
  const int outs = (p.dweight ? 1 : 0) + (p.dbias ? 1 : 0);
  const int64_t pitch = (p.cols + 3) / 4 * 4;
  float *weight_parts = nullptr, *bias_parts = nullptr;
  if (outs > 0) {
    DC_RETURN_IF(ensure_partials(ctx, (size_t)(grid * outs * pitch) * sizeof(float)));
    float* parts = static_cast<float*>(ctx->partials);
    if (p.dweight) weight_parts = parts;
    if (p.dbias) bias_parts = parts + (outs - 1) * pitch;
  }
  const LayerNormGradArgs a{p.dy,        p.h,         p.weight,    p.dh,         p.dx,            weight_parts, bias_parts, p.rows,
                            p.dy_stride, p.h_stride, p.dh_stride, p.dx_stride, outs * pitch, (int32_t)p.cols, p.eps};
  DC_RETURN_IF(p.dtype == DC_DTYPE_F32 ? norm_grad_by_shape<float>(ctx, a, grid, c, waves) : norm_grad_by_shape<bf16>(ctx, a, grid, c, waves));
  if (outs == 0) return DC_OK;
  return launch_column_sums_of(ctx, static_cast<const float*>(ctx->partials), outs * pitch, pitch, p.dweight ? p.dweight : p.dbias,
                               outs > 1 ? p.dbias : nullptr, grid, p.cols);
}

DC_HIP_API int32_t dc_hip_quantize_fp8_blocks(dc_hip_ctx* ctx, const void* x, int32_t dtype, int64_t x_stride, uint8_t* q,
                                              int64_t q_stride, uint8_t* scales, int64_t scales_stride, int64_t rows, int64_t cols) {
  DC_RETURN_IF(check_shape(rows, cols));
  if (!float_dtype(dtype)) return DC_ERR_INVALID_ARGUMENT;
  if (rows > 0 && cols > 0) {
    if (!x || !q || !scales) return DC_ERR_INVALID_ARGUMENT;
    DC_RETURN_IF(check_rows(x, dtype, x_stride, rows, cols));
    DC_RETURN_IF(check_rows(q, DC_DTYPE_FP8, q_stride, rows, cols));
    if (cols > kScaleBlock && scales_stride < rows) return DC_ERR_DIMENSION;
  }
  DC_CTX_ENTER(ctx);
  if (rows == 0 || cols == 0) return DC_OK;
  const int64_t piece = 64 * 16 / size_of(dtype), across = (cols + piece - 1) / piece;
  const QuantizeArgs a{x, q, scales, rows, cols, x_stride, q_stride, scales_stride, across};
  const unsigned grid = (unsigned)std::min(across * ((rows + kPieceRows - 1) / kPieceRows), kMaxGrid);
  if (dtype == DC_DTYPE_F32) quantize_blocks_kernel<float><<<grid, 256, 0, ctx->stream>>>(a);
  else quantize_blocks_kernel<bf16><<<grid, 256, 0, ctx->stream>>>(a);
  return last_launch_status();
}

}  // extern "C"
