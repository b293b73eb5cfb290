// dc_norm.hip — RMS norm with the residual's addition, its gradients, and rows in 8 bits with scales.
//
// Forward, a row at a time: h = x + r, s = 1 / sqrt(mean(h^2) + eps), y = h w s. Memory-bound: 8 bytes an element in
// bf16 (x, r in; h, y out), 7 with y in 8 bits. A row stays in registers between its one read and its write, so nothing
// is read twice: as many waves as it needs hold it in C 16-byte chunks a lane, and their sums meet in LDS. Rows too long
// for 16 waves are read again from the caches for each pass.
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

// Waves that share a row, at most: each leaves its sum in a word of LDS, and every wave adds the words in order, those of
// waves that are not there too (zeros from the start of the kernel): few wide reads and no loop.
constexpr int kWaves = 16;

__device__ inline float add_words(const float* scratch, int waves) {
  const dc::f32x4* q = reinterpret_cast<const dc::f32x4*>(scratch);
  const dc::f32x4 a = q[0], b = q[1];
  float v = ((a.x + a.y) + (a.z + a.w)) + ((b.x + b.y) + (b.z + b.w));
  if (waves > 8) {
    const dc::f32x4 c = q[2], d = q[3];
    v += ((c.x + c.y) + (c.z + c.w)) + ((d.x + d.y) + (d.z + d.w));
  }
  return v;
}

// Sum (or unsigned maximum) over the `waves` waves that share a row, in every lane. `scratch`: nobody writes it again
// before the caller's next barrier.
__device__ inline float row_sum(float v, float* scratch, int wave, int waves) {
  v = dc::wave_sum_f32(v);
  if (waves > 1) {
    if ((threadIdx.x & 63) == 0) scratch[wave] = v;
    __syncthreads();
    v = add_words(scratch, waves);
  }
  return v;
}
__device__ inline uint32_t row_max(uint32_t v, float* scratch, int wave, int waves) {
  v = dc::wave_max_u32(v);
  if (waves > 1) {
    uint32_t* s = reinterpret_cast<uint32_t*>(scratch);
    if ((threadIdx.x & 63) == 0) s[wave] = v;
    __syncthreads();
    const dc::u32x4* q = reinterpret_cast<const dc::u32x4*>(scratch);
    const dc::u32x4 a = q[0], b = q[1], c = q[2], d = q[3];
    v = max(max(max(max(a.x, a.y), max(a.z, a.w)), max(max(b.x, b.y), max(b.z, b.w))),
            max(max(max(c.x, c.y), max(c.z, c.w)), max(max(d.x, d.y), max(d.z, d.w))));
  }
  return v;
}
// Zeros in `sets` sets of words, before their first use.
__device__ inline void clear_words(float (*scratch)[kWaves], int sets, int waves) {
  if (waves > 1) {
    if ((int)threadIdx.x < sets * kWaves) scratch[0][threadIdx.x] = 0.0f;
    __syncthreads();
  }
}

// The chunks c_i = ((i waves + wave) 64 + lane) E, i < C, of a row of `cols` elements, as they lie in memory, zeros past its
// end. No branch stands between the loads, so that all of them are in flight at once: a chunk that reaches past the end is
// cut out of the row's last 16 bytes, one beyond it loads those too, to no effect.
template <typename T, int C>
struct Row {
  static constexpr int E = kElems<T>;
  int64_t cols;
  int waves, wave, lane;
  __device__ inline int64_t at(int i) const { return (int64_t)((i * waves + wave) * 64 + lane) * E; }
  __device__ inline void load(const T* p, dc::u32x4 (&raw)[C]) const {
    if (cols >= E) {
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const int64_t c = at(i);
        raw[i] = dc::load_raw(p + (c < cols - E ? c : cols - E));
      }
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i) {
        float v[E];
        dc::load_some(p, i == 0 && wave == 0 && lane == 0 ? cols : 0, v);
        raw[i] = dc::u32x4{0, 0, 0, 0};
        if constexpr (E == 4) raw[i] = __builtin_bit_cast(dc::u32x4, dc::f32x4{v[0], v[1], v[2], v[3]});
        else
#pragma unroll
          for (int e = 0; e < 4; ++e) raw[i][e] = dc::pack_bf16(v[2 * e], v[2 * e + 1]);
      }
    }
  }
  // What load() left of the row's last 16 bytes in the chunks at and past its end.
  __device__ inline void cut(dc::u32x4 (&raw)[C]) const {
    if (cols < E) return;
#pragma unroll
    for (int i = 0; i < C; ++i)
      if ((int64_t)((i * waves + wave) * 64 + 64) * E > cols) {  // (uniform)
        const int64_t past = at(i) - (cols - E);
        if (past > 0) raw[i] = dc::shift_down(raw[i], past * (int64_t)sizeof(T));
      }
  }
};

// A row a workgroup; or, where a wave holds a row, one for each of its four waves.
// kNorm false: y = x itself (a conversion to 8 bits), no norm, no weight. Memory-bound too, 3 bytes an element of bf16 and 5 of float32; the row's
// maximum is a barrier between its read and its write. us with the call (TB/s), bf16 and float32: 16384×4096 42.4 (4.75), 67.0 (5.0);
// 2048×4096 7.8 (3.2), 9.4 (4.5); 8191×2050 16.5 (3.05), 23.1 (3.6); 8×4096 4.3, 4.4, of which the call is 3.7.
template <typename T, typename Y, int C, bool kNorm>
__global__ __launch_bounds__(C == 4 ? 1024 : 512) void rms_norm_kernel(NormArgs a, int waves) {
  constexpr int E = kElems<T>;
  constexpr bool kFp8 = sizeof(Y) == 1;
  __shared__ __align__(16) float scratch[2][kWaves];
  const int lane = threadIdx.x & 63, group = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = waves == 1 ? 0 : group;
  const int64_t cols = a.cols;
  const Row<T, C> R{cols, waves, wave, lane};
  clear_words(scratch, 2, waves);
  const int per = waves == 1 ? 4 : 1;
  const int64_t step = (int64_t)gridDim.x * per;
  for (int64_t row = (int64_t)blockIdx.x * per + (waves == 1 ? group : 0); row < a.rows; row += step) {
    T* sum = a.sum ? static_cast<T*>(a.sum) + row * a.sum_stride : nullptr;
    Y* y = static_cast<Y*>(a.y) + row * a.y_stride;
    dc::u32x4 xr[C], rr[C], wr[C];
    R.load(static_cast<const T*>(a.x) + row * a.x_stride, xr);
    if (a.residual) R.load(static_cast<const T*>(a.residual) + row * a.residual_stride, rr);
    if constexpr (kNorm) R.load(static_cast<const T*>(a.weight), wr);
    R.cut(xr);
    if (a.residual) R.cut(rr);
    float h[C][E];
#pragma unroll
    for (int i = 0; i < C; ++i) dc::unpack(xr[i], h[i]);
    if (a.residual)
#pragma unroll
      for (int i = 0; i < C; ++i) {
        float u[E];
        dc::unpack(rr[i], u);
#pragma unroll
        for (int e = 0; e < E; ++e) h[i][e] += u[e];
      }
    if constexpr (kNorm) {
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < C; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) ss += h[i][e] * h[i][e];
      if (sum)
#pragma unroll
        for (int i = 0; i < C; ++i) {
          const int64_t c = R.at(i);
          if (c < cols) dc::store_some(sum + c, cols - c, h[i]);
        }
      const float s = 1.0f / sqrtf(row_sum(ss, scratch[0], wave, waves) / (float)a.cols + a.eps);
      R.cut(wr);
#pragma unroll
      for (int i = 0; i < C; ++i) {
        float w[E];
        dc::unpack(wr[i], w);
#pragma unroll
        for (int e = 0; e < E; ++e) h[i][e] = h[i][e] * s * w[e];
      }
    }
    if constexpr (kFp8) {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < C; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (R.at(i) + e < cols) top = max(top, dc::magnitude(h[i][e]));
      const float t = __builtin_bit_cast(float, row_max(top, scratch[1], wave, waves));
      const float factor = dc::fp8_factor(t);
      if (lane == 0 && wave == 0) a.scales[row] = dc::fp8_scale(t);
#pragma unroll
      for (int i = 0; i < C; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) h[i][e] *= factor;
    }
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int64_t c = R.at(i);
      if (c < cols) dc::store_some(y + c, cols - c, h[i]);
    }
    if (waves > 1) __syncthreads();  // the next row writes the scratch words again
  }
}

// The same for rows that 16 waves cannot hold: read again, from the caches where they last, for each pass.
template <typename T, typename Y, bool kNorm>
__global__ __launch_bounds__(1024) void rms_norm_long_kernel(NormArgs a) {
  constexpr int E = kElems<T>;
  constexpr bool kFp8 = sizeof(Y) == 1;
  constexpr int64_t kStep = 64 * kWaves * E;
  __shared__ __align__(16) float scratch[2][kWaves];
  const int wave = threadIdx.x >> 6;
  const int64_t cols = a.cols, first = (int64_t)threadIdx.x * E;
  const T* weight = static_cast<const T*>(a.weight);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* r = a.residual ? static_cast<const T*>(a.residual) + row * a.residual_stride : nullptr;
    T* sum = a.sum ? static_cast<T*>(a.sum) + row * a.sum_stride : nullptr;
    Y* y = static_cast<Y*>(a.y) + row * a.y_stride;
    float s = 1.0f;
    auto read = [&](int64_t c, float (&v)[E]) __attribute__((always_inline)) {
      dc::load_some(x + c, cols - c, v);
      if (r) {
        float u[E];
        dc::load_some(r + c, cols - c, u);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] += u[e];
      }
    };
    auto normed = [&](int64_t c, float (&v)[E]) __attribute__((always_inline)) {
      if constexpr (kNorm) {
        float w[E];
        dc::load_some(weight + c, cols - c, w);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = v[e] * s * w[e];
      }
    };
    if constexpr (kNorm) {
      float ss = 0.0f;
      for (int64_t c = first; c < cols; c += kStep) {
        float v[E];
        read(c, v);
#pragma unroll
        for (int e = 0; e < E; ++e) ss += v[e] * v[e];
      }
      s = 1.0f / sqrtf(row_sum(ss, scratch[0], wave, kWaves) / (float)a.cols + a.eps);
    }
    float factor = 1.0f;
    if constexpr (kFp8) {
      uint32_t top = 0;
      for (int64_t c = first; c < cols; c += kStep) {
        float v[E];
        read(c, v);
        normed(c, v);
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (c + e < cols) top = max(top, dc::magnitude(v[e]));
      }
      const float t = __builtin_bit_cast(float, row_max(top, scratch[1], wave, kWaves));
      factor = dc::fp8_factor(t);
      if (threadIdx.x == 0) a.scales[row] = dc::fp8_scale(t);
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
    __syncthreads();
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

// The sums of h^2 and g h over the waves that share a row; two sets of words in turn, so that one barrier a row does: a
// wave writes a set again only past the barrier of the row between.
__device__ inline void row_sums(float& hh, float& gh, float (*scratch)[kWaves], int lane, int wave, int waves) {
  hh = dc::wave_sum_f32(hh);
  gh = dc::wave_sum_f32(gh);
  if (waves > 1) {
    if (lane == 0) {
      scratch[0][wave] = hh;
      scratch[1][wave] = gh;
    }
    __syncthreads();
    hh = add_words(scratch[0], waves);
    gh = add_words(scratch[1], waves);
  }
}

// A workgroup's rows are blockIdx.x, + gridDim.x, ...; with kAhead the next row's operands are asked for before this one's sums
// (without, sixteen floats of each operand a lane leave registers for 16 waves).
// Workgroups a CU: as many waves as hide a row's latency, and no more, as each workgroup leaves a row of dweight's parts to be
// added. Measured, us for 1 / 2 / 3 / 4 workgroups of a row's waves a CU: 8192×4096 51.4 / 55.5 (8 waves; 5.2 TB/s), 8191×2050 45 /
// 34.9 / 32.8 (5 waves; 4.1 TB/s); 16384×512 with 8 of one wave 19.1, with 16 23.2.
template <typename T, int C, bool kAhead>
__global__ __launch_bounds__(C == 4 && kAhead ? 512 : 1024) void rms_norm_grad_kernel(NormGradArgs a, int waves) {
  constexpr int E = kElems<T>;
  __shared__ __align__(16) float scratch[4][kWaves];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t cols = a.cols;
  const Row<T, C> R{cols, waves, wave, lane};
  clear_words(scratch, 4, waves);
  float acc[C][E];
#pragma unroll
  for (int i = 0; i < C; ++i)
#pragma unroll
    for (int e = 0; e < E; ++e) acc[i][e] = 0.0f;
  dc::u32x4 wr[C], hr[C], dr[C], ur[C];
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
    float hv[C][E], dv[C][E];
    dc::u32x4 uv[C];
    float hh = 0.0f, gh = 0.0f;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      float wv[E];
      dc::unpack(hr[i], hv[i]);
      dc::unpack(dr[i], dv[i]);
      dc::unpack(wr[i], wv);
      uv[i] = ur[i];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        hh += hv[i][e] * hv[i][e];
        gh += dv[i][e] * wv[e] * hv[i][e];
      }
    }
    if constexpr (kAhead)
      if (row + gridDim.x < a.rows) load(row + gridDim.x);
    row_sums(hh, gh, scratch + 2 * flip, lane, wave, waves);
    flip ^= 1;
    const float s = 1.0f / sqrtf(hh / (float)a.cols + a.eps);
    const float mean = s * (s * (gh / (float)a.cols));  // mean(g h s) s (s^2 alone may be no float where eps is 0)
    if (a.dx) {
      T* dx = static_cast<T*>(a.dx) + row * a.dx_stride;
      if (a.dh) R.cut(uv);
#pragma unroll
      for (int i = 0; i < C; ++i) {
        float o[E], wv[E];
        dc::unpack(wr[i], wv);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = s * (dv[i][e] * wv[e] - hv[i][e] * mean);
        if (a.dh) {
          float u[E];
          dc::unpack(uv[i], u);
#pragma unroll
          for (int e = 0; e < E; ++e) o[e] += u[e];
        }
        const int64_t c = R.at(i);
        if (c < cols) dc::store_some(dx + c, cols - c, o);
      }
    }
#pragma unroll
    for (int i = 0; i < C; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e) acc[i][e] += dv[i][e] * (hv[i][e] * s);
  }
  if (a.parts) {
    float* part = a.parts + (int64_t)blockIdx.x * cols;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int64_t c = R.at(i);
#pragma unroll
      for (int e = 0; e < E; e += 4)
        if (c + e < cols) dc::store_some(part + c + e, cols - c - e, *reinterpret_cast<const float (*)[4]>(acc[i] + e));
    }
  }
}

// The same for rows that a workgroup cannot hold: read twice, and dweight's part kept in memory.
template <typename T>
__global__ __launch_bounds__(1024) void rms_norm_grad_long_kernel(NormGradArgs a) {
  constexpr int E = kElems<T>;
  __shared__ __align__(16) float scratch[4][kWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t cols = a.cols;
  const T* weight = static_cast<const T*>(a.weight);
  float* part = a.parts ? a.parts + (int64_t)blockIdx.x * cols : nullptr;
  int flip = 0;
  bool fresh = true;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* dy = static_cast<const T*>(a.dy) + row * a.dy_stride;
    const T* h = static_cast<const T*>(a.h) + row * a.h_stride;
    const T* dh = a.dh ? static_cast<const T*>(a.dh) + row * a.dh_stride : nullptr;
    T* dx = a.dx ? static_cast<T*>(a.dx) + row * a.dx_stride : nullptr;
    float hh = 0.0f, gh = 0.0f;
    float hv[E], dv[E], wv[E];
    auto read = [&](int64_t c) __attribute__((always_inline)) {
      dc::load_some(h + c, cols - c, hv);
      dc::load_some(dy + c, cols - c, dv);
      dc::load_some(weight + c, cols - c, wv);
    };
    for (int64_t c = (int64_t)threadIdx.x * E; c < cols; c += 64 * kWaves * E) {
      read(c);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        hh += hv[e] * hv[e];
        gh += dv[e] * wv[e] * hv[e];
      }
    }
    row_sums(hh, gh, scratch + 2 * flip, lane, wave, kWaves);
    flip ^= 1;
    const float s = 1.0f / sqrtf(hh / (float)a.cols + a.eps);
    const float mean = s * (s * (gh / (float)a.cols));
    for (int64_t c = (int64_t)threadIdx.x * E; c < cols; c += 64 * kWaves * E) {
      read(c);
      if (dx) {
        float o[E], u[E];
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = s * (dv[e] * wv[e] - hv[e] * mean);
        if (dh) {
          dc::load_some(dh + c, cols - c, u);
#pragma unroll
          for (int e = 0; e < E; ++e) o[e] += u[e];
        }
        dc::store_some(dx + c, cols - c, o);
      }
      if (part)  // (a thread's own columns)
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (c + e < cols) part[c + e] = (fresh ? 0.0f : part[c + e]) + dv[e] * (hv[e] * s);
    }
    fresh = false;
  }
}

// out[c] = parts[0][c] + ... + parts[count - 1][c]: 16 columns a workgroup, 64 threads a column that each add every 64th
// part, then those sums in order (16 columns: enough workgroups for rows of a few thousand).
constexpr int kSumGroups = 64, kSumCols = 16;
__global__ __launch_bounds__(kSumCols * kSumGroups) void column_sums_kernel(const float* __restrict__ parts, float* __restrict__ out,
                                                                            int64_t count, int64_t cols) {
  __shared__ float sums[kSumGroups][kSumCols + 1];
  const int lane = threadIdx.x % kSumCols, g = threadIdx.x / kSumCols;
  const int64_t c = (int64_t)blockIdx.x * kSumCols + lane;
  float v = 0.0f;
  if (c < cols)
    for (int64_t i = g; i < count; i += 8 * kSumGroups) {  // (eight in flight, the last ones too)
      float u[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int64_t at = i + j * kSumGroups;
        u[j] = parts[(at < count ? at : count - 1) * cols + c];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) v += i + j * kSumGroups < count ? u[j] : 0.0f;
    }
  sums[g][lane] = v;
  __syncthreads();
  if (g < 4) {  // (a wave: 16 columns, 4 quarters of the sums)
    v = sums[16 * g][lane];
#pragma unroll
    for (int i = 1; i < 16; ++i) v += sums[16 * g + i][lane];
    sums[16 * g][lane] = v;
  }
  __syncthreads();
  if (g == 0 && c < cols) out[c] = ((v + sums[16][lane]) + sums[32][lane]) + sums[48][lane];
}

constexpr int64_t kMaxCols = int64_t(1) << 25;
constexpr int64_t kMaxGrid = 1 << 20;  // rows beyond are walked over by the same workgroups

// Waves that hold a row of `chunks` 16-byte chunks, C to a lane.
int waves_for(int64_t chunks, int c) { return (int)((chunks + 64 * c - 1) / (64 * c)); }

template <typename T, typename Y, int C, bool kNorm>
int32_t launch_norm(dc_hip_ctx* ctx, const NormArgs& a, int64_t chunks) {
  const int waves = waves_for(chunks, C);
  const int64_t groups = waves == 1 ? (a.rows + 3) / 4 : a.rows;
  rms_norm_kernel<T, Y, C, kNorm>
      <<<(unsigned)std::min(groups, kMaxGrid), waves == 1 ? 256 : 64 * waves, 0, ctx->stream>>>(a, waves);
  return dc::last_launch_status();
}

// Measured, us, bf16 with a residual (TB/s): 16384×4096 with C = 2 and 4 waves 89.8 (5.98), C = 1 and 8 waves 88.8, a wave a row
// (C = 8) 100; to 8 bits 81.8 (5.75), 92.1, 106, as its second sum over the row is another barrier; 8191×2050, whose
// rows lie at 4-byte boundaries, 27.2 (4.95), C = 1 29.8; 16384×512 11.4 (5.9). Rows of 65 to 128 chunks: a wave each with C = 2, so no
// barrier, but where rows are read and written in float32; C = 1 / 2, with the call: 16384×1001 30.0 / 26.4, to 8 bits 28.8 / 24.6,
// 16384×576 to 8 bits 23.4 / 18.6, 4000×640 6.7 / 5.9, 2000×1001 5.4 / 5.6; float32 to 8 bits 4000×512 8.1 / 6.9, 16384×384 21.5 / 22.4.
template <typename T, typename Y, bool kNorm>
int32_t norm_by_shape(dc_hip_ctx* ctx, const NormArgs& a) {
  const int64_t chunks = (a.cols + kElems<T> - 1) / kElems<T>;
  const bool wave = chunks > 64 && chunks <= 128 && (sizeof(T) == 2 || sizeof(Y) == 1);
  if (chunks <= 256 && !wave) return launch_norm<T, Y, 1, kNorm>(ctx, a, chunks);
  if (chunks <= 1024) return launch_norm<T, Y, 2, kNorm>(ctx, a, chunks);
  if (chunks <= 64 * 4 * kWaves) return launch_norm<T, Y, 4, kNorm>(ctx, a, chunks);
  rms_norm_long_kernel<T, Y, kNorm><<<(unsigned)std::min(a.rows, kMaxGrid), 64 * kWaves, 0, ctx->stream>>>(a);
  return dc::last_launch_status();
}

template <typename T>
int32_t norm_grad_by_shape(dc_hip_ctx* ctx, const NormGradArgs& a, int64_t grid, int c, int waves) {
  const unsigned g = (unsigned)grid;
  constexpr bool kF32 = sizeof(T) == 4;
  if (c == 1) rms_norm_grad_kernel<T, 1, true><<<g, 64 * waves, 0, ctx->stream>>>(a, waves);
  else if (kF32 && c == 2) rms_norm_grad_kernel<float, 2, true><<<g, 64 * waves, 0, ctx->stream>>>(a, waves);
  else if (c == 4) rms_norm_grad_kernel<T, 4, !kF32><<<g, 64 * waves, 0, ctx->stream>>>(a, waves);
  else rms_norm_grad_long_kernel<T><<<g, 64 * kWaves, 0, ctx->stream>>>(a);
  return dc::last_launch_status();
}

// 16-byte chunks of a row that a lane of the gradient's kernel holds (0: the long kernel). Few, and many waves: four of bf16
// take all 256 registers; of float32, two do better than one with 16 waves. One workgroup a CU for more than one chunk, so that
// fewer parts of dweight are left. Measured, us, with the call, for 1 / 2 / 4 chunks: bf16 8000×8192 103 / 138 / 110, 300×8192 13.3 / 14.9 /
// 18.1, 3000×12000 - / 79 / 69, 4000×16384 - / 127 / 112; float32 8000×4096 111 / 97 / 103, 1443×5056 - / 29.0 / 29.4 (two
// workgroups of 4 chunks a CU 36.5), 3000×6000 - / 59 / 59; 2000×12000 101 with 4, 140 by the long kernel, 300×16384 34, 46.
int norm_grad_chunks(bool f32, int64_t chunks) {
  if (f32) return chunks <= 512 ? 1 : chunks <= 2048 ? 2 : chunks <= 4096 ? 4 : 0;
  return chunks <= 1024 ? 1 : chunks <= 2048 ? 4 : 0;
}

bool float_dtype(int32_t t) { return t == DC_DTYPE_F32 || t == DC_DTYPE_BF16; }
int64_t size_of(int32_t t) { return t == DC_DTYPE_F32 ? 4 : t == DC_DTYPE_BF16 ? 2 : 1; }
bool aligned_to(const void* p, int64_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }

// Rows of nothing: their maxima, and so their scales, are zeros.
int32_t empty_scales(dc_hip_ctx* ctx, float* scales, int64_t rows) {
  return scales && rows > 0 ? dc::zero_async(ctx, scales, (size_t)rows * sizeof(float)) : DC_OK;
}

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
  // (1024 work items for 16 columns, at most kMaxCols of them: within the 2^32 of a launch)
  column_sums_kernel<<<(unsigned)((cols + kSumCols - 1) / kSumCols), kSumCols * kSumGroups, 0, ctx->stream>>>(parts, out, count, cols);
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
  }
  if (!aligned_to(p.scales, 4)) return DC_ERR_MISALIGNED;
  DC_CTX_ENTER(ctx);
  if (p.rows == 0 || p.cols == 0) return empty_scales(ctx, p.scales, p.rows);
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
  const int64_t elems = 16 / size_of(p.dtype), chunks = (p.cols + elems - 1) / elems;
  const int c = norm_grad_chunks(p.dtype == DC_DTYPE_F32, chunks), waves = c ? waves_for(chunks, c) : kWaves;
  const int per_cu = waves <= 2 ? 8 / waves : c > 1 ? 1 : std::max(1, 15 / waves);
  const int64_t held = per_cu * (int64_t)std::max(1, ctx->cu_count);  // workgroups
  // (Few rows: no more parts than workgroups of that many rows each leave. us, 900×3000 14.3 / 13.7; of many rows
  // it would leave CUs idle: 8191×2050 32.4 / 33.1. A workgroup a row up to two rows each: 17.8, 17.0.)
  const int64_t each = (p.rows + held - 1) / held, grid = each <= 4 ? (p.rows + each - 1) / each : held;
  float* parts = nullptr;
  if (p.dweight) {
    DC_RETURN_IF(dc::ensure_partials(ctx, (size_t)(grid * p.cols) * sizeof(float)));
    parts = static_cast<float*>(ctx->partials);
  }
  const NormGradArgs a{p.dy,   p.h,         p.weight,   p.dh,        p.dx,        parts,
                       p.rows, p.dy_stride, p.h_stride, p.dh_stride, p.dx_stride, (int32_t)p.cols, p.eps};
  DC_RETURN_IF(p.dtype == DC_DTYPE_F32 ? norm_grad_by_shape<float>(ctx, a, grid, c, waves) : norm_grad_by_shape<bf16>(ctx, a, grid, c, waves));
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
  }
  if (!aligned_to(scales, 4)) return DC_ERR_MISALIGNED;
  DC_CTX_ENTER(ctx);
  if (rows == 0 || cols == 0) return empty_scales(ctx, scales, rows);
  const NormArgs a{x, nullptr, nullptr, nullptr, q, scales, rows, x_stride, 0, 0, q_stride, (int32_t)cols, 0.0f};
  return dtype == DC_DTYPE_F32 ? norm_by_shape<float, uint8_t, false>(ctx, a) : norm_by_shape<bf16, uint8_t, false>(ctx, a);
}

}  // extern "C"
