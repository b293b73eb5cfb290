// dc_norm_row.hpp — what the norms share: a row in registers over the waves that hold it, their sums, the column sums of the
// weights' gradients, and the checks of rows.
#pragma once

#include "dc_internal.hpp"
#include "dc_numeric.hpp"

namespace dc {

// Waves that share a row, at most: each leaves its sum in a word of LDS, and every wave adds the words in order, those of
// waves that are not there too (zeros from the start of the kernel): few wide reads and no loop.
constexpr int kWaves = 16;

__device__ inline float add_words(const float* scratch, int waves) {
  const f32x4* q = reinterpret_cast<const f32x4*>(scratch);
  const f32x4 a = q[0], b = q[1];
  float v = ((a.x + a.y) + (a.z + a.w)) + ((b.x + b.y) + (b.z + b.w));
  if (waves > 8) {
    const f32x4 c = q[2], d = q[3];
    v += ((c.x + c.y) + (c.z + c.w)) + ((d.x + d.y) + (d.z + d.w));
  }
  return v;
}

// Sum (or unsigned maximum) over the `waves` waves that share a row, in every lane. `scratch`: nobody writes it again
// before the caller's next barrier.
__device__ inline float row_sum(float v, float* scratch, int wave, int waves) {
  v = wave_sum_f32(v);
  if (waves > 1) {
    if ((threadIdx.x & 63) == 0) scratch[wave] = v;
    __syncthreads();
    v = add_words(scratch, waves);
  }
  return v;
}
__device__ inline uint32_t row_max(uint32_t v, float* scratch, int wave, int waves) {
  v = wave_max_u32(v);
  if (waves > 1) {
    uint32_t* s = reinterpret_cast<uint32_t*>(scratch);
    if ((threadIdx.x & 63) == 0) s[wave] = v;
    __syncthreads();
    const u32x4* q = reinterpret_cast<const u32x4*>(scratch);
    const u32x4 a = q[0], b = q[1], c = q[2], d = q[3];
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
  __device__ inline void load(const T* p, u32x4 (&raw)[C]) const {
    if (cols >= E) {
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const int64_t c = at(i);
        raw[i] = load_raw(p + (c < cols - E ? c : cols - E));
      }
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i) {
        float v[E];
        load_some(p, i == 0 && wave == 0 && lane == 0 ? cols : 0, v);
        raw[i] = u32x4{0, 0, 0, 0};
        if constexpr (E == 4) raw[i] = __builtin_bit_cast(u32x4, f32x4{v[0], v[1], v[2], v[3]});
        else
#pragma unroll
          for (int e = 0; e < 4; ++e) raw[i][e] = pack_bf16(v[2 * e], v[2 * e + 1]);
      }
    }
  }
  // What load() left of the row's last 16 bytes in the chunks at and past its end.
  __device__ inline void cut(u32x4 (&raw)[C]) const {
    if (cols < E) return;
#pragma unroll
    for (int i = 0; i < C; ++i)
      if ((int64_t)((i * waves + wave) * 64 + 64) * E > cols) {  // (uniform)
        const int64_t past = at(i) - (cols - E);
        if (past > 0) raw[i] = shift_down(raw[i], past * (int64_t)sizeof(T));
      }
  }
};

constexpr int64_t kMaxCols = int64_t(1) << 25;
constexpr int64_t kMaxGrid = 1 << 20;  // rows beyond are walked over by the same workgroups

// Waves that hold a row of `chunks` 16-byte chunks, C to a lane.
inline int waves_for(int64_t chunks, int c) { return (int)((chunks + 64 * c - 1) / (64 * c)); }

inline bool float_dtype(int32_t t) { return t == DC_DTYPE_F32 || t == DC_DTYPE_BF16; }
inline int64_t size_of(int32_t t) { return t == DC_DTYPE_F32 ? 4 : t == DC_DTYPE_BF16 ? 2 : 1; }
inline bool aligned_to(const void* p, int64_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }

// Rows of nothing: their maxima, and so their scales, are zeros.
inline int32_t empty_scales(dc_hip_ctx* ctx, float* scales, int64_t rows) {
  return scales && rows > 0 ? zero_async(ctx, scales, (size_t)rows * sizeof(float)) : DC_OK;
}

// One row, or several with a stride of at least a row's length.
inline int32_t check_rows(const void* p, int32_t dtype, int64_t stride, int64_t rows, int64_t cols) {
  if (!aligned_to(p, size_of(dtype))) return DC_ERR_MISALIGNED;
  return rows > 1 && stride < cols ? DC_ERR_DIMENSION : DC_OK;
}

inline int32_t check_shape(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 0) return DC_ERR_INVALID_ARGUMENT;
  return cols > kMaxCols ? DC_ERR_UNSUPPORTED : DC_OK;
}

}  // namespace dc
