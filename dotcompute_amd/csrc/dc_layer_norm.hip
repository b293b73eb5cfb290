// dc_layer_norm.hip — layer norm with the residual's addition, its gradients, and rows in 8 bits with a scale for each 128 elements.
//
// Forward, a row at a time: h = x + r, y = (h - mean) s w + b with s = 1 / sqrt(var + eps). Memory-bound: 8 bytes an element in bf16 (x, r
// in; h, y out), 7 with y in 8 bits. A row stays in registers between its one read and its write, as an RMS norm's. 16384×4096 93.3 us (5.8 TB/s),
// 8191×2050, whose rows lie at 4-byte boundaries, 25.9 (5.2); 8×4096 to 8 bits 4.2, of which the call is 3.7. To 8 bits with block scales 16384×4096 79 (5.9), but
// without a residual 67 (3.0), with a scale a row 77: bound by a row's way through its statistics and maxima there.
// Most of the forms for 8 bits, and of those with more than one chunk a lane, spill scalar registers, up to 92, beside the vector ones that are named at norm_by_shape.
//
// Backward: u = (h - mean) s, g = dy w: dx = s (g - mean(g) - u mean(g u)) + dh, dw = the sum over rows of dy u, db of dy. One read of each
// operand; the statistics are formed again from h, which is read anyway. A workgroup walks over rows and keeps its parts of dw
// and db in registers, or of long rows in LDS; a second kernel adds the parts in a fixed order (no atomics: the same bits from call to call).
// Memory-bound: 8192×4096 50 us with that kernel (5.4 TB/s), 8191×2050 36.8 (3.7: five waves a row, the last with one lane's worth, so that a CU's 15
// do the work of twelve, at 4-byte boundaries); 500×1024 in float32 7.8, two launches.
//
// Statistics. The difference of mean(h^2) and mean(h)^2 loses the variance's digits where the mean is large, and a second sum over a row that
// several waves share would be a second barrier. So each wave takes a value k near its own part's mean, the mean of its lanes' first chunks, and the sums
// of d = h - k and d^2, in registers; the waves' triples meet in LDS once, and every wave joins them: M is
// the rounded mean, e what is left, and sum((h - M)^2) = the sum over waves of sum(d^2) + 2 c sum(d) + n c^2, c = k - M. An
// element's u is d s + ((k - M) - e) s, whose terms are of u's size. However a row's values lie, a lane with C chunks has the sum of n c^2 at C times the row's
// squares at most (one chunk of C is the sample): with one chunk nothing cancels, with four the sum of d^2 is at most (1 + sqrt 4)^2 = 9 times what is left
// of it, three bits. (The mean of the first 32 elements, 16 of float32, as k, which is four additions less a row, lost up to six where those lie apart from the
// rest. us, that / this: bf16 8191×2050 25.7 / 25.9, its gradients 36.2 / 36.7, 16384×512 11.8 / 11.9, 16384×4096 93.3 both.)
#include <algorithm>
#include <type_traits>

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

__device__ inline void store_chunk_once(float* p, const float (&v)[4]) {
  __builtin_nontemporal_store(f32x4_at4{v[0], v[1], v[2], v[3]}, reinterpret_cast<f32x4_at4*>(p));
}
__device__ inline void store_chunk_once(bf16* p, const float (&v)[8]) {
  u32x4_at2 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
  __builtin_nontemporal_store(w, reinterpret_cast<u32x4_at2*>(p));
}

// The chunks c_i = ((i waves + wave) 64 + lane) E, i < C, of a row, as dc::Row has them; offsets in 32 bits (a row has at most 2^27 bytes), beside a
// pointer that all lanes share, which saves registers and additions for each of a row's operands. The first kInside chunks are in the row for every wave: where
// half of them would hold a row there are fewer waves. (The gradients use that: float32 2000×12000 94 us, else 110. Forward it moves the loads' order:
// float32 8192×2048 51.7, else 48.5.)
template <typename T, int C, int kInside = 0>
struct Span {
  static constexpr int E = kElems<T>;
  uint32_t cols, first, step, end;  // first: of the lane; step: from chunk to chunk; end: of the wave's first chunks (uniform)
  __device__ inline Span(int64_t cols_, int waves, int wave, int lane)
      : cols((uint32_t)cols_), first((uint32_t)((wave * 64 + lane) * E)), step((uint32_t)(waves * 64 * E)),
        end((uint32_t)((wave + 1) * 64 * E)) {}
  __device__ inline uint32_t at(int i) const { return first + i * step; }
  template <typename P>
  static __device__ inline P* past(P* p, uint32_t elements) {
    typedef std::conditional_t<std::is_const_v<P>, const char, char> Byte;
    return reinterpret_cast<P*>(reinterpret_cast<Byte*>(p) + elements * (uint32_t)sizeof(P));
  }
  template <bool kOnce = false>
  __device__ inline void load(const T* p, u32x4 (&raw)[C]) const {
    if (kInside > 0 || cols >= E) {
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const uint32_t c = at(i);
        const T* from = past(p, inside(i) || c < cols - E ? c : cols - E);
        raw[i] = kOnce ? load_raw_once(from) : load_raw(from);
      }
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i) {
        float v[E];
        load_some(p, i == 0 && first == 0 ? (int64_t)cols : 0, v);
        raw[i] = u32x4{0, 0, 0, 0};
        if constexpr (E == 4) raw[i] = __builtin_bit_cast(u32x4, f32x4{v[0], v[1], v[2], v[3]});
        else
#pragma unroll
          for (int e = 0; e < 4; ++e) raw[i][e] = pack_bf16(v[2 * e], v[2 * e + 1]);
      }
    }
  }
  // Whether all elements of the wave's chunk i are in the row (uniform).
  static __device__ constexpr bool inside(int i) { return i < kInside; }
  __device__ inline bool whole(int i) const { return inside(i) || end + i * step <= cols; }
  // What load() left of the row's last 16 bytes in the chunks at and past its end.
  __device__ inline void cut(u32x4 (&raw)[C]) const {
    if (kInside == 0 && cols < E) return;
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (!whole(i)) {
        const int over = (int)(at(i) - (cols - E));
        if (over > 0) raw[i] = shift_down(raw[i], (int64_t)over * (int)sizeof(T));
      }
  }
  template <typename Y>
  __device__ inline void store(Y* p, int i, const float (&v)[E]) const {
    const uint32_t c = at(i);
    if (inside(i)) store_chunk(past(p, c), v);
    else if (c < cols) store_some(past(p, c), (int64_t)cols - c, v);
  }
  // What no cache need keep.
  __device__ inline void store_once(T* p, int i, const float (&v)[E]) const {
    const uint32_t c = at(i);
    if (c + E <= cols) store_chunk_once(past(p, c), v);
    else if (c < cols) store_some(past(p, c), (int64_t)cols - c, v);
  }
};

// Elements of a row that a wave holds.
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

// A value near the mean of a wave's elements, and the sums of what is left over it and of that squared (elements past the row's end are zeros in h).
struct Moments {
  float near, left, squares;
};
// 1 / the number of elements that `near` is the mean of: those of the wave's first chunks.
template <int E>
__device__ inline float near_weight(int64_t cols, int wave) {
  const int64_t left = cols - (int64_t)wave * 64 * E;
  return 1.0f / (float)(left < 64 * E ? left : 64 * E);
}
template <typename T, int C>
__device__ inline float value_near(const float (&h)[C][kElems<T>], float weight) {
  constexpr int E = kElems<T>;
  float v = 0.0f;
#pragma unroll
  for (int e = 0; e < E; e += 4) v += (h[0][e] + h[0][e + 1]) + (h[0][e + 2] + h[0][e + 3]);
  return wave_sum_f32(v * weight);  // (weighted before the lanes meet: the sum of a wave's largest floats is none)
}
// h becomes d = h - near (zeros past the row's end); the lane's part of the sums.
template <typename T, int C, int kInside>
__device__ inline Moments lane_moments(const Span<T, C, kInside>& R, float (&h)[C][kElems<T>], float near) {
  constexpr int E = kElems<T>;
  Moments m{near, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const bool whole = R.whole(i);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      h[i][e] -= near;
      if (!whole) h[i][e] = R.at(i) + e < R.cols ? h[i][e] : 0.0f;
      m.left += h[i][e];
      m.squares = __builtin_fmaf(h[i][e], h[i][e], m.squares);
    }
  }
  return m;
}

// The variance, from sums of what is left over a value near the mean (no less than zero where rounding would have it so: a row of equal values).
__device__ inline float variance(float squares, float left, float rest, float per) {
  const float v = (squares - left * rest) * per;
  return v < 0.0f ? 0.0f : v;
}

// 1 / sqrt(v), an ulp off; v among the smallest floats keeps its digits.
__device__ inline float inverse_root(float v) {
  const bool small = v < 0x1p-96f;
  const float r = __builtin_amdgcn_rsqf(small ? v * 0x1p96f : v);
  return small ? r * 0x1p48f : r;
}

// Of a row: s = 1 / sqrt(var + eps), and what u is past d s in this lane's wave.
struct RowStats {
  float shift, s;
};
// What the waves left, a wave's in each of 16 lanes (`n`: of how many elements, 0 where there is no wave), joined: what `near` (this lane's wave's) is
// away from the row's mean by, in two parts.
struct Joined {
  float off, rest;
  RowStats row;
};
__device__ inline Joined join_moments(const Moments& m, float n, float near, float per, float eps) {
  Joined j;
  const float mean = row16_sum_f32(__builtin_fmaf(n, m.near, m.left)) * per;
  j.off = m.near - mean;
  const float rest = row16_sum_f32(__builtin_fmaf(n, j.off, m.left));
  const float squares = row16_sum_f32(__builtin_fmaf(j.off, __builtin_fmaf(n, j.off, 2.0f * m.left), m.squares));
  j.rest = rest * per;
  j.row.s = inverse_root(variance(squares, rest, j.rest, per) + eps);
  j.row.shift = ((near - mean) - j.rest) * j.row.s;
  return j;
}
// Of a row that one wave holds.
__device__ inline RowStats own_stats(const Moments& m, float per, float eps) {
  const float rest = m.left * per, s = inverse_root(variance(m.squares, m.left, rest, per) + eps);
  return RowStats{-rest * s, s};
}

typedef float f32x4_lds __attribute__((ext_vector_type(4)));

// A workgroup walks over rows, one at a time, or, where a wave holds a row, four; the weights stay in registers, and the next row's operands are asked
// for before this one's sums. (`sum` and y may lie over x or the residual: each lane writes what it alone has read, and a load that reaches back over the
// row's end drops what is not its own.) 8 bits: a scale a row, or (kBlocks) one for each 128.
template <typename T, typename Y, int C, bool kBlocks, bool kOnce>
__global__ __launch_bounds__(1024) void layer_norm_kernel(LayerNormArgs a, int waves) {
  constexpr int E = kElems<T>;
  constexpr bool kFp8 = sizeof(Y) == 1;
  __shared__ __align__(16) f32x4_lds words[kWaves];
  __shared__ __align__(16) float scratch[1][kWaves];
  const int lane = threadIdx.x & 63, group = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = waves == 1 ? 0 : group;
  const int64_t cols = a.cols;
  const Span<T, C> R(cols, waves, wave, lane);
  const int other = lane & (kWaves - 1);  // whose moments this lane joins
  const float weight = near_weight<E>(cols, wave), n_other = other < waves ? wave_count<E, C>(cols, waves, other) : 0.0f;
  const float per_col = 1.0f / (float)a.cols;
  clear_words(scratch, 1, waves);
  const int per = waves == 1 ? 4 : 1;
  const int64_t step = (int64_t)gridDim.x * per;
  u32x4 xr[C], rr[C], wr[C], br[C];
  auto load = [&](int64_t row) __attribute__((always_inline)) {
    R.template load<kOnce>(static_cast<const T*>(a.x) + row * a.x_stride, xr);
    if (a.residual) R.template load<kOnce>(static_cast<const T*>(a.residual) + row * a.residual_stride, rr);
  };
  const int64_t first = (int64_t)blockIdx.x * per + (waves == 1 ? group : 0);
  if (first < a.rows) load(first);
  R.load(static_cast<const T*>(a.weight), wr);
  if (a.bias) R.load(static_cast<const T*>(a.bias), br);
  R.cut(wr);
  if (a.bias) R.cut(br);
  for (int64_t row = first; row < a.rows; row += step) {
    T* sum = a.sum ? static_cast<T*>(a.sum) + row * a.sum_stride : nullptr;
    Y* y = static_cast<Y*>(a.y) + row * a.y_stride;
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
    if (row + step < a.rows) load(row + step);
    // (the sum is read again only after the block's products; y, which they read, is kept. us for both kept / this / neither: 16384×4096 95.9 / 93.2 / 89.9,
    // 8191×2050 25.5 / 25.6 / 27.0, 2000×12000 34.7 / 34.7 / 35.8, float32 8192×2048 47.4 / 43.4 / 45.5)
    if (sum)
#pragma unroll
      for (int i = 0; i < C; ++i) kOnce ? R.store_once(sum, i, h[i]) : R.store(sum, i, h[i]);
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
      r = join_moments(q, n_other, m.near, per_col, a.eps).row;
    }
#pragma unroll
    for (int i = 0; i < C; ++i) {
      float w[E], b[E];
      unpack(wr[i], w);
      if (a.bias) unpack(br[i], b);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        h[i][e] = __builtin_fmaf(h[i][e], r.s, r.shift);
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
          if (R.at(i) + e < R.cols) top[i] = max(top[i], magnitude(h[i][e]));
      }
      if constexpr (kBlocks) {
#pragma unroll
        for (int i = 0; i < C; ++i) {
          const uint32_t scale = block_scale(block_max_u32<E>(top[i]));
          const float factor = block_factor(scale);
          const uint32_t c = R.at(i);
          if (c % kScaleBlock == 0 && c < R.cols) static_cast<uint8_t*>(a.scales)[c / kScaleBlock * a.scales_stride + row] = (uint8_t)scale;
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
    for (int i = 0; i < C; ++i) R.store(y, i, h[i]);
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
    const float rest = left / (float)a.cols, s = 1.0f / sqrtf(variance(squares, left, rest, 1.0f / (float)a.cols) + a.eps);
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

// `groups` rows at a time to a workgroup, `waves` waves to each, at most 16 in all; their parts of dweight and dbias meet in LDS at the end, so that a
// workgroup leaves one of each. With kAhead the next rows' operands are asked for before these ones' sums. With kShared (one row at a time) the parts
// lie in LDS all along, up to 128 KiB, each lane's where it alone reads them: beside the rest of rows that long registers do not hold them.
template <typename T, int C, bool kAhead, bool kShared, bool kOnce>
__global__ __launch_bounds__(1024) void layer_norm_grad_kernel(LayerNormGradArgs a, int waves, int groups) {
  constexpr int E = kElems<T>, kQuads = C * (E / 4);  // of dweight's parts to a lane
  constexpr bool kKeep = C == 1;  // g over the barrier (of two chunks a lane it does not fit beside the rest, and is formed again)
  __shared__ __align__(16) float words[2][kWaves][8];  // (of a wave: sums of d, d^2, g, g d, and the value that d is of)
  __shared__ __align__(16) f32x4_lds kept[kShared ? 2 * kQuads * 64 * kWaves : 1];
  extern __shared__ __align__(16) float left_by[];  // (groups - 1) waves 64 2 C E floats
  const int lane = threadIdx.x & 63, place = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = place / waves, wave = place - group * waves, first = group * waves;
  const int64_t cols = a.cols;
  const Span<T, C, C / 2> R(cols, waves, wave, lane);
  const int other = lane & (kWaves - 1);
  const float weight = near_weight<E>(cols, wave), n_other = other < waves ? wave_count<E, C>(cols, waves, other) : 0.0f;
  const float per_col = 1.0f / (float)a.cols;
  float dw[C][E], db[C][E];
#pragma unroll
  for (int i = 0; i < C; ++i)
#pragma unroll
    for (int e = 0; e < E; ++e) dw[i][e] = db[i][e] = 0.0f;
  if constexpr (kShared)
#pragma unroll
    for (int q = 0; q < 2 * kQuads; ++q) kept[q * 64 * kWaves + threadIdx.x] = f32x4_lds{0.0f, 0.0f, 0.0f, 0.0f};
  u32x4 wr[C], hr[C], dr[C], ur[C];
  auto load = [&](int64_t row) __attribute__((always_inline)) {
    R.template load<kOnce>(static_cast<const T*>(a.h) + row * a.h_stride, hr);
    R.template load<kOnce>(static_cast<const T*>(a.dy) + row * a.dy_stride, dr);
    if (a.dh && a.dx) R.template load<kOnce>(static_cast<const T*>(a.dh) + row * a.dh_stride, ur);
  };
  R.load(static_cast<const T*>(a.weight), wr);
  const int64_t step = (int64_t)gridDim.x * groups;
  // (a group without a row goes along to the barrier with what it last read, and adds nothing)
  auto last = [&](int64_t row) __attribute__((always_inline)) { return row < a.rows ? row : a.rows - 1; };
  if constexpr (kAhead) load(last((int64_t)blockIdx.x * groups + group));
  R.cut(wr);
  int flip = 0;
  for (int64_t base = (int64_t)blockIdx.x * groups; base < a.rows; base += step) {
    const int64_t row = base + group;
    if constexpr (!kAhead) load(last(row));
    R.cut(hr);
    R.cut(dr);
    float d[C][E], g[kKeep ? C : 1][E];
    u32x4 yv[C], uv[C];
#pragma unroll
    for (int i = 0; i < C; ++i) {
      unpack(hr[i], d[i]);
      yv[i] = dr[i];
      uv[i] = ur[i];
    }
    if constexpr (kAhead)
      if (row + step < a.rows) load(row + step);
    Moments m = lane_moments(R, d, value_near<T, C>(d, weight));
    float g_sum = 0.0f, gd_sum = 0.0f;  // of g and of g d
#pragma unroll
    for (int i = 0; i < C; ++i) {
      float w[E], dy[E];
      float(&gi)[E] = g[kKeep ? i : 0];
      unpack(wr[i], w);
      unpack(yv[i], dy);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        gi[e] = dy[e] * w[e];
        g_sum += gi[e];
        gd_sum = __builtin_fmaf(gi[e], d[i][e], gd_sum);
      }
    }
    const float sums_of_lanes = wave_sums_of_four(m.left, m.squares, g_sum, gd_sum, lane);
    RowStats r;
    if (waves == 1) {
      m.left = lane_value(sums_of_lanes, 0);
      r = own_stats(Moments{m.near, m.left, lane_value(sums_of_lanes, 1)}, per_col, a.eps);
      g_sum = lane_value(sums_of_lanes, 2);
      gd_sum = lane_value(sums_of_lanes, 3) - m.left * per_col * g_sum;
    } else {
      if (lane < 5) words[flip][place][lane] = lane < 4 ? sums_of_lanes : m.near;
      __syncthreads();  // (two sets in turn: a wave writes a set again only past the barrier of the row between)
      f32x4_lds v = {0.0f, 0.0f, 0.0f, 0.0f};
      float near = 0.0f;
      if (other < waves) {
        v = *reinterpret_cast<const f32x4_lds*>(words[flip][first + other]);
        near = words[flip][first + other][4];
      }
      flip ^= 1;
      const Joined j = join_moments(Moments{near, v.x, v.y}, n_other, m.near, per_col, a.eps);
      r = j.row;
      g_sum = row16_sum_f32(v.z);
      gd_sum = row16_sum_f32(__builtin_fmaf(j.off, v.z, v.w)) - j.rest * g_sum;
    }
    if (row >= a.rows) continue;
    // dx = s g - u s mean(g u) - s mean(g) + dh (s^2 alone may be no float where eps is 0)
    const float along = -r.s * (r.s * (gd_sum * per_col)), flat = -r.s * (g_sum * per_col);
    T* dx = a.dx ? static_cast<T*>(a.dx) + row * a.dx_stride : nullptr;
    if (dx && a.dh) R.cut(uv);
#pragma unroll
    for (int i = 0; i < C; ++i) {
      float o[E], dy[E], w[E];
      unpack(yv[i], dy);
      if constexpr (!kKeep) unpack(wr[i], w);
      f32x4_lds sums[2];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float u = __builtin_fmaf(d[i][e], r.s, r.shift);
        if constexpr (kShared) {
          f32x4_lds* at = kept + (i * (E / 4) + e / 4) * 64 * kWaves + threadIdx.x;
          if (e % 4 == 0) sums[0] = at[0], sums[1] = at[kQuads * 64 * kWaves];
          sums[0][e % 4] = __builtin_fmaf(dy[e], u, sums[0][e % 4]);
          sums[1][e % 4] += dy[e];
          if (e % 4 == 3) at[0] = sums[0], at[kQuads * 64 * kWaves] = sums[1];
        } else {
          dw[i][e] = __builtin_fmaf(dy[e], u, dw[i][e]);
          db[i][e] += dy[e];
        }
        o[e] = __builtin_fmaf(kKeep ? g[kKeep ? i : 0][e] : dy[e] * w[e], r.s, __builtin_fmaf(u, along, flat));
      }
      if (dx) {
        if (a.dh) {
          float q[E];
          unpack(uv[i], q);
#pragma unroll
          for (int e = 0; e < E; ++e) o[e] += q[e];
        }
        R.store(dx, i, o);
      }
    }
  }
  if (groups > 1) {
    const int lanes = waves * 64, at = wave * 64 + lane;
    f32x4_lds* own = reinterpret_cast<f32x4_lds*>(left_by);
    auto slot = [&](int g, int q) { return ((g - 1) * 2 * C * (E / 4) + q) * lanes + at; };
    auto quad = [&](int q) -> f32x4_lds* {
      const int half = C * (E / 4), i = q % half;
      return reinterpret_cast<f32x4_lds*>(q < half ? &dw[i / (E / 4)][4 * (i % (E / 4))] : &db[i / (E / 4)][4 * (i % (E / 4))]);
    };
    if (group > 0)
#pragma unroll
      for (int q = 0; q < 2 * C * (E / 4); ++q) own[slot(group, q)] = *quad(q);
    __syncthreads();
    if (group > 0) return;
    for (int g = 1; g < groups; ++g)
#pragma unroll
      for (int q = 0; q < 2 * C * (E / 4); ++q) *quad(q) += own[slot(g, q)];
  }
  if constexpr (kShared)
#pragma unroll
    for (int q = 0; q < kQuads; ++q) {
      *reinterpret_cast<f32x4_lds*>(&dw[q / (E / 4)][4 * (q % (E / 4))]) = kept[q * 64 * kWaves + threadIdx.x];
      *reinterpret_cast<f32x4_lds*>(&db[q / (E / 4)][4 * (q % (E / 4))]) = kept[(kQuads + q) * 64 * kWaves + threadIdx.x];
    }
  auto leave = [&](float* parts, const float (&v)[C][E]) __attribute__((always_inline)) {
    float* part = parts + (int64_t)blockIdx.x * a.part_pitch;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const uint32_t c = R.at(i);
#pragma unroll
      for (int e = 0; e < E; e += 4)
        if (c + e < R.cols) store_some(R.past(part, c + e), (int64_t)R.cols - c - e, *reinterpret_cast<const float (*)[4]>(v[i] + e));
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
    const float n = (float)a.cols, rest = left / n, s = 1.0f / sqrtf(variance(squares, left, rest, 1.0f / n) + a.eps);
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
// Memory-bound: 3 bytes an element of bf16, 5 of float32. A wave takes 64 chunks of 16 bytes (512 elements of bf16, 256 of float32) of kRows rows below each
// other, all asked for at once; a block's maximum is found among 16 or 32 lanes, without LDS, and its first lane writes the rows' scales, which
// lie beside each other, in one piece. bf16 8192×8192 34.7 us (5.8 TB/s), 8191×8190, whose rows end inside lines, 40.4; with eight rows to a wave 34.1 and 41.7.
struct QuantizeArgs {
  const void* x;
  uint8_t *q, *scales;
  int64_t rows, cols, x_stride, q_stride, scales_stride, across, total;  // across: pieces to a row; total: pieces
};
template <typename T, int kRows, bool kOnce>
__global__ __launch_bounds__(256) void quantize_blocks_kernel(QuantizeArgs a) {
  constexpr int E = kElems<T>;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (int64_t t = (int64_t)blockIdx.x * 4 + wave; t < a.total; t += (int64_t)gridDim.x * 4) {
    const int64_t down = a.total <= UINT32_MAX ? (int64_t)((uint32_t)t / (uint32_t)a.across) : t / a.across;
    const int64_t row0 = down * kRows, c0 = (t - down * a.across) * 64 * E, left = a.cols - c0;  // left: elements from here on
    const int at = lane * E, rows = (int)(a.rows - row0 < kRows ? a.rows - row0 : kRows);
    const T* x = static_cast<const T*>(a.x) + row0 * a.x_stride + c0;
    u32x4 raw[kRows];
    if (a.cols >= E) {  // (a chunk at the row's end is cut out of its last 16 bytes, one past it is zeros; no branch between the loads)
      const int64_t from = at < left - E ? at : left - E;
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const T* p = x + (i < rows ? i : rows - 1) * a.x_stride + from;
        raw[i] = kOnce ? load_raw_once(p) : load_raw(p);
      }
      if (left < 64 * E)
#pragma unroll
        for (int i = 0; i < kRows; ++i) raw[i] = shift_down(raw[i], (at - from) * (int64_t)sizeof(T));
    } else {
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        float v[E];
        load_some(x + (i < rows ? i : rows - 1) * a.x_stride, at == 0 ? left : 0, v);
        if constexpr (E == 4) raw[i] = __builtin_bit_cast(u32x4, f32x4{v[0], v[1], v[2], v[3]});
        else
#pragma unroll
          for (int e = 0; e < 4; ++e) raw[i][e] = pack_bf16(v[2 * e], v[2 * e + 1]);
      }
    }
    uint32_t scales = 0;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      float v[E];
      unpack(raw[i], v);
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) top = max(top, magnitude(v[e]));
      const uint32_t scale = block_scale(block_max_u32<E>(top));
      const float factor = block_factor(scale);
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] *= factor;
      scales |= scale << (8 * i);
      if (i < rows && at < left) store_some(a.q + (row0 + i) * a.q_stride + c0 + at, left - at, v);
    }
    if (at % kScaleBlock == 0 && at < left) {
      uint8_t* to = a.scales + (c0 + at) / kScaleBlock * a.scales_stride + row0;
      if (kRows == 4 && rows == 4) {
        *reinterpret_cast<u32_at1*>(to) = scales;
      } else {
#pragma unroll
        for (int i = 0; i < kRows; ++i)
          if (i < rows) to[i] = (uint8_t)(scales >> (8 * i));
      }
    }
  }
}

// ---- host --------------------------------------------------------------------------------------------------
template <typename T, typename Y, int C, bool kBlocks>
int32_t launch_norm(dc_hip_ctx* ctx, const LayerNormArgs& a, int64_t chunks) {
  const int waves = waves_for(chunks, C), group = waves == 1 ? 4 : waves;  // (16 waves to a CU)
  const int64_t groups = waves == 1 ? (a.rows + 3) / 4 : a.rows, held = (int64_t)std::max(1, ctx->cu_count) * std::max(1, kWaves / group);
  const int64_t size = sizeof(T), bytes = size * (1 + (a.residual != nullptr) + (a.sum != nullptr)) + (int64_t)sizeof(Y);
  auto* kernel = read_once(a.rows, a.cols, bytes) ? layer_norm_kernel<T, Y, C, kBlocks, true> : layer_norm_kernel<T, Y, C, kBlocks, false>;
  kernel<<<(unsigned)std::min(groups, held), 64 * group, 0, ctx->stream>>>(a, waves);
  return last_launch_status();
}

// Chunks that a lane holds: one of bf16, over up to 16 waves; two where they let a wave hold a row by itself (but not where it is read and written in float32),
// and in longer rows. us, with the call, for a workgroup to each row with one to two chunks / workgroups that walk with two / with one, bf16: 16384×4096 95.6 /
// 103 / 96.0, to 8 bits 98.7 / 93.1 / 94.0; 8191×2050 34.8 / 29.8 / 28.0; 4096×8192 55.7 / 48.5 / 48.6; 2000×12000 53 / 38;
// 1000×4096 8.6 / 8.5 / 7.6; float32 8192×2048 48.3 / 48.5 / 50.3 (all before large operands were loaded as read once). With 24 waves a CU 16384×4096
// takes 101, with 32 108. Four chunks for float32 rows of more than 16 waves of two, which spill 9 to 23 registers,
// or such rows read again by the long kernel: 2322×15219 119 / 155, 2000×9000 57 / 80, to 8 bits 2000×12000 78 / 117, 20×12000 7.3 / 7.7; of bf16, whose
// rows' values take twice the registers, 2048×24576 222 / 124.
template <typename T, typename Y, bool kBlocks>
int32_t norm_by_shape(dc_hip_ctx* ctx, const LayerNormArgs& a) {
  const int64_t chunks = (a.cols + kElems<T> - 1) / kElems<T>;
  const bool wave = chunks > 64 && chunks <= 128 && (sizeof(T) == 2 || sizeof(Y) == 1), one = sizeof(T) == 2 || a.rows <= ctx->cu_count;
  if (!wave && chunks <= (one ? 64 * kWaves : 256)) return launch_norm<T, Y, 1, kBlocks>(ctx, a, chunks);
  if (chunks <= 64 * 2 * kWaves) return launch_norm<T, Y, 2, kBlocks>(ctx, a, chunks);
  if constexpr (sizeof(T) == 4)
    if (chunks <= 64 * 4 * kWaves) return launch_norm<T, Y, 4, kBlocks>(ctx, a, chunks);
  layer_norm_long_kernel<T, Y, kBlocks><<<(unsigned)std::min(a.rows, kMaxGrid), 64 * kWaves, 0, ctx->stream>>>(a);
  return last_launch_status();
}

template <typename T>
int32_t norm_by_output(dc_hip_ctx* ctx, const LayerNormArgs& a, bool fp8, bool blocks) {
  if (!fp8) return norm_by_shape<T, T, false>(ctx, a);
  return blocks ? norm_by_shape<T, uint8_t, true>(ctx, a) : norm_by_shape<T, uint8_t, false>(ctx, a);
}

// The gradient's workgroups, and the rows that each takes at a time.
struct GradGrid {
  int64_t workgroups;
  int groups;
};
// A workgroup a CU, of 16 waves where rows are short, as each leaves parts of dweight and dbias to be added; but no more rows at a time than leave every CU
// some. us, with the call, bf16, for workgroups of one row (as many as a CU holds) / of 8 waves / of 16: 16384×512 21.1 / 17.7 / 16.7, 8192×1024
// 22.0 / 18.5 / 18.5, 8191×2050 38.7 / 61 / 37.5; 1000×1000, in workgroups of one row, 4 and 8 rows 14.9 / 9.2 / 10.3. Float32 rows of 6 to 8 waves:
// two workgroups of one row, 8192×2048 55.2, one of two rows 59.5, one of one 74; bf16 8192×4096 59.5, 55.4, 53.8, 8192×3500 one of two rows 53.3, of one 77.
GradGrid norm_grad_grid(bool f32, int64_t rows, int c, int waves, int64_t cus) {
  const int64_t share = (rows + cus - 1) / cus;
  const int groups = c == 1 && !(f32 && waves >= 6) ? (int)std::min<int64_t>(std::max(1, kWaves / waves), share) : 1;
  const int64_t held = cus * (f32 && c == 1 && waves >= 6 && waves <= 8 ? 2 : 1);
  // (Few rows: no more workgroups than take as many of them each)
  const int64_t each = (rows + held * groups - 1) / (held * groups);
  return {each <= 4 ? (rows + each * groups - 1) / (each * groups) : held, groups};
}

template <typename T>
int32_t norm_grad_by_shape(dc_hip_ctx* ctx, const LayerNormGradArgs& a, const GradGrid& grid, int c, int waves) {
  constexpr bool kShort = sizeof(T) == 2;
  const int groups = grid.groups;
  const unsigned g = (unsigned)grid.workgroups, threads = 64 * waves * groups;
  const size_t lds = (size_t)(groups - 1) * waves * 64 * 2 * c * kElems<T> * sizeof(float);
  auto launch = [&](auto* often, auto* once) {
    const int64_t bytes = (int64_t)sizeof(T) * (2 + (a.dx ? 1 + (a.dh != nullptr) : 0));
    (read_once(a.rows, a.cols, bytes) ? once : often)<<<g, threads, lds, ctx->stream>>>(a, waves, groups);
  };
  if (c == 1) launch(layer_norm_grad_kernel<T, 1, true, false, false>, layer_norm_grad_kernel<T, 1, true, false, true>);
  else if (c == 2) launch(layer_norm_grad_kernel<T, 2, kShort, kShort, false>, layer_norm_grad_kernel<T, 2, kShort, kShort, true>);
  else if (sizeof(T) == 4 && c == 4) launch(layer_norm_grad_kernel<float, 4, false, true, false>, layer_norm_grad_kernel<float, 4, false, true, true>);
  else layer_norm_grad_long_kernel<T><<<g, 64 * kWaves, 0, ctx->stream>>>(a);
  return last_launch_status();
}

// 16-byte chunks of a row that a lane of the gradient's kernel holds (0: the long kernel). us, with the call, for rows of more than 1024 chunks in bf16, 2048
// in float32, with their parts of dweight and dbias in registers (bf16: 8 waves of four chunks) / in LDS / by the long kernel: bf16 2000×12000
// 74.4 / 58.5 / 236, 4096×16384 147 / 125 / 582; float32 2000×12000 145 / 94 / 209.
int norm_grad_chunks(bool f32, int64_t chunks) {
  if (f32) return chunks <= 64 * kWaves ? 1 : chunks <= 128 * kWaves ? 2 : chunks <= 256 * kWaves ? 4 : 0;
  return chunks <= 64 * kWaves ? 1 : chunks <= 128 * kWaves ? 2 : 0;
}

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
  const int c = norm_grad_chunks(p.dtype == DC_DTYPE_F32, chunks), waves = c ? waves_for(chunks, c) : kWaves;
  const GradGrid grid = norm_grad_grid(p.dtype == DC_DTYPE_F32, p.rows, c, waves, std::max(1, ctx->cu_count));
  const int outs = (p.dweight ? 1 : 0) + (p.dbias ? 1 : 0);
  const int64_t pitch = (p.cols + 3) / 4 * 4;
  float *weight_parts = p.dweight, *bias_parts = p.dbias;  // (one workgroup's parts are the sums)
  const bool join = outs > 0 && grid.workgroups > 1;
  if (join) {
    DC_RETURN_IF(ensure_partials(ctx, (size_t)(grid.workgroups * outs * pitch) * sizeof(float)));
    float* parts = static_cast<float*>(ctx->partials);
    if (p.dweight) weight_parts = parts;
    if (p.dbias) bias_parts = parts + (outs - 1) * pitch;
  }
  const LayerNormGradArgs a{p.dy,        p.h,         p.weight,    p.dh,         p.dx,            weight_parts, bias_parts, p.rows,
                            p.dy_stride, p.h_stride, p.dh_stride, p.dx_stride, outs * pitch, (int32_t)p.cols, p.eps};
  DC_RETURN_IF(p.dtype == DC_DTYPE_F32 ? norm_grad_by_shape<float>(ctx, a, grid, c, waves) : norm_grad_by_shape<bf16>(ctx, a, grid, c, waves));
  if (!join) return DC_OK;
  return launch_column_sums_of(ctx, static_cast<const float*>(ctx->partials), outs * pitch, pitch, p.dweight ? p.dweight : p.dbias,
                               outs > 1 ? p.dbias : nullptr, grid.workgroups, p.cols);
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
  auto launch = [&](auto kernel, int64_t each) {
    const int64_t total = across * ((rows + each - 1) / each);
    const QuantizeArgs a{x, q, scales, rows, cols, x_stride, q_stride, scales_stride, across, total};
    kernel<<<(unsigned)std::min((total + 3) / 4, kMaxGrid), 256, 0, ctx->stream>>>(a);
  };
  // (four rows to a wave where that leaves every CU some waves, else a row to a wave)
  const bool few = across * ((rows + 3) / 4) < 4 * (int64_t)ctx->cu_count, once = read_once(rows, cols, size_of(dtype) + 1);
  auto by_type = [&](auto zero) {
    typedef decltype(zero) T;
    if (few) launch(quantize_blocks_kernel<T, 1, false>, 1);
    else once ? launch(quantize_blocks_kernel<T, 4, true>, 4) : launch(quantize_blocks_kernel<T, 4, false>, 4);
  };
  dtype == DC_DTYPE_F32 ? by_type(0.0f) : by_type(bf16{});
  return last_launch_status();
}

}  // extern "C"
