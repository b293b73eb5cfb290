// dc_numeric.hpp — element types of the feed-forward block's operators (float32, bfloat16, 8-bit e4m3) in
// 16-byte chunks at the elements' own alignment, conversions, and wave64 reductions of 32-bit values.
#pragma once

#include "dc_device.hpp"

namespace dc {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// The same at the alignment of one element (global memory takes such accesses whole).
typedef float f32x4_at4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4_at2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4_at1 __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t u32x2_at2 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32x2_at1 __attribute__((ext_vector_type(2), aligned(1)));
typedef uint32_t u32_at1 __attribute__((aligned(1)));

struct bf16 {
  uint16_t bits;
};

constexpr float kFp8Top = 448.0f;         // the largest e4m3 value
constexpr float kFp8Least = 0x1p-9f;      // the smallest one above zero

// Two floats to packed bf16, round-to-nearest-even (v_cvt_pk_bf16_f32), and back.
__device__ inline uint32_t pack_bf16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2));
}
__device__ inline float bf16_lo(uint32_t w) { return __builtin_bit_cast(float, w << 16); }
__device__ inline float bf16_hi(uint32_t w) { return __builtin_bit_cast(float, w & 0xffff0000u); }
__device__ inline float to_f32(bf16 v) { return __builtin_bit_cast(float, (uint32_t)v.bits << 16); }
__device__ inline float to_f32(float v) { return v; }
template <typename T>
__device__ inline T from_f32(float v);
template <>
__device__ inline float from_f32<float>(float v) { return v; }
template <>
__device__ inline bf16 from_f32<bf16>(float v) { return bf16{(uint16_t)pack_bf16(v, 0.0f)}; }

// Four floats to packed e4m3, round-to-nearest-even. Values past the largest become it (the conversion itself
// makes them NaN); NaN stays NaN, for which a median would not do.
__device__ inline float clamp_fp8(float v) { return v > kFp8Top ? kFp8Top : v < -kFp8Top ? -kFp8Top : v; }
__device__ inline uint32_t pack_fp8(float a, float b, float c, float d) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(clamp_fp8(a), clamp_fp8(b), 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(clamp_fp8(c), clamp_fp8(d), lo, true);
}
// The scale of values of at most `top`, and what they are multiplied with to become codes. 448 / top is no float where top is below
// 448 2^-128: such values are held as their products with 2^128 (the largest float, within its rounding), zeros as zeros.
__device__ inline float fp8_scale(float top) {
  const float s = top / kFp8Top;
  return top > 0.0f && s < 0x1p-128f ? 0x1p-128f : s;
}
__device__ inline float fp8_factor(float top) {
  const float f = kFp8Top / top;
  return f > __FLT_MAX__ ? __FLT_MAX__ : f;
}

// 16-byte chunks: kElems<T> elements of T as floats, at the elements' own alignment.
template <typename T>
constexpr int kElems = 16 / (int)sizeof(T);

__device__ inline void load_chunk(const float* p, float (&v)[4]) {
  const f32x4_at4 w = *reinterpret_cast<const f32x4_at4*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = w[i];
}
__device__ inline void unpack_bf16(u32x4 w, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = bf16_lo(w[i]);
    v[2 * i + 1] = bf16_hi(w[i]);
  }
}
__device__ inline void load_chunk(const bf16* p, float (&v)[8]) {
  unpack_bf16(*reinterpret_cast<const u32x4_at2*>(p), v);
}
__device__ inline void store_chunk(float* p, const float (&v)[4]) {
  const f32x4 w = {v[0], v[1], v[2], v[3]};
  *reinterpret_cast<f32x4_at4*>(p) = w;
}
__device__ inline void store_chunk(bf16* p, const float (&v)[8]) {
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<u32x4_at2*>(p) = w;
}
__device__ inline void store_chunk(uint8_t* p, const float (&v)[8]) {
  u32x2 w = {pack_fp8(v[0], v[1], v[2], v[3]), pack_fp8(v[4], v[5], v[6], v[7])};
  *reinterpret_cast<u32x2_at1*>(p) = w;
}
__device__ inline void store_chunk(uint8_t* p, const float (&v)[4]) {
  *reinterpret_cast<u32_at1*>(p) = pack_fp8(v[0], v[1], v[2], v[3]);
}
template <>
__device__ inline uint8_t from_f32<uint8_t>(float v) { return (uint8_t)pack_fp8(v, v, v, v); }

// Chunks as they lie in memory, and their values.
template <typename T>
__device__ inline u32x4 load_raw(const T* p) {
  if constexpr (sizeof(T) == 4) return __builtin_bit_cast(u32x4, *reinterpret_cast<const f32x4_at4*>(p));
  else return *reinterpret_cast<const u32x4_at2*>(p);
}
// The same of what no cache need keep.
template <typename T>
__device__ inline u32x4 load_raw_once(const T* p) {
  if constexpr (sizeof(T) == 4) return __builtin_bit_cast(u32x4, __builtin_nontemporal_load(reinterpret_cast<const f32x4_at4*>(p)));
  else return __builtin_nontemporal_load(reinterpret_cast<const u32x4_at2*>(p));
}
// Whether a call's operands, `bytes` for each element, are more than the last cache (256 MiB) keeps beside twice as much of others; then no cache need keep them.
// us, kept / not, each call over one of three sets of operands in turn: layer norm bf16 2000×4096 (66 MB) 11.8 / 13.0, 3000×4096 18.3 / 18.2, 4000×4096
// 25.2 / 23.1, 8191×2050 28.1 / 25.5, 2000×12000 37.7 / 35.0; gradients 16384×512 (67 MB) 16.5 / 18.0, 8192×4096 56 / 51, float32 2000×2048 (66 MB)
// 17.2 / 19.6, 4000×2048 31.6 / 29.0, 8192×2048 56.5 / 49.2; rows in 8 bits 3000×8192 (74 MB) 14.0 / 15.6, 5000×8192 25.2 / 23.3, 8191×8190 43.5 / 40.4;
// a gated layer's gradients 2000×2504×1000 (70 MB beside the products) 80.6 / 86.0, 7819×2048×64 (224 MB) 93.7 / 77.2, 8192×8192×2048 1069 / 1062.
inline bool read_once(int64_t rows, int64_t cols, int64_t bytes) { return rows * cols > (int64_t(96) << 20) / bytes; }
__device__ inline void unpack(u32x4 w, float (&v)[8]) { unpack_bf16(w, v); }
__device__ inline void unpack(u32x4 w, float (&v)[4]) {
  const f32x4 f = __builtin_bit_cast(f32x4, w);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = f[i];
}
// w moved down by `bytes`, zeros from above (none left from 16 on).
__device__ inline u32x4 shift_down(u32x4 w, int64_t bytes) {
  const unsigned __int128 all = __builtin_bit_cast(unsigned __int128, w);
  return __builtin_bit_cast(u32x4, bytes < 16 ? all >> (8 * (int)bytes) : (unsigned __int128)0);
}

// The chunk at p of which `left` elements exist (the rest reads as zero, and is not stored).
template <typename T, int E>
__device__ inline void load_some(const T* p, int64_t left, float (&v)[E]) {
  if (left >= E) {
    load_chunk(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = i < left ? to_f32(p[i]) : 0.0f;
  }
}
template <typename T, int E>
__device__ inline void store_some(T* p, int64_t left, const float (&v)[E]) {
  if (left >= E) {
    store_chunk(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (i < left) p[i] = from_f32<T>(v[i]);
  }
}

// Sum and unsigned maximum over the 64 lanes of a wave, in every lane (fixed tree; all lanes active).
__device__ inline float wave_sum_f32(float v) {
  v += __builtin_bit_cast(float, dpp_u32<0xB1, 0xF>(__builtin_bit_cast(uint32_t, v)));
  v += __builtin_bit_cast(float, dpp_u32<0x4E, 0xF>(__builtin_bit_cast(uint32_t, v)));
  v += __builtin_bit_cast(float, dpp_u32<0x141, 0xF>(__builtin_bit_cast(uint32_t, v)));
  v += __builtin_bit_cast(float, dpp_u32<0x140, 0xF>(__builtin_bit_cast(uint32_t, v)));
  v += __builtin_bit_cast(float, dpp_u32<0x142, 0xA>(__builtin_bit_cast(uint32_t, v)));
  v += __builtin_bit_cast(float, dpp_u32<0x143, 0xC>(__builtin_bit_cast(uint32_t, v)));
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
__device__ inline uint32_t wave_max_u32(uint32_t v) {
  v = max(v, dpp_u32<0xB1, 0xF>(v));
  v = max(v, dpp_u32<0x4E, 0xF>(v));
  v = max(v, dpp_u32<0x141, 0xF>(v));
  v = max(v, dpp_u32<0x140, 0xF>(v));
  v = max(v, dpp_u32<0x142, 0xA>(v));
  v = max(v, dpp_u32<0x143, 0xC>(v));
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
// Sums over the 64 lanes of a wave of two values, or four: in every lane l that of the (l % 2)-th, or (l % 4)-th (fixed tree; all lanes
// active). The first steps add one value's lanes and another's in one instruction, which is half the instructions of one sum after the other.
template <int kCtrl>
__device__ inline float dpp_add(float to, float v) {
  return to + __builtin_bit_cast(float, dpp_u32<kCtrl, 0xF>(__builtin_bit_cast(uint32_t, v)));
}
// The sum over the four rows of 16 lanes of what lies in a lane's place: the instructions exchange rows 1 and 3 of one copy with 0 and 2 of another, then halves.
__device__ inline float across_rows(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto rows = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t even = rows[0], odd = rows[1];  // (a bit cast of a vector's element itself reads the first)
  const uint32_t w = __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, even) + __builtin_bit_cast(float, odd));
  const auto halves = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  const uint32_t low = halves[0], high = halves[1];
  return __builtin_bit_cast(float, low) + __builtin_bit_cast(float, high);
}
__device__ inline float pair_sums(float a, float b, bool odd) { return dpp_add<0xB1>(odd ? b : a, odd ? a : b); }
__device__ inline float wave_sums_of_four(float a, float b, float c, float d, int lane) {
  const float low = pair_sums(a, b, lane & 1), high = pair_sums(c, d, lane & 1);
  float v = dpp_add<0x4E>(lane & 2 ? high : low, lane & 2 ? low : high);
  v = dpp_add<0x124>(v, v);
  v = dpp_add<0x128>(v, v);
  return across_rows(v);
}
__device__ inline float lane_value(float v, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
// The sum over each 16 lanes, in all of them.
__device__ inline float row16_sum_f32(float v) {
  v += __builtin_bit_cast(float, dpp_u32<0xB1, 0xF>(__builtin_bit_cast(uint32_t, v)));
  v += __builtin_bit_cast(float, dpp_u32<0x4E, 0xF>(__builtin_bit_cast(uint32_t, v)));
  v += __builtin_bit_cast(float, dpp_u32<0x141, 0xF>(__builtin_bit_cast(uint32_t, v)));
  v += __builtin_bit_cast(float, dpp_u32<0x140, 0xF>(__builtin_bit_cast(uint32_t, v)));
  return v;
}
// |v| as an ordered integer: larger magnitudes compare larger, infinities above all finite ones, NaN above those.
__device__ inline uint32_t magnitude(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }


// Blocks of 128 elements of a row in 8 bits share a scale that is a power of two, held as its exponent plus 127 in a byte (255: NaN): what
// the matrix cores take beside the codes. Of values of at most `top` (a magnitude) it is the least that takes them to 448 = 1.75 2^8
// or below, 2^-127 at the least; NaN where top is infinite or NaN.
constexpr int kScaleBlock = 128;
__device__ inline uint32_t block_scale(uint32_t top) {
  const int e = (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  return top >= 0x7f800000u ? 255u : (uint32_t)(e > 0 ? e : 0);
}
// What values are multiplied with to become codes: 2^(127 - scale), exact.
__device__ inline float block_factor(uint32_t scale) {
  return __builtin_bit_cast(float, scale == 255u ? 0x7fc00000u : (254u - scale) << 23);
}
// The largest of a block's magnitudes, in its lanes, of which each holds E neighbouring elements: 16 lanes, or 32.
template <int E>
__device__ inline uint32_t block_max_u32(uint32_t v) {
  static_assert(E == 8 || E == 4, "16 or 32 lanes to a block");
  v = max(v, dpp_u32<0xB1, 0xF>(v));
  v = max(v, dpp_u32<0x4E, 0xF>(v));
  v = max(v, dpp_u32<0x141, 0xF>(v));
  v = max(v, dpp_u32<0x140, 0xF>(v));
  if constexpr (E == 4) v = max(v, (uint32_t)__shfl_xor((int)v, 16));
  return v;
}

}  // namespace dc
