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
// |v| as an ordered integer: larger magnitudes compare larger, infinities above all finite ones, NaN above those.
__device__ inline uint32_t magnitude(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }

}  // namespace dc
