// dc_linear_device.hpp — what the linear and the gated layers are made of: activations, the epilogue, the product kernels, copies of odd
// rows, the sums of parts of c, and the host's plans of scratch.
#pragma once

#include <algorithm>

#include <cstddef>
#include <type_traits>

#include "dc_gemm_tile.hpp"
#include "dc_internal.hpp"
#include "dc_linear_route.hpp"
#include "dc_numeric.hpp"

namespace {

using dc::bf16;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4_ptr;

// ---- activations -----------------------------------------------------------------------------------
// exp and the reciprocal are the hardware's (about an ulp): the results are rounded to bf16, or are float32
// values whose sums carry more error than that.
__device__ inline float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.0f + __expf(-v)); }
constexpr float kTanhArg = 2.0f * 0.7978845608f;  // 2 sqrt(2 / pi)
constexpr float kTanhCube = 0.044715f;

// P(z), the normal distribution's function, from *e = exp(-z^2 / 2). Left of zero it is e^(-x^2) erfc(x) e^(x^2) / 2 with x = |z| / sqrt(2), a
// product in which nothing cancels; the scaled erfc is t times a polynomial in t = 1 / (1 + 0.33 x), whose eight coefficients here
// were fitted to it for the least relative error over x < 9.4 (8.2e-8, by reweighted least squares). So P is within 8e-7 of
// itself down to z = -5, and 5e-6 down to -13, where e's exponent is what is rounded: results in float32 keep their digits in
// the tail too. (A polynomial of the fifth degree with an absolute bound, which is three products cheaper, was off by 0.16 %
// of P at -5 and 1 % at -8, more than the rounding to bf16. Measured, us, that / this:
// 1537×2049×1023 25.9 / 25.8, 8192×8192×1024 169 / 172, both gradients of 8192,8192,2048 550 / 549.)
__device__ inline float normal_part(float z, float* e) {
  const float x = __builtin_fabsf(z) * 0.70710678f;
  *e = __expf(-0.5f * z * z);
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.33f, x, 1.0f));
  float q = __builtin_fmaf(-0.0679644048f, t, 0.231344149f);
  q = __builtin_fmaf(q, t, -0.177719533f);
  q = __builtin_fmaf(q, t, 0.206270859f);
  q = __builtin_fmaf(q, t, 0.0225052908f);
  q = __builtin_fmaf(q, t, 0.100961924f);
  q = __builtin_fmaf(q, t, 0.0914186165f);
  q = __builtin_fmaf(q, t, 0.0931830555f);
  q *= t * *e;
  return z > 0.0f ? 1.0f - q : q;
}

// z = act(z), E of them; the choice is made once.
template <int E>
__device__ inline void activate(int act, float (&z)[E]) {
  switch (act) {
    case DC_ACT_RELU:
#pragma unroll
      for (int e = 0; e < E; ++e) z[e] = z[e] < 0.0f ? 0.0f : z[e];
      break;
    case DC_ACT_GELU:
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float t;
        z[e] *= normal_part(z[e], &t);
      }
      break;
    case DC_ACT_GELU_TANH:
#pragma unroll
      for (int e = 0; e < E; ++e) z[e] *= sigmoid(kTanhArg * z[e] * __builtin_fmaf(kTanhCube, z[e] * z[e], 1.0f));
      break;
    case DC_ACT_SILU:
#pragma unroll
      for (int e = 0; e < E; ++e) z[e] *= sigmoid(z[e]);
      break;
    default: break;
  }
}

// g *= act'(z)
template <int E>
__device__ inline void apply_slope(int act, const float (&z)[E], float (&g)[E]) {
  switch (act) {
    case DC_ACT_RELU:
#pragma unroll
      for (int e = 0; e < E; ++e) g[e] *= z[e] > 0.0f ? 1.0f : 0.0f;
      break;
    case DC_ACT_GELU:
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float t;
        const float part = normal_part(z[e], &t);
        g[e] *= part + z[e] * t * 0.3989422804f;
      }
      break;
    case DC_ACT_GELU_TANH:
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float zz = fminf(z[e] * z[e], 1e4f);  // (past |z| = 100 the slope is 0 or 1, and z^2 may not be finite)
        const float s = sigmoid(kTanhArg * z[e] * __builtin_fmaf(kTanhCube, zz, 1.0f));
        g[e] *= s + z[e] * s * (1.0f - s) * (kTanhArg * __builtin_fmaf(3.0f * kTanhCube, zz, 1.0f));
      }
      break;
    case DC_ACT_SILU:
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float s = sigmoid(z[e]);
        g[e] *= s * __builtin_fmaf(z[e], 1.0f - s, 1.0f);
      }
      break;
    default: break;
  }
}

// ---- epilogue --------------------------------------------------------------------------------------
struct Epilogue {
  const float *a_scales, *b_scales;  // both or neither
  const bf16 *bias, *residual;
  bf16* pre;
  void* y;
  int64_t residual_stride, pre_stride, y_stride;
  int32_t act;
  int32_t y_f32;
  int64_t part_stride;  // elements of y from one part of c to the next, where c is split (0: it is not)
};

// E neighbouring bf16 values of which `left` exist (zeros for the others).
template <int E>
__device__ inline void load_bf16(const bf16* q, int64_t left, float (&v)[E]) {
  if constexpr (E == 8) {
    dc::load_some(q, left, v);
  } else if (left >= 4) {
    const dc::u32x2_at2 w = *reinterpret_cast<const dc::u32x2_at2*>(q);
    v[0] = dc::bf16_lo(w.x), v[1] = dc::bf16_hi(w.x), v[2] = dc::bf16_lo(w.y), v[3] = dc::bf16_hi(w.y);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = e < left ? dc::to_f32(q[e]) : 0.0f;
  }
}
template <int E>
__device__ inline void store_bf16(bf16* q, int64_t left, const float (&v)[E]) {
  if constexpr (E == 8) {
    dc::store_some(q, left, v);
  } else if (left >= 4) {
    const dc::u32x2 w = {dc::pack_bf16(v[0], v[1]), dc::pack_bf16(v[2], v[3])};
    *reinterpret_cast<dc::u32x2_at2*>(q) = w;
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e < left) q[e] = dc::from_f32<bf16>(v[e]);
  }
}

// Eight of them as they lie in memory.
__device__ inline dc::u32x4 load_raw_some(const bf16* q, int64_t left) {
  if (left >= 8) return dc::load_raw(q);
  dc::u32x4 w = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < left) w[e / 2] |= (uint32_t)q[e].bits << (16 * (e & 1));
  return w;
}

// What the results of E neighbouring columns j.. share, whatever their row: read once.
template <int E>
struct Columns {
  float bias[E], scale[E];
  int64_t j, left;  // columns there are from j on

  __device__ inline void read(const Epilogue& p, int64_t first, int64_t n) {
    j = first, left = n - first;
#pragma unroll
    for (int e = 0; e < E; ++e) bias[e] = scale[e] = 0.0f;
    if (left <= 0) return;
    if (p.bias) load_bf16(p.bias + j, left, bias);
    if (p.b_scales)
#pragma unroll
      for (int e = 0; e < E; e += 4)
        dc::load_some(p.b_scales + j + e, left - e, *reinterpret_cast<float (*)[4]>(scale + e));
  }
};

// What E neighbouring results of one row take from memory, and the results from that and their sums.
template <int E>
struct Results {
  float residual[E], scale;

  __device__ inline void read(const Epilogue& p, const Columns<E>& c, int64_t i) {
    if (p.residual) load_bf16(p.residual + i * p.residual_stride + c.j, c.left, residual);
    if (p.a_scales) scale = p.a_scales[i];
  }
  template <bool kResidual = true>
  __device__ inline void finish(const Epilogue& p, const Columns<E>& c, int64_t i, float (&z)[E], int part = 0) const {
    if (p.a_scales)
#pragma unroll
      for (int e = 0; e < E; ++e) z[e] = z[e] * scale * c.scale[e];
    if (p.bias)
#pragma unroll
      for (int e = 0; e < E; ++e) z[e] += c.bias[e];
    if (p.pre) store_bf16(p.pre + i * p.pre_stride + c.j, c.left, z);
    activate(p.act, z);
    if (kResidual && p.residual)
#pragma unroll
      for (int e = 0; e < E; ++e) z[e] += residual[e];
    if (p.y_f32) {
      float* q = static_cast<float*>(p.y) + i * p.y_stride + c.j + part * p.part_stride;
#pragma unroll
      for (int e = 0; e < E; e += 4) dc::store_some(q + e, c.left - e, *reinterpret_cast<const float (*)[4]>(z + e));
    } else {
      store_bf16(static_cast<bf16*>(p.y) + i * p.y_stride + c.j, c.left, z);
    }
  }
};

// ---- epilogue of a gated layer: y = act(g) u from the sums of both projections ------------------------------------
struct GatedEpilogue {
  const float *a_scales, *b_scales, *b2_scales;  // all or none
  const bf16 *bias, *bias2;
  bf16 *pre, *pre2;
  void* y;
  int64_t pre_stride, pre2_stride, y_stride;
  int32_t act;
  int32_t y_f32;
  // Where c is split (else 0): elements of y, then float32 sums, from one part to the next, and from a gate's sum to its other factor's.
  int64_t part_stride, part_up;
};

template <int E>
struct GatedColumns {
  float bias[E], bias2[E], scale[E], scale2[E];
  int64_t j, left;

  __device__ inline void read(const GatedEpilogue& p, int64_t first, int64_t n) {
    j = first, left = n - first;
#pragma unroll
    for (int e = 0; e < E; ++e) bias[e] = bias2[e] = scale[e] = scale2[e] = 0.0f;
    if (left <= 0) return;
    if (p.bias) load_bf16(p.bias + j, left, bias);
    if (p.bias2) load_bf16(p.bias2 + j, left, bias2);
    if (p.b_scales)
#pragma unroll
      for (int e = 0; e < E; e += 4) {
        dc::load_some(p.b_scales + j + e, left - e, *reinterpret_cast<float (*)[4]>(scale + e));
        dc::load_some(p.b2_scales + j + e, left - e, *reinterpret_cast<float (*)[4]>(scale2 + e));
      }
  }
};

// E neighbouring results of row i from their sums g and u; `scale`: the row's.
template <int E>
__device__ inline void gated_finish(const GatedEpilogue& p, const GatedColumns<E>& c, int64_t i, float scale, float (&g)[E], float (&u)[E],
                                    int part = 0) {
  if (p.part_stride) {
    float* q = static_cast<float*>(p.y) + part * p.part_stride + i * p.y_stride + c.j;
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      dc::store_some(q + e, c.left - e, *reinterpret_cast<const float (*)[4]>(g + e));
      dc::store_some(q + p.part_up + e, c.left - e, *reinterpret_cast<const float (*)[4]>(u + e));
    }
    return;
  }
  if (p.a_scales)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      g[e] = g[e] * scale * c.scale[e];
      u[e] = u[e] * scale * c.scale2[e];
    }
  if (p.bias)
#pragma unroll
    for (int e = 0; e < E; ++e) g[e] += c.bias[e];
  if (p.bias2)
#pragma unroll
    for (int e = 0; e < E; ++e) u[e] += c.bias2[e];
  if (p.pre) store_bf16(p.pre + i * p.pre_stride + c.j, c.left, g);
  if (p.pre2) store_bf16(p.pre2 + i * p.pre2_stride + c.j, c.left, u);
  activate(p.act, g);
#pragma unroll
  for (int e = 0; e < E; ++e) g[e] *= u[e];
  if (p.y_f32) {
    float* q = static_cast<float*>(p.y) + i * p.y_stride + c.j;
#pragma unroll
    for (int e = 0; e < E; e += 4) dc::store_some(q + e, c.left - e, *reinterpret_cast<const float (*)[4]>(g + e));
  } else {
    store_bf16(static_cast<bf16*>(p.y) + i * p.y_stride + c.j, c.left, g);
  }
}

// ---- tiles -----------------------------------------------------------------------------------------
// Macro tile TM×TN, 128 bytes of c at a time (64 bf16 or 128 e4m3), double-buffered LDS, WM×WN waves of
// 32·kMT × 32·kNT results on v_mfma_f32_32x32x16_bf16 / v_mfma_f32_32x32x64_f8f6f4; KS > 1: KS such groups of waves take the
// tiles along c in turn, and their sums are added in group order at the end.
//
// LDS image of an operand whose rows run along c: T rows of 128 bytes; the 16-byte piece q of row R sits at
// q ^ ((R >> 1) & 7), so a fragment read (rows R0..R0+15 at one piece for each 16 lanes) touches 16 distinct 16-byte
// bank groups. Of an operand with rows c: 64 rows of 2·T bytes, the 64-byte block b of row c at b ^ (c & 3) (T = 64:
// b ^ ((c >> 1) & 1)), read through ds_read_b64_tr_b16, which hands a lane four c of one column. The swizzles are
// applied where the direct-to-LDS loads fetch: lane L of a load fills LDS bytes 16·L of a 1 KiB block.
//
// The instructions get B's fragment first and A's second, so a lane ends up with four neighbouring j of one i: the
// sums go through LDS once more, a wave at a time in its own part, and the epilogue reads and writes rows of 8 results
// a lane, 64 or 128 bytes a row, whatever the activation, in one short loop.
//
// Bound by the matrix cores (by the clock they hold) in 256-tiles: bf16 8192^3 842-853 us (1.29-1.31 PFLOP/s), 876 with tanh-gelu
// and pre; 8192×2048×8192 213; both gradients of 8192,8192,2048 445 for 550 GFLOP; e4m3 4096×8192×4096 113.6 (2.42). What is left is each round's end: the
// 256 tiles of a round write 33.5 MB at once, and their epilogue has no products beside it (8-14 us a round; a persistent workgroup that
// loads its next tile over its epilogue gained 2-3 % in bf16 and spilled in 8 bits). Smaller tiles are bound by the 28
// bytes a cycle that a CU's direct-to-LDS loads bring, and by launch and latency: 2048^3 22.7, 1537×2049×1024 13.7.
constexpr int kTileBytes = 128;  // of c
constexpr int kRange = dc::kLinearRange;
constexpr uint32_t kPast = 0x80000000u;  // a byte offset past every range: loads zeros

struct Operands {
  const unsigned char *a, *b;
  int64_t a_pitch, b_pitch;  // bytes from row to row
  int32_t m, n;              // results
  int32_t c_bytes;           // A's row length; B's too, or c_rows of them
  int32_t c_rows;
  int32_t b_cols;            // B's columns with their padding, a multiple of 8 (rows c only)
};

// What a second weight, and block scales of e4m3 operands, add to those.
struct MoreOperands : Operands {
  // Gated forward: the other projection's weight. Its gradient: what B's rows c are from c_half (a whole number of tiles) on; c_rows of each.
  const unsigned char* b2;
  int64_t b2_pitch;
  int32_t c_half;
  // Block scales, [blocks][rows]: of A, B and b2.
  const uint8_t *a_codes, *b_codes, *b2_codes;
  int64_t a_codes_pitch, b_codes_pitch, b2_codes_pitch;
};
// A byte for each of 64 lanes from `offset` (the lane's) past `base`, of which `left` are there: zeros for the others. (The scale of a row that is not
// there reaches no result that is.)
__device__ inline int load_code(const uint8_t* base, int left, int offset) {
  return __builtin_amdgcn_raw_buffer_load_b8(dc::range_rsrc(base, left > 0 ? left : 0), offset, 0, 0);
}

template <int TM, int TN>
struct TileSmem {
  unsigned char a[2][TM * kTileBytes];
  unsigned char b[2][TN * kTileBytes];
};

template <bool kFp8>
struct Frag;
template <>
struct Frag<false> {
  bf16x8 v;
};
template <>
struct Frag<true> {
  i32x8 v;
};

// 16 bytes a lane to 1 KiB of LDS, from `voff` (the lane's, kPast for zeros) + `soff` bytes past `base`. kOnce: of what no cache need keep (nontemporal).
template <bool kOnce = false>
__device__ inline void load_block(const unsigned char* base, unsigned char* to, uint32_t voff, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(dc::range_rsrc(base, kRange), (dc::lds_ptr_t)to, 16, voff, soff, 0, kOnce ? 2 : 0);
}

// The products of one launch. Workgroups take the first's tiles, part of c by part, then the second's: the two
// gradients of a layer seldom fill the chip by themselves, and a launch saved is 3-5 us.
template <class O, class E>
struct JobOf {
  O o;
  E ep;
  int32_t tiles_m, tiles_n;
  int32_t parts, turns;  // of c, and tiles along c in each
};
// The workgroups after those add the parts of dbias. (A launch of their own took 2 us more: both gradients with dbias,
// 200,400,512 13.0 / 11.2, 2000,3000,1000 60.7 / 58.5.)
struct ColumnParts {
  const float* parts;  // [count][n]
  float* out;
  int32_t count, n;
};
// Of two projections: columns from `half` on are out2's. Either may be NULL.
struct ColumnPartsOfTwo : ColumnParts {
  float* out2;
  int32_t half;
};
// What product_kernel takes. kGated forward: both projections' products in one, and the gate; rows c: three gradients, the first of both
// weights' rows along c.
template <bool kRowsC, bool kGated, bool kBlocks>
struct ProductTypes {
  static constexpr int kJobs = !kRowsC ? 1 : kGated ? 3 : 2;
  typedef std::conditional_t<kGated || kBlocks, MoreOperands, Operands> O;
  typedef std::conditional_t<kGated && !kRowsC, GatedEpilogue, Epilogue> E;
  typedef std::conditional_t<kGated && kRowsC, ColumnPartsOfTwo, ColumnParts> Columns;
  struct Jobs {
    JobOf<O, E> job[kJobs];
    int32_t ends[kJobs];  // workgroups of the first, of the first two, ...
    int32_t base;         // of the launches before this one
    Columns columns;
  };
};

// out[c] = parts[0][c] + ... for kThr / 16 columns a workgroup: 16 threads a column add every 16th part each, then those
// sums in order.
template <int kThr, class A>
__device__ inline void add_parts(const A& a, int block, float* lds) {
  constexpr int kCols = kThr / 16;
  const int at = threadIdx.x % kCols, g = threadIdx.x / kCols;
  const int64_t c = (int64_t)block * kCols + at;
  float v = 0.0f;
  if (c < a.n)
#pragma unroll 4
    for (int64_t i = g; i < a.count; i += 16) v += a.parts[i * a.n + c];
  lds[threadIdx.x] = v;
  __syncthreads();
  if (g > 0 || c >= a.n) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) v += lds[i * kCols + at];
  if constexpr (std::is_same_v<A, ColumnPartsOfTwo>) {
    float* out = c < a.half ? a.out : a.out2;
    if (out) out[c < a.half ? c : c - a.half] = v;
  } else {
    a.out[c] = v;
  }
}

// kGated forward: B's LDS rows are 32 of the gate's weight, 32 of the other's and so on, so that a lane gets both sums of an output; TN counts both.
// kBlocks: the instructions take a scale for each row and 128 bytes of c, a tile's, beside the operands: asked for from memory a tile ahead, 32 neighbouring
// bytes for each 32 rows.
template <int TM, int TN, int WM, int WN, int KS, bool kFp8, bool kRowsC, bool kGated, bool kBlocks>
__global__ __launch_bounds__(64 * WM * WN * KS, (WM * WN == 8 ? 1 : 2)) void product_kernel(typename ProductTypes<kRowsC, kGated, kBlocks>::Jobs jobs) {
  static_assert(!(kFp8 && kRowsC), "8-bit operands run along c");
  static_assert(!kBlocks || kFp8, "bf16 operands have no scales");
  typedef ProductTypes<kRowsC, kGated, kBlocks> Types;
  constexpr bool kPairs = kGated && !kRowsC;  // of sums
  constexpr int kWaves = WM * WN;
  constexpr int kMT = TM / WM / 32, kNT = TN / WN / 32;
  constexpr int kABlocks = TM / 8 / kWaves, kBBlocks = TN / 8 / kWaves;  // 1 KiB blocks of a wave and tile
  constexpr int kSteps = kFp8 ? 2 : 4;                                   // instructions along c of a tile
  using Smem = TileSmem<TM, TN>;
  __shared__ __align__(16) Smem sms[KS];
  int block = jobs.base + (int)blockIdx.x;
  if constexpr (kRowsC)
    if (block >= jobs.ends[Types::kJobs - 1])
      return add_parts<64 * kWaves * KS>(jobs.columns, block - jobs.ends[Types::kJobs - 1], reinterpret_cast<float*>(sms));
  int which = 0, before = 0;
#pragma unroll
  for (int i = 0; i + 1 < Types::kJobs; ++i)
    if (block >= jobs.ends[i]) which = i + 1, before = jobs.ends[i];
  block -= before;
  const auto& job = jobs.job[which];
  const auto& o = job.o;
  const auto& ep = job.ep;
  const int tiles = job.tiles_m * job.tiles_n, part = job.parts > 1 ? block / tiles : 0, turns = job.turns;
  const dc::TileCoord tc = dc::map_tile(block - part * tiles, job.tiles_m, job.tiles_n);
  const int m0 = tc.tm * TM, n0 = tc.tn * (kPairs ? TN / 2 : TN);
  const int tid = threadIdx.x, lane = tid & 63, gwave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = gwave / kWaves, wave = gwave % kWaves;
  Smem& sm = sms[group];
  const int wm = wave / WN, wn = wave % WN;
  const int r = lane & 31, h = lane >> 5;
  const int tiles_c = (o.c_bytes + kTileBytes - 1) / kTileBytes;
  // Tiles along c of a group: `turns` of them from kt_first on, fewer in the last of the parts that c is split into
  const int kt_first = part * turns;
  const int kt_count = min((tiles_c + KS - 1) / KS - kt_first, turns);
  // Where c ends here. kAlways: tiles past it are asked for too, as zeros, so that no branch stands between a tile's products
  // (the compiler would move those before it past it, and past the barrier).
  constexpr bool kAlways = TM == 256 && kFp8;
  const int c_end = min(o.c_bytes, (kt_first + kt_count) * KS * kTileBytes), c_rows = min(o.c_rows, c_end / 2);

  // ---- load side. Rows along c: lane -> row lane / 8 of a block, slot lane % 8, which holds the piece of the swizzle.
  const int lrow = lane >> 3;
  const int piece = 16 * ((lane & 7) ^ ((4 * wave + (lrow >> 1)) & 7));  // byte offset in the row's 128
  // Rows c: lane -> row of the block and 16-byte chunk of it.
  constexpr int kRowChunks = TN / 8, kRows = 64 / kRowChunks;
  auto bswz = [](int c) __attribute__((always_inline)) { return TN == 64 ? (c >> 1) & 1 : c & 3; };
  const int brow = lane / kRowChunks, bc = lane % kRowChunks;
  const int bchunk = 4 * ((bc >> 2) ^ bswz(kRows * wave + brow)) + (bc & 3);
  uint32_t avoff[kABlocks], bvoff[kRowsC ? 1 + kGated : kBBlocks];
  // (pairs: whether a wave's block i is of the other weight, 32 rows of each in turn)
  auto of_second = [&](int i) __attribute__((always_inline)) { return ((i * kWaves + wave) >> 2 & 1) != 0; };
#pragma unroll
  for (int i = 0; i < kABlocks; ++i)
    avoff[i] = (uint32_t)min(8 * (i * kWaves + wave) + lrow, o.m - 1 - m0) * (uint32_t)o.a_pitch + (uint32_t)piece;
  if constexpr (kRowsC) {
    bvoff[0] = (uint32_t)brow * (uint32_t)o.b_pitch + (uint32_t)(2 * min(8 * bchunk, o.b_cols - 8 - n0));
    if constexpr (kGated) bvoff[1] = (uint32_t)brow * (uint32_t)o.b2_pitch + (uint32_t)(2 * min(8 * bchunk, o.b_cols - 8 - n0));
  } else if constexpr (kPairs) {
#pragma unroll
    for (int i = 0; i < kBBlocks; ++i) {
      const int row = 8 * (i * kWaves + wave) + lrow;
      bvoff[i] = (uint32_t)min((row >> 6) * 32 + (row & 31), o.n - 1 - n0) * (uint32_t)(of_second(i) ? o.b2_pitch : o.b_pitch) + (uint32_t)piece;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kBBlocks; ++i)
      bvoff[i] = (uint32_t)min(8 * (i * kWaves + wave) + lrow, o.n - 1 - n0) * (uint32_t)o.b_pitch + (uint32_t)piece;
  }
  const unsigned char* abase = o.a + (int64_t)m0 * o.a_pitch;
  const unsigned char* bbase = kRowsC ? o.b + (int64_t)n0 * 2 : o.b + (int64_t)n0 * o.b_pitch;
  const unsigned char* b2base = nullptr;
  if constexpr (kGated) b2base = kRowsC ? o.b2 + (int64_t)n0 * 2 : o.b2 + (int64_t)n0 * o.b2_pitch;
  auto load_tile = [&](auto BUF, int KT) __attribute__((always_inline)) {
    constexpr int kBuf = decltype(BUF)::value;
    const int t = (kt_first + KT) * KS + group;
    const int at = t * kTileBytes;  // bytes into A's rows (past the last: every load is past the range)
    const int left = c_end - at;
#pragma unroll
    for (int i = 0; i < kABlocks; ++i)
      load_block(abase + at, sm.a[kBuf] + (i * kWaves + wave) * 1024, piece < left ? avoff[i] : kPast, 0);
    if constexpr (kRowsC && kGated) {
      // (dz has a whole number of tiles for each weight, so that only a tile past c_end is not all one's; a row past the weight's last is zeros)
      const bool other = t * (kTileBytes / 2) >= o.c_half;
      const int c0 = t * (kTileBytes / 2) - (other ? o.c_half : 0), rows = left > 0 ? o.c_rows : 0;
      const int64_t pitch = other ? o.b2_pitch : o.b_pitch;
#pragma unroll
      for (int i = 0; i < kBBlocks; ++i) {
        const int row = kRows * (i * kWaves + wave);
        load_block((other ? b2base : bbase) + (int64_t)c0 * pitch, sm.b[kBuf] + (i * kWaves + wave) * 1024,
                   c0 + row + brow < rows ? (other ? bvoff[1] : bvoff[0]) : kPast, row * (int)pitch);
      }
    } else if constexpr (kRowsC) {
      const int c0 = t * (kTileBytes / 2);
#pragma unroll
      for (int i = 0; i < kBBlocks; ++i) {
        const int row = kRows * (i * kWaves + wave);
        load_block(bbase + (int64_t)c0 * o.b_pitch, sm.b[kBuf] + (i * kWaves + wave) * 1024,
                   c0 + row + brow < c_rows ? bvoff[0] : kPast, row * (int)o.b_pitch);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kBBlocks; ++i)
        load_block((kPairs && of_second(i) ? b2base : bbase) + at, sm.b[kBuf] + (i * kWaves + wave) * 1024, piece < left ? bvoff[i] : kPast, 0);
    }
  };

  // ---- read side: byte offsets in buffer 0 of a step's pieces, for rows 32·t + r (so the swizzle is (r >> 1) & 7).
  // bf16: piece 2·step + h; e4m3: pieces 4·step + 2h and + 1 (any split of c over the lanes' halves will do, as both
  // operands use the same).
  const int rswz = (r >> 1) & 7;
  uint32_t poff[8 / 2];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    poff[i] = 16u * (uint32_t)((kFp8 ? 4 * (i >> 1) + 2 * h + (i & 1) : 2 * i + h) ^ rswz);
  const uint32_t arow = (uint32_t)((wm * 32 * kMT + r) * kTileBytes);
  const uint32_t brow_l = (uint32_t)offsetof(Smem, b) + (uint32_t)((wn * 32 * kNT + r) * kTileBytes);
  uint32_t boff[kNT];
  if constexpr (kRowsC) {
    const int j = (lane & 15) >> 2, p4 = lane & 3, cg = (lane >> 4) & 1;
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt)
      boff[nt] = (uint32_t)offsetof(Smem, b) + (uint32_t)((8 * h + j) * 2 * TN) +
                 64u * (uint32_t)((kNT * wn + nt) ^ bswz(j)) + (uint32_t)(32 * cg + 8 * p4);
  }
  const unsigned char* lds = reinterpret_cast<const unsigned char*>(&sm);

  f32x16 acc[kMT][kNT];
#pragma unroll
  for (int i = 0; i < kMT; ++i)
#pragma unroll
    for (int j = 0; j < kNT; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.0f;

  // Block scales of the tiles in turn, of the rows that this lane's fragments hold.
  int ascale[2][kBlocks ? kMT : 1], bscale[2][kBlocks ? kNT : 1];
  // (`mark`: set in bits that the instructions do not look at, in the first tiles' alone. Without it the compiler sees bytes come into the loop from
  // both ends, carries bytes round it, and widens them at its head, where it waits for the loads that have just gone out.)
  auto load_scales = [&](auto BUF, int KT, int mark = 0) __attribute__((always_inline)) {
    if constexpr (kBlocks) {
      constexpr int kBuf = decltype(BUF)::value;
      const int64_t kb = min((kt_first + KT) * KS + group, tiles_c - 1);
      const int i0 = m0 + wm * 32 * kMT, j0 = n0 + wn * (kPairs ? 16 : 32) * kNT;
#pragma unroll
      for (int mt = 0; mt < kMT; ++mt) ascale[kBuf][mt] = load_code(o.a_codes + kb * o.a_codes_pitch + i0, o.m - i0, 32 * mt + r) | mark;
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
        if constexpr (kPairs)
          bscale[kBuf][nt] = load_code((nt & 1 ? o.b2_codes + kb * o.b2_codes_pitch : o.b_codes + kb * o.b_codes_pitch) + j0, o.n - j0, 32 * (nt >> 1) + r) | mark;
        else
          bscale[kBuf][nt] = load_code(o.b_codes + kb * o.b_codes_pitch + j0, o.n - j0, 32 * nt + r) | mark;
      }
    }
  };

  typedef Frag<kFp8> F;
  auto read_row = [&](uint32_t at, int step) __attribute__((always_inline)) {
    F f;
    if constexpr (kFp8) {
      const dc::u32x4 lo = *reinterpret_cast<const dc::u32x4*>(lds + at + poff[2 * step]);
      const dc::u32x4 hi = *reinterpret_cast<const dc::u32x4*>(lds + at + poff[2 * step + 1]);
      f.v = __builtin_bit_cast(i32x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      f.v = __builtin_bit_cast(bf16x8, *reinterpret_cast<const dc::u32x4*>(lds + at + poff[step]));
    }
    return f;
  };
  auto read_a = [&](auto BUF, int step, F* a) __attribute__((always_inline)) {
    constexpr uint32_t kBufA = (uint32_t)decltype(BUF)::value * TM * kTileBytes;
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt) a[mt] = read_row(arow + kBufA + mt * 32 * kTileBytes, step);
  };
  auto read_b = [&](auto BUF, int step, F* b) __attribute__((always_inline)) {
    constexpr uint32_t kBufB = (uint32_t)decltype(BUF)::value * TN * kTileBytes;
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) b[nt] = read_row(brow_l + kBufB + nt * 32 * kTileBytes, step);
  };
  // Rows c: the fragments of a whole tile in one burst. The compiler cannot tell these reads apart from the LDS that the
  // direct-to-LDS loads write, and waits for every load in flight before each of them: they go out while none is.
  auto read_b_tile = [&](auto BUF, F (*b)[kNT]) __attribute__((always_inline)) {
    if constexpr (kRowsC) {
      constexpr uint32_t kBufB = (uint32_t)decltype(BUF)::value * TN * kTileBytes;
#pragma unroll
      for (int st = 0; st < kSteps; ++st)
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) {
          const unsigned char* q = lds + boff[nt] + kBufB + st * 16 * 2 * TN;
          const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(q));
          const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(q + 4 * 2 * TN));
          b[st][nt].v = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
  };
  auto mfmas_of = [&](int mt, const F* a, const F* b, auto BUF) __attribute__((always_inline)) {
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      if constexpr (kBlocks)
        acc[mt][nt] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b[nt].v, a[mt].v, acc[mt][nt], 0, 0, 0, bscale[decltype(BUF)::value][nt], 0,
                                                                     ascale[decltype(BUF)::value][mt]);
      else if constexpr (kFp8)
        acc[mt][nt] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b[nt].v, a[mt].v, acc[mt][nt], 0, 0, 0, 0x7f7f7f7f, 0,
                                                                     0x7f7f7f7f);
      else
        acc[mt][nt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(b[nt].v, a[mt].v, acc[mt][nt], 0, 0, 0);
    }
  };
  auto mfmas = [&](const F* a, const F* b, auto BUF) __attribute__((always_inline)) {
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt) mfmas_of(mt, a, b, BUF);
  };
  // LDS reads between the products: as many as there are of each.
  constexpr int kReads = (kMT + (kRowsC ? 0 : kNT)) * (kFp8 ? 2 : 1), kProducts = kMT * kNT;
  auto interleave = []() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kProducts; ++i) {
      constexpr int kPer = (kReads + kProducts - 1) / kProducts;
      __builtin_amdgcn_sched_group_barrier(0x100, kPer, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    }
  };

  // Where registers are short (scales beside the largest tiles' sums and fragments): the next step's fragments of A are read one by one, each into the
  // place of one whose products have gone out, so that a wave holds five of A's and not eight.
  constexpr bool kRolled = kFp8 && (kBlocks || kPairs) && TM == 256;
  auto rolled = [&](auto FROM, int from_step, F* a, F* b, F* a_next, F* b_next, auto BUF) __attribute__((always_inline)) {
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt) {
      mfmas_of(mt, a, b, BUF);
      __builtin_amdgcn_sched_barrier(0);
      if (mt == 0) read_b(FROM, from_step, b_next);
      a_next[mt] = read_row(arow + (uint32_t)decltype(FROM)::value * TM * kTileBytes + mt * 32 * kTileBytes, from_step);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // Tile kt in buffer kt & 1: its steps run their products with the next step's reads between them; before the last
  // step comes the tile's one barrier, which also waits for tile kt+1's loads, issued a tile earlier; then tile
  // kt+2's loads go out into the buffer that tile kt is done with.
  F fa[2][kMT], fb[2][kRowsC ? kSteps : 1][kNT];
  constexpr std::integral_constant<int, 0> kBuf0{};
  constexpr std::integral_constant<int, 1> kBuf1{};
  load_tile(kBuf0, 0);
  load_scales(kBuf0, 0, kRolled ? 0x100 : 0);
  dc::dma_barrier();
  if constexpr (kRowsC) read_b_tile(kBuf0, fb[0]);
  else read_b(kBuf0, 0, fb[0][0]);
  read_a(kBuf0, 0, fa[0]);
  __builtin_amdgcn_sched_barrier(0);
  if (kAlways || kt_count > 1) load_tile(kBuf1, 1);
  load_scales(kBuf1, 1, kRolled ? 0x100 : 0);
  // (a macro, so that the fragment arrays stay plain registers)
#define DC_TILE(BUF, KT)                                                                            \
  {                                                                                                 \
    _Pragma("unroll") for (int step = 0; step + 1 < kSteps; ++step) {                               \
      const int cur = step & 1;                                                                     \
      __builtin_amdgcn_sched_barrier(0);                                                            \
      if constexpr (kRolled) {                                                                      \
        rolled(kBuf##BUF, step + 1, fa[cur], fb[cur][0], fa[cur ^ 1], fb[cur ^ 1][0], kBuf##BUF);   \
        continue;                                                                                   \
      }                                                                                             \
      read_a(kBuf##BUF, step + 1, fa[cur ^ 1]);                                                     \
      if constexpr (!kRowsC) read_b(kBuf##BUF, step + 1, fb[cur ^ 1][0]);                           \
      mfmas(fa[cur], kRowsC ? fb[BUF][kRowsC ? step : 0] : fb[cur][0], kBuf##BUF);                  \
      interleave();                                                                                 \
      __builtin_amdgcn_sched_barrier(0);                                                            \
    }                                                                                               \
    dc::dma_barrier();                                                                              \
    if constexpr (kRowsC) read_b_tile(kBuf##BUF##Other, fb[1 - (BUF)]);                             \
    __builtin_amdgcn_sched_barrier(0);                                                              \
    if (kAlways || (KT) + 2 < kt_count) load_tile(kBuf##BUF, (KT) + 2);                             \
    __builtin_amdgcn_sched_barrier(0);                                                              \
    if constexpr (kRolled) {                                                                        \
      rolled(kBuf##BUF##Other, 0, fa[1], fb[1][0], fa[0], fb[0][0], kBuf##BUF);                     \
    } else {                                                                                        \
      read_a(kBuf##BUF##Other, 0, fa[0]);                                                           \
      if constexpr (!kRowsC) read_b(kBuf##BUF##Other, 0, fb[0][0]);                                 \
      mfmas(fa[1], kRowsC ? fb[BUF][kRowsC ? kSteps - 1 : 0] : fb[1][0], kBuf##BUF);                \
      interleave();                                                                                 \
    }                                                                                               \
    __builtin_amdgcn_sched_barrier(0);                                                              \
  }
  constexpr auto kBuf0Other = kBuf1;
  constexpr auto kBuf1Other = kBuf0;
  __builtin_assume(kt_count > 0);
  int kt = 0;
  if constexpr (kRolled && kBlocks) {
    // (no branch within two tiles: where one ends, scales loaded on one side of it would be copied, and waited for: 4096×4096×8192 130 us, 124 without;
    // smaller tiles lose a workgroup of a CU's five to the registers that it takes, 2048^3 17.2 us, 18.5)
    for (; kt + 1 < kt_count; kt += 2) {
      DC_TILE(0, kt);
      load_scales(kBuf0, kt + 2);
      __builtin_amdgcn_sched_barrier(0);
      DC_TILE(1, kt + 1);
      load_scales(kBuf1, kt + 3);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (kt < kt_count) DC_TILE(0, kt);
  } else {
    do {
      DC_TILE(0, kt);
      load_scales(kBuf0, kt + 2);
      if (kt + 1 < kt_count) {
        DC_TILE(1, kt + 1);
        load_scales(kBuf1, kt + 3);
      }
      kt += 2;
    } while (kt < kt_count);
  }
#undef DC_TILE

  // (after the last tile: loads of zeros, and reads of the other buffer, that nobody uses; all are over beyond this barrier)
  dc::dma_barrier();
  if constexpr (KS > 1) {  // the groups' sums, added in group order by group 0
    static_assert(sizeof(Smem) >= kWaves * 64 * kMT * kNT * 16 * sizeof(float), "a group's sums fit in its buffers");
    float* part = reinterpret_cast<float*>(&sm) + tid % (64 * kWaves);
    if (group > 0)
#pragma unroll
      for (int i = 0; i < kMT * kNT * 16; ++i) part[i * 64 * kWaves] = acc[i / 16 / kNT][i / 16 % kNT][i % 16];
    __syncthreads();
    if (group > 0) return;
#pragma unroll
    for (int g = 1; g < KS; ++g) {
      const float* other = reinterpret_cast<const float*>(&sms[g]) + tid;
#pragma unroll
      for (int i = 0; i < kMT * kNT * 16; ++i) acc[i / 16 / kNT][i / 16 % kNT][i % 16] += other[i * 64 * kWaves];
    }
  }

  // acc[mt][nt][v]: i = r, j = 8·(v / 4) + 4·h + v % 4 of the 32×32 block. A wave's 32 rows of 32·kNT sums at a time, with the
  // rows' scales in the columns past them; a lane's residual is asked for kTurns turns of the loop ahead.
  constexpr int kCols = 32 * kNT, kPitch = kCols + 4, kLanes = kCols / 8, kRowsTurn = 64 / kLanes, kTurns = 32 / kRowsTurn;
  static_assert(sizeof(Smem) >= kWaves * 32 * kPitch * sizeof(float), "the waves' blocks fit in the buffers");
  float* own = reinterpret_cast<float*>(&sms[0]) + wave * 32 * kPitch;
  auto leave_rows = [&](int mt) __attribute__((always_inline)) {
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4 v = {acc[mt][nt][4 * q], acc[mt][nt][4 * q + 1], acc[mt][nt][4 * q + 2], acc[mt][nt][4 * q + 3]};
        *reinterpret_cast<f32x4*>(own + r * kPitch + 32 * nt + 8 * q + 4 * h) = v;
      }
  };
  if constexpr (kPairs) {
    // Columns 64 p + 0..31 are the gate's sums of outputs 32 p + 0..31, the next 32 the other projection's.
    constexpr int kPairLanes = kCols / 16, kPairRows = 64 / kPairLanes;
    const int i0 = m0 + wm * kMT * 32, own_row = lane / kPairLanes, own_out = 8 * (lane % kPairLanes);
    const int at = (own_out >> 5) * 64 + (own_out & 31);
    GatedColumns<8> cols;
    cols.read(ep, n0 + wn * (kCols / 2) + own_out, o.n);
    float scales[kMT];
    if constexpr (kFp8 && !kBlocks)
#pragma unroll
      for (int mt = 0; mt < kMT; ++mt) scales[mt] = ep.a_scales ? ep.a_scales[min(i0 + 32 * mt + r, o.m - 1)] : 1.0f;
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt) {
      leave_rows(mt);
      if constexpr (kFp8 && !kBlocks) own[r * kPitch + kCols] = scales[mt];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 1
      for (int r0 = 0; r0 < 32; r0 += kPairRows) {
        const int row = r0 + own_row;
        const int64_t i = i0 + 32 * mt + row;
        float g[8], u[8], scale = 1.0f;
        if constexpr (kFp8 && !kBlocks) scale = own[row * kPitch + kCols];
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = own[row * kPitch + at + e], u[e] = own[row * kPitch + at + 32 + e];
        if (i < o.m && cols.left > 0) gated_finish(ep, cols, i, scale, g, u, part);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  } else {
    const int i0 = m0 + wm * kMT * 32, own_row = lane / kLanes, own_col = 8 * (lane % kLanes);
    Columns<8> cols;
    cols.read(ep, n0 + wn * kCols + own_col, o.n);
    float scales[kMT];
    if constexpr (kFp8)
#pragma unroll
      for (int mt = 0; mt < kMT; ++mt) scales[mt] = ep.a_scales ? ep.a_scales[min(i0 + 32 * mt + r, o.m - 1)] : 1.0f;
    auto write = [&](auto RESIDUAL) __attribute__((always_inline)) {
      constexpr bool kResidual = decltype(RESIDUAL)::value;
      dc::u32x4 ahead[kTurns];
      auto ask = [&](int row) __attribute__((always_inline)) {
        dc::u32x4 w = {0, 0, 0, 0};
        if (ep.residual && i0 + row < o.m && cols.left > 0) w = load_raw_some(ep.residual + (i0 + row) * ep.residual_stride + cols.j, cols.left);
        return w;
      };
      if constexpr (kResidual)
#pragma unroll
        for (int q = 0; q < kTurns; ++q) ahead[q] = ask(own_row + q * kRowsTurn);
#pragma unroll
      for (int mt = 0; mt < kMT; ++mt) {
        leave_rows(mt);
        if constexpr (kFp8) own[r * kPitch + kCols] = scales[mt];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 1
        for (int r0 = 0; r0 < 32; r0 += kRowsTurn) {
          const int row = r0 + own_row;
          const int64_t i = i0 + 32 * mt + row;
          Results<8> out;
          if constexpr (kResidual) {
            dc::unpack(ahead[0], out.residual);
#pragma unroll
            for (int q = 0; q + 1 < kTurns; ++q) ahead[q] = ahead[q + 1];
            if (mt + 1 < kMT) ahead[kTurns - 1] = ask(32 * mt + row + 32);
          }
          if constexpr (kFp8) out.scale = own[row * kPitch + kCols];
          float z[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) z[e] = own[row * kPitch + own_col + e];
          if (i < o.m && cols.left > 0) out.template finish<kResidual>(ep, cols, i, z, part);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      }
    };
    // (8 bits go one way for both: with two the compiler spills, and 4096×8192×4096 measured 115.9 us, with a residual 123.5, where
    // this is 113.6 and 121.7. Residual asked for in the turn that needs it: 126.9; bf16 4096^3 120.2, as it is now 117.3.)
    if constexpr (kFp8) write(std::true_type{});
    else if (!kRowsC && ep.residual) write(std::true_type{});
    else write(std::false_type{});
  }
}

// ---- few rows ----------------------------------------------------------------------------------------
// Bound by reading w once (for every 64 rows of x). A workgroup takes a few outputs (rows of w) and up to 64 rows of x; its W waves take the 128-byte
// steps along c in turn, each on its own, and their sums are added in the order of the waves at the end. What the loads
// cost was found by measurement: a CU takes about 14 bytes a cycle in loads to registers, whatever their number in flight and
// whether they ask for whole 128-byte lines, and 28 in direct-to-LDS loads. So:
//   - few_rows_kernel: 16-byte aligned operands, through LDS. 16·NB outputs and 8·XB rows of x a workgroup; each wave has
//     D stages of LDS to itself (1 KiB for 8 rows and a step, in product_kernel's image) and keeps D - 1 steps' loads in
//     flight, so the loop has no barrier. us for bf16, loads to registers / tiles of 64 / this: 1×4096×4096 8.8 / 16.6 / 7.4 (4.6
//     TB/s with the launch), 16×4096×4096 10.0 / 16.0 / 8.0, 32×8192×4096 19.1 / 17.5 / 14.0, 32×2048×8192 23.8 / 28.4 / 11.5,
//     64×2048×8192 38.0 / 30.6 / 16.0.
//   - few_rows_any_kernel: any alignment, straight from memory to the operands of v_mfma_f32_16x16x32_*. A load asks for 8 rows
//     of 128 bytes: lane l the piece 4·p + g of row l % 8, with p = l / 8 % 2 and g = l / 16. As the instruction's operands that is
//     16 rows (8 of w, each with both halves p of the step) times 16 columns (8 of x, likewise); of its results those with
//     the same half on both sides are wanted, and the two halves' are added.
// The 16 bytes at `from`, of which `left` exist, in a row of `bytes`: a ragged piece is cut out of the row's last 16 bytes.
__device__ inline dc::u32x4 load_piece(const unsigned char* from, int64_t left, int64_t bytes) {
  dc::u32x4 w = {0, 0, 0, 0};
  if (left >= 16) {
    w = *reinterpret_cast<const dc::u32x4_at1*>(from);
  } else if (left > 0 && bytes >= 16) {
    w = *reinterpret_cast<const dc::u32x4_at1*>(from + left - 16);
    w = __builtin_bit_cast(dc::u32x4, __builtin_bit_cast(unsigned __int128, w) >> (8 * (16 - (int)left)));
  } else if (left > 0) {
    unsigned char* p = reinterpret_cast<unsigned char*>(&w);
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < left) p[i] = from[i];
  }
  return w;
}

template <bool kFp8, int MT, int NB, int W, int U>
__global__ __launch_bounds__(64 * W) void few_rows_any_kernel(Operands o, Epilogue ep) {
  __shared__ f32x4 sums[W][NB * MT][32];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool wanted = (lane >> 3 & 1) == lane >> 5;  // of the results
  const int r = lane & 7, piece = 16 * (4 * (lane >> 3 & 1) + (lane >> 4));
  const int64_t n0 = (int64_t)blockIdx.x * 8 * NB;
  const unsigned char* wrow[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) wrow[i] = o.b + std::min<int64_t>(n0 + 8 * i + r, o.n - 1) * o.b_pitch + piece;
  const int bytes = o.c_bytes, whole = bytes / kTileBytes, steps = (bytes + kTileBytes - 1) / kTileBytes;
  for (int64_t m0 = (int64_t)blockIdx.y * 8 * MT; m0 < o.m; m0 += (int64_t)gridDim.y * 8 * MT) {
    const unsigned char* xrow[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) xrow[i] = o.a + std::min<int64_t>(m0 + 8 * i + r, o.m - 1) * o.a_pitch + piece;
    f32x4 acc[NB][MT];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int j = 0; j < MT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // U steps of this wave from step s on: the next U steps' loads are in flight while the products of these run. (Steps past
    // the last whole one are zeros; the conditions are uniform.)
    auto load = [&](dc::u32x4 (&wv)[U][NB], dc::u32x4 (&xv)[U][MT], int s) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t at = (int64_t)(s + u * W) * kTileBytes;
        if (s + u * W < whole) {
#pragma unroll
          for (int i = 0; i < NB; ++i) wv[u][i] = *reinterpret_cast<const dc::u32x4_at1*>(wrow[i] + at);
#pragma unroll
          for (int i = 0; i < MT; ++i) xv[u][i] = *reinterpret_cast<const dc::u32x4_at1*>(xrow[i] + at);
        } else {
#pragma unroll
          for (int i = 0; i < NB; ++i) wv[u][i] = dc::u32x4{0, 0, 0, 0};
#pragma unroll
          for (int i = 0; i < MT; ++i) xv[u][i] = dc::u32x4{0, 0, 0, 0};
        }
      }
      __builtin_amdgcn_sched_barrier(0);  // (else the compiler saves registers by waiting for each pair)
    };
    auto add = [&](const dc::u32x4 (&wv)[NB], const dc::u32x4 (&xv)[MT]) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          const dc::u32x4 a = wv[i], b = xv[j];
          if constexpr (kFp8) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const dc::u32x2 ah = {a[2 * q], a[2 * q + 1]}, bh = {b[2 * q], b[2 * q + 1]};
              acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_fp8_fp8(__builtin_bit_cast(long, ah), __builtin_bit_cast(long, bh),
                                                                    acc[i][j], 0, 0, 0);
            }
          } else {
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b),
                                                               acc[i][j], 0, 0, 0);
          }
        }
    };
    dc::u32x4 wa[U][NB], xa[U][MT], wb[U][NB], xb[U][MT];
    load(wa, xa, wave);
    for (int s = wave; s < whole; s += 2 * U * W) {
      load(wb, xb, s + U * W);
#pragma unroll
      for (int u = 0; u < U; ++u) add(wa[u], xa[u]);
      if (s + U * W >= whole) break;
      load(wa, xa, s + 2 * U * W);
#pragma unroll
      for (int u = 0; u < U; ++u) add(wb[u], xb[u]);
    }
    if (steps > whole && whole % W == wave) {  // the last, ragged step
      const int64_t at = (int64_t)whole * kTileBytes;
#pragma unroll
      for (int i = 0; i < NB; ++i) wa[0][i] = load_piece(wrow[i] + at, bytes - at - piece, bytes);
#pragma unroll
      for (int i = 0; i < MT; ++i) xa[0][i] = load_piece(xrow[i] + at, bytes - at - piece, bytes);
      add(wa[0], xa[0]);
    }
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int j = 0; j < MT; ++j)
        if (wanted) sums[wave][i * MT + j][lane & 31] = acc[i][j];
    __syncthreads();
    // acc[i][j][v] of lane 16·g + c: row 4·g + v, column c. Output 8·i + 4·q + v of row 8·j + l of x: row 4·q + v, column l
    // (the first halves: lane 16·q + l) and row 8 + 4·q + v, column 8 + l (lane 32 + 16·q + 8 + l).
    for (int t = threadIdx.x; t < NB * MT * 16; t += 64 * W) {
      const int b = t >> 4, l = t & 7, q = t >> 3 & 1;
      f32x4 v = sums[0][b][16 * q + l] + sums[0][b][16 * q + 8 + l];
#pragma unroll
      for (int w = 1; w < W; ++w) v += sums[w][b][16 * q + l] + sums[w][b][16 * q + 8 + l];
      const int64_t i = m0 + 8 * (b % MT) + l, j = n0 + 8 * (b / MT) + 4 * q;
      float z[4] = {v.x, v.y, v.z, v.w};
      if (i < o.m && j < o.n) {
        Columns<4> cols;
        Results<4> out;
        cols.read(ep, j, o.n);
        out.read(ep, cols, i);
        out.finish(ep, cols, i, z);
      }
    }
    __syncthreads();
  }
}

template <int N>
__device__ inline void wait_loads() {  // until at most N of the wave's loads are in flight
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// kGated: the second half of the NB blocks of 16 rows of w are the other weight's, so that a workgroup has 8 NB outputs. kBlocks: the lanes of group g
// hold the scales of every fourth of the wave's steps from its g-th on, a load for four steps; a step's are handed over within the wave. kOnce: the weights
// are more than the caches keep.
template <bool kFp8, int XB, int NB, int W, int D, bool kGated, bool kBlocks, bool kOnce = false>
__global__ __launch_bounds__(64 * W) void few_rows_kernel(typename ProductTypes<false, kGated, kBlocks>::O o,
                                                          typename ProductTypes<false, kGated, kBlocks>::E ep) {
  static_assert(!kGated || NB % 2 == 0, "as many blocks of both weights");
  constexpr int kOut = kGated ? NB / 2 : NB;  // blocks of 16 outputs
  constexpr int MT = (XB + 1) / 2, kStage = (2 * NB + XB) * 1024, kLoads = 2 * NB + XB;
  static_assert((D - 1) * kLoads < 64 && W * D * kStage <= 160 * 1024 && W * NB * MT * 1024 <= W * D * kStage);
  __shared__ __align__(16) unsigned char ring[W * D * kStage];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  unsigned char* own = ring + wave * D * kStage;
  const int64_t n0 = (int64_t)blockIdx.x * 16 * kOut, m0 = (int64_t)blockIdx.y * 8 * XB;
  // load side: lane -> row lane / 8 of a block of 8, slot lane % 8, which holds the piece of the swizzle
  const int piece = 16 * ((lane & 7) ^ (lane >> 4));  // of even blocks; of odd ones 64 bytes away
  uint32_t woff[2 * NB], xoff[XB];
#pragma unroll
  for (int i = 0; i < 2 * NB; ++i) {
    const int row = 8 * (i % (2 * kOut)) + (lane >> 3);
    int64_t pitch = o.b_pitch;
    if constexpr (kGated) pitch = i < 2 * kOut ? o.b_pitch : o.b2_pitch;
    woff[i] = n0 + row < o.n ? (uint32_t)row * (uint32_t)pitch + (uint32_t)(piece ^ (64 * (i & 1))) : kPast;
  }
#pragma unroll
  for (int i = 0; i < XB; ++i) {
    const int row = 8 * i + (lane >> 3);
    xoff[i] = m0 + row < o.m ? (uint32_t)row * (uint32_t)o.a_pitch + (uint32_t)(piece ^ (64 * (i & 1))) : kPast;
  }
  const unsigned char *wbase = o.b + n0 * o.b_pitch, *xbase = o.a + m0 * o.a_pitch, *w2base = nullptr;
  if constexpr (kGated) w2base = o.b2 + n0 * o.b2_pitch;
  const int steps = (o.c_bytes + kTileBytes - 1) / kTileBytes;
  auto load = [&](unsigned char* stage, int s) __attribute__((always_inline)) {
    const int64_t at = (int64_t)s * kTileBytes;
    const int left = o.c_bytes - s * kTileBytes;
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i)
      load_block<kOnce>((kGated && i >= 2 * kOut ? w2base : wbase) + at, stage + i * 1024, (piece ^ (64 * (i & 1))) < left ? woff[i] : kPast, 0);
#pragma unroll
    for (int i = 0; i < XB; ++i)
      load_block(xbase + at, stage + (2 * NB + i) * 1024, (piece ^ (64 * (i & 1))) < left ? xoff[i] : kPast, 0);
  };
  // read side: pieces g and 4 + g of row lane % 16 (of an x block that is not there: another's, to no effect)
  const int r = lane & 15, g = lane >> 4, swz = (r >> 1) & 7;
  const uint32_t lo = 16u * (uint32_t)(g ^ swz), hi = 16u * (uint32_t)((4 + g) ^ swz);
  f32x4 acc[NB][MT];
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  auto read = [&](const unsigned char* stage, int row, dc::u32x4 (&v)[2]) __attribute__((always_inline)) {
    v[0] = *reinterpret_cast<const dc::u32x4*>(stage + row * kTileBytes + lo);
    v[1] = *reinterpret_cast<const dc::u32x4*>(stage + row * kTileBytes + hi);
  };
  // Block scales of four of the wave's steps, from step t on, of the rows of w and x that this lane's operands hold.
  struct Codes {
    int w[kBlocks ? NB : 1], x[kBlocks ? MT : 1];
  };
  auto load_codes = [&](Codes& c, int t) __attribute__((always_inline)) {
    if constexpr (kBlocks) {
      const int kb = min(wave + (t + g) * W, steps - 1);
      const int left_n = (int)min((int64_t)o.n - n0, (int64_t)16 * kOut), left_m = (int)min((int64_t)o.m - m0, (int64_t)8 * XB);
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const uint8_t* from = o.b_codes + kb * o.b_codes_pitch + n0;
        if constexpr (kGated) from = i < kOut ? from : o.b2_codes + kb * o.b2_codes_pitch + n0;
        c.w[i] = from[min(16 * (i % kOut) + r, left_n - 1)];
      }
#pragma unroll
      for (int j = 0; j < MT; ++j) c.x[j] = (o.a_codes + kb * o.a_codes_pitch + m0)[min(16 * j + r, left_m - 1)];
    }
  };
  // Those of step t, in every lane.
  auto hand_over = [&](const Codes& c, int t) __attribute__((always_inline)) {
    Codes now;
    if constexpr (kBlocks) {
      const int from = 4 * (16 * (t & 3) + r);
#pragma unroll
      for (int i = 0; i < NB; ++i) now.w[i] = __builtin_amdgcn_ds_bpermute(from, c.w[i]);
#pragma unroll
      for (int j = 0; j < MT; ++j) now.x[j] = __builtin_amdgcn_ds_bpermute(from, c.x[j]);
    }
    return now;
  };
  auto add = [&](const unsigned char* stage, const Codes& c) __attribute__((always_inline)) {
    dc::u32x4 wv[NB][2], xv[MT][2];
#pragma unroll
    for (int i = 0; i < NB; ++i) read(stage, 16 * i + r, wv[i]);
#pragma unroll
    for (int j = 0; j < MT; ++j) read(stage + 2 * NB * 1024, 16 * j + (16 * j + 8 < 8 * XB ? r : r & 7), xv[j]);
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        if constexpr (kFp8) {
          const i32x8 a = __builtin_bit_cast(i32x8, __builtin_shufflevector(wv[i][0], wv[i][1], 0, 1, 2, 3, 4, 5, 6, 7));
          const i32x8 b = __builtin_bit_cast(i32x8, __builtin_shufflevector(xv[j][0], xv[j][1], 0, 1, 2, 3, 4, 5, 6, 7));
          if constexpr (kBlocks)
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc[i][j], 0, 0, 0, c.w[i], 0, c.x[j]);
          else
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc[i][j], 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);
        } else {
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const dc::u32x4 a = wv[i][p], b = xv[j][p];
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b),
                                                               acc[i][j], 0, 0, 0);
          }
        }
      }
  };
  const int count = steps > wave ? (steps - wave + W - 1) / W : 0;  // this wave's steps: wave, wave + W, ...
  Codes four, ahead;
  load_codes(four, 0);
#pragma unroll
  for (int d = 0; d < D - 1; ++d)
    if (d < count) load(own + d * kStage, wave + d * W);
  // The results this thread will finish, and what they take from memory, asked for before the loop: acc[i][j][v] of lane
  // 16·g + r is output 16·i + 4·g + v of row 16·j + r of x.
  constexpr int kItems = (kOut * MT + W - 1) / W;
  typedef std::conditional_t<kGated, GatedColumns<4>, Columns<4>> ItemColumns;
  ItemColumns cols[kItems];
  Results<4> out[kItems];
  bool mine[kItems];
#pragma unroll
  for (int q = 0; q < kItems; ++q) {
    const int t = threadIdx.x + q * 64 * W, b = t >> 6, l = t & 63;
    const int64_t i = m0 + 16 * (b % MT) + (l & 15), j = n0 + 16 * (b / MT) + 4 * (l >> 4);
    mine[q] = b < kOut * MT && 16 * (b % MT) + (l & 15) < 8 * XB && i < o.m && j < o.n;
    if (mine[q]) {
      cols[q].read(ep, j, o.n);
      if constexpr (!kGated) out[q].read(ep, cols[q], i);
      else if (ep.a_scales) out[q].scale = ep.a_scales[i];
    }
  }
  int slot = 0;
  auto turn = [&](int t) __attribute__((always_inline)) {
    const int next = t + D - 1;
    Codes now;
    if (next < count) {
      // (its stage was read in the turn before; those reads have returned, as their products have been issued. The wait leaves scales out of
      // its count: wherever they stand among the loads, no fewer have landed.)
      load(own + (slot == 0 ? D - 1 : slot - 1) * kStage, wave + next * W);
      now = hand_over(four, t);
      wait_loads<(D - 1) * kLoads>();
    } else {
      now = hand_over(four, t);
      wait_loads<0>();
    }
    __builtin_amdgcn_sched_barrier(0);
    add(own + slot * kStage, now);
    __builtin_amdgcn_sched_barrier(0);
    slot = slot + 1 == D ? 0 : slot + 1;
  };
  if constexpr (kBlocks) {
    // (four turns at a time, with no way round any of them into the next four: else the compiler cannot tell how many loads have gone out since the
    // scales', and waits for all before it takes those)
    for (int t = 0; t < count; t += 4) {
      load_codes(ahead, t + 4);
      turn(t);
      if (t + 1 >= count) break;
      turn(t + 1);
      if (t + 2 >= count) break;
      turn(t + 2);
      if (t + 3 >= count) break;
      turn(t + 3);
      four = ahead;
    }
  } else {
    for (int t = 0; t < count; ++t) turn(t);
  }
  __syncthreads();
  f32x4* sums = reinterpret_cast<f32x4*>(ring);
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) sums[(wave * NB * MT + i * MT + j) * 64 + lane] = acc[i][j];
  __syncthreads();
#pragma unroll
  for (int q = 0; q < kItems; ++q) {
    const int t = threadIdx.x + q * 64 * W, b = t >> 6, l = t & 63;
    if (!mine[q]) continue;
    f32x4 v = sums[b * 64 + l];
#pragma unroll
    for (int w = 1; w < W; ++w) v += sums[(w * NB * MT + b) * 64 + l];
    float z[4] = {v.x, v.y, v.z, v.w};
    const int64_t i = m0 + 16 * (b % MT) + (l & 15);
    if constexpr (kGated) {
      f32x4 u = sums[(kOut * MT + b) * 64 + l];
#pragma unroll
      for (int w = 1; w < W; ++w) u += sums[(w * NB * MT + kOut * MT + b) * 64 + l];
      float up[4] = {u.x, u.y, u.z, u.w};
      gated_finish(ep, cols[q], i, out[q].scale, z, up);
    } else {
      out[q].finish(ep, cols[q], i, z);
    }
  }
}

// ---- copies ------------------------------------------------------------------------------------------------
// Rows of `bytes` bytes at any alignment to rows of `to_pitch` (a multiple of 16), padded with zeros. Bound by launch and latency
// at ordinary sizes: 1537 and 2049 rows of 2046 bytes, both operands in one launch, 5.5-8 us, a third of the product's call.
struct PackJob {
  const unsigned char* from;
  unsigned char* to;
  int64_t rows, bytes, from_pitch, to_pitch;
};
struct PackArgs {
  PackJob job[3];
};
constexpr int64_t kPackBytes = 4096;  // of a row that a wave takes, all asked for at once
// Workgroup `block` of `blocks`, of four waves.
__device__ inline void pack_rows(const PackJob& a, int64_t block, int64_t blocks) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t across = (a.to_pitch + kPackBytes - 1) / kPackBytes, total = a.rows * across;
  for (int64_t t = block * 4 + wave; t < total; t += blocks * 4) {
    const int64_t row = total <= UINT32_MAX ? (int64_t)((uint32_t)t / (uint32_t)across) : t / across;
    const unsigned char* from = a.from + row * a.from_pitch;
    unsigned char* to = a.to + row * a.to_pitch;
    const int64_t first = (t - row * across) * kPackBytes + 16 * lane;
    dc::u32x4 w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = load_piece(from + first + 1024 * i, a.bytes - first - 1024 * i, a.bytes);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (first + 1024 * i < a.to_pitch) *reinterpret_cast<dc::u32x4*>(to + first + 1024 * i) = w[i];
  }
}
__global__ __launch_bounds__(256) void pack_kernel(PackArgs args) { pack_rows(args.job[blockIdx.y], blockIdx.x, gridDim.x); }

// The results from the sums over `count` parts of c: a lane takes eight neighbouring columns, and adds the parts in order.
// (The parts have just been written, and come from the caches.)
struct JoinJob {
  const float* parts;  // [count][m][pitch]
  int64_t m, n, pitch;
  int32_t count;
  Epilogue ep;
};
struct JoinArgs {
  JoinJob job[3];
};
__global__ __launch_bounds__(256) void join_kernel(JoinArgs args) {
  const JoinJob& a = args.job[blockIdx.y];
  const int64_t across = (a.n + 7) / 8, total = a.m * across, step = (int64_t)gridDim.x * 256;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += step) {
    const int64_t i = total <= UINT32_MAX ? (int64_t)((uint32_t)t / (uint32_t)across) : t / across, j = 8 * (t - i * across);
    Columns<8> cols;
    Results<8> out;
    cols.read(a.ep, j, a.n);
    out.read(a.ep, cols, i);
    const f32x4* q = reinterpret_cast<const f32x4*>(a.parts + i * a.pitch + j);
    f32x4 lo = q[0], hi = q[1];
#pragma unroll 4
    for (int32_t c = 1; c < a.count; ++c) {
      const f32x4* r = reinterpret_cast<const f32x4*>(a.parts + (c * a.m + i) * a.pitch + j);
      lo += r[0];
      hi += r[1];
    }
    float z[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    out.finish(a.ep, cols, i, z);
  }
}

// ---- host ------------------------------------------------------------------------------------------------
int64_t padded(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// Scratch of one call: pieces of ctx->partials, each at a multiple of 256 bytes.
struct Scratch {
  size_t bytes = 0;
  size_t take(int64_t n) {
    const size_t at = bytes;
    bytes += (size_t)padded(n, 256);
    return at;
  }
};

// A product's tile and the parts that c is split into, whose sums stand in scratch.
struct ProductPlan {
  dc::LinearTile tile;
  dc::LinearSplit split;
  size_t at = 0;
  ProductPlan(Scratch& s, const dc::LinearSize& size, dc::LinearTile t, const dc::LinearSplit& c) : tile(t), split(c) {
    if (split.parts > 1) at = s.take(split.parts * size.m * padded(size.n, 8) * (int64_t)sizeof(float));
  }
};

// One product to launch: all of it, its results in scratch where c is split.
template <class O, class E>
struct ProductOf {
  O o;
  E ep;
  ProductPlan plan;
  float* parts(dc_hip_ctx* ctx) const { return reinterpret_cast<float*>(static_cast<unsigned char*>(ctx->partials) + plan.at); }
  int64_t pitch() const { return padded(o.n, 8); }  // of those
};

typedef ProductOf<Operands, Epilogue> Product;

constexpr int64_t kLaunchItems = int64_t(1) << 32;  // a launch has fewer work items

// The workgroups of `jobs`' products, `total` of them, and those that add columns' parts, in as many launches as their work items need.
template <int TM, int TN, int WM, int WN, int KS, bool kFp8, bool kRowsC, bool kGated, bool kBlocks>
int32_t launch_jobs(dc_hip_ctx* ctx, typename ProductTypes<kRowsC, kGated, kBlocks>::Jobs& jobs, int64_t total) {
  constexpr int kThr = 64 * WM * WN * KS;
  total += (jobs.columns.n + kThr / 16 - 1) / (kThr / 16);
  for (int64_t base = 0; base < total;) {
    const int64_t count = std::min(total - base, kLaunchItems / kThr - 1);
    jobs.base = (int32_t)base;
    product_kernel<TM, TN, WM, WN, KS, kFp8, kRowsC, kGated, kBlocks><<<(unsigned)count, kThr, 0, ctx->stream>>>(jobs);
    DC_RETURN_IF(dc::last_launch_status());
    base += count;
  }
  return DC_OK;
}

// The parts of those (at most three) products that have them, added in one launch.
int32_t join(dc_hip_ctx* ctx, const Product* const* products, int count) {
  JoinArgs args{};
  int jobs = 0;
  int64_t most = 0;
  for (int i = 0; i < count; ++i) {
    if (!products[i] || products[i]->plan.split.parts == 1) continue;
    const Product& p = *products[i];
    args.job[jobs++] = JoinJob{p.parts(ctx), p.o.m, p.o.n, p.pitch(), (int32_t)p.plan.split.parts, p.ep};
    most = std::max(most, (p.o.m * (p.pitch() / 8) + 255) / 256);
  }
  if (jobs == 0) return DC_OK;
  join_kernel<<<dim3((unsigned)std::min<int64_t>(most, 1 << 16), (unsigned)jobs), 256, 0, ctx->stream>>>(args);
  return dc::last_launch_status();
}

bool aligned_to(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
// An operand as the direct-to-LDS loads take it: 16-byte aligned rows of whole 16-byte pieces, with a pitch that keeps
// a tile's rows in range; else a copy that is.
struct Rows {
  const unsigned char* p;
  int64_t pitch, rows, bytes;
  bool copied = false;
  size_t at = 0;
  void plan(Scratch& s) {
    copied = !aligned_to(p, 16) || pitch % 16 != 0 || bytes % 16 != 0 || pitch > dc::kLinearPitch;
    if (copied) at = s.take(rows * padded(bytes, 16));
  }
  int64_t width() const { return copied ? padded(bytes, 16) : pitch; }  // the pitch it will have
};

// The copies of those of the (at most three) operands that have to be laid out, which are taken to be in place from here on.
struct Copies {
  PackArgs args{};
  int jobs = 0;
  int64_t groups = 0;  // of workgroups for the larger
};
Copies lay_out(dc_hip_ctx* ctx, Rows* a, Rows* b, Rows* d = nullptr) {
  Copies c;
  for (Rows* r : {a, b, d}) {
    if (!r || !r->copied) continue;
    unsigned char* to = static_cast<unsigned char*>(ctx->partials) + r->at;
    c.args.job[c.jobs++] = PackJob{r->p, to, r->rows, r->bytes, r->pitch, r->width()};
    c.groups = std::max(c.groups, (r->rows * ((r->width() + kPackBytes - 1) / kPackBytes) + 3) / 4);
    r->p = to;
    r->pitch = r->width();
  }
  c.groups = std::min<int64_t>(c.groups, 65536);
  return c;
}
int32_t copy_rows(dc_hip_ctx* ctx, const Copies& c) {
  if (c.jobs == 0) return DC_OK;
  pack_kernel<<<dim3((unsigned)c.groups, (unsigned)c.jobs), 256, 0, ctx->stream>>>(c.args);
  return dc::last_launch_status();
}

int32_t check_rows(const void* p, int64_t size, int64_t stride, int64_t rows, int64_t cols) {
  if (!p) return DC_ERR_INVALID_ARGUMENT;
  if (!aligned_to(p, (uintptr_t)size)) return DC_ERR_MISALIGNED;
  return rows > 1 && stride < cols ? DC_ERR_DIMENSION : DC_OK;
}

// Block scales of rows of k: bytes, at any alignment.
int32_t check_codes(const void* p, int64_t stride, int64_t rows, int64_t k) {
  if (!p) return DC_ERR_INVALID_ARGUMENT;
  return k > DC_SCALE_BLOCK && stride < rows ? DC_ERR_DIMENSION : DC_OK;
}

// Bytes from row to row. (The stride of a single row says nothing, and is not looked at.)
int64_t pitch_of(int64_t stride, int64_t rows, int64_t cols, int64_t size) { return (rows > 1 ? stride : cols) * size; }

int32_t check_dims(int64_t m, int64_t n, int64_t k, int32_t act) {
  if (m < 0 || n < 0 || k < 0 || act < DC_ACT_NONE || act > DC_ACT_SILU) return DC_ERR_INVALID_ARGUMENT;
  if (m > INT32_MAX / 2) return DC_ERR_INVALID_ARGUMENT;
  return n > dc::kLinearWidth || k > dc::kLinearWidth ? DC_ERR_UNSUPPORTED : DC_OK;
}

}  // namespace
