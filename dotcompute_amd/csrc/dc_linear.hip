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

// 16 bytes a lane to 1 KiB of LDS, from `voff` (the lane's, kPast for zeros) + `soff` bytes past `base`.
__device__ inline void load_block(const unsigned char* base, unsigned char* to, uint32_t voff, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(dc::range_rsrc(base, kRange), (dc::lds_ptr_t)to, 16, voff, soff, 0, 0);
}

// The products of one launch. Workgroups take the first's tiles, part of c by part, then the second's: the two
// gradients of a layer seldom fill the chip by themselves, and a launch saved is 3-5 us.
struct Job {
  Operands o;
  Epilogue ep;
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
template <int N>
struct Jobs {
  Job job[N];
  int32_t first;   // workgroups of the first
  int32_t second;  // of both
  int32_t base;    // of the launches before this one
  ColumnParts columns;
};
template <bool kRowsC>
constexpr int kJobs = kRowsC ? 2 : 1;

// out[c] = parts[0][c] + ... for kThr / 16 columns a workgroup: 16 threads a column add every 16th part each, then those
// sums in order.
template <int kThr>
__device__ inline void add_parts(const ColumnParts& a, int block, float* lds) {
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
  a.out[c] = v;
}

template <int TM, int TN, int WM, int WN, int KS, bool kFp8, bool kRowsC>
__global__ __launch_bounds__(64 * WM * WN * KS, (WM * WN == 8 ? 1 : 2)) void product_kernel(Jobs<kJobs<kRowsC>> jobs) {
  static_assert(!(kFp8 && kRowsC), "8-bit operands run along c");
  constexpr int kWaves = WM * WN;
  constexpr int kMT = TM / WM / 32, kNT = TN / WN / 32;
  constexpr int kABlocks = TM / 8 / kWaves, kBBlocks = TN / 8 / kWaves;  // 1 KiB blocks of a wave and tile
  constexpr int kSteps = kFp8 ? 2 : 4;                                   // instructions along c of a tile
  using Smem = TileSmem<TM, TN>;
  __shared__ __align__(16) Smem sms[KS];
  int block = jobs.base + (int)blockIdx.x;
  if constexpr (kRowsC)
    if (block >= jobs.second) return add_parts<64 * kWaves * KS>(jobs.columns, block - jobs.second, reinterpret_cast<float*>(sms));
  const bool second = kRowsC && block >= jobs.first;
  if (second) block -= jobs.first;
  const Job& job = jobs.job[second ? kJobs<kRowsC> - 1 : 0];
  const Operands& o = job.o;
  const Epilogue& ep = job.ep;
  const int tiles = job.tiles_m * job.tiles_n, part = job.parts > 1 ? block / tiles : 0, turns = job.turns;
  const dc::TileCoord tc = dc::map_tile(block - part * tiles, job.tiles_m, job.tiles_n);
  const int m0 = tc.tm * TM, n0 = tc.tn * TN;
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
  uint32_t avoff[kABlocks], bvoff[kRowsC ? 1 : kBBlocks];
#pragma unroll
  for (int i = 0; i < kABlocks; ++i)
    avoff[i] = (uint32_t)min(8 * (i * kWaves + wave) + lrow, o.m - 1 - m0) * (uint32_t)o.a_pitch + (uint32_t)piece;
  if constexpr (kRowsC) {
    bvoff[0] = (uint32_t)brow * (uint32_t)o.b_pitch + (uint32_t)(2 * min(8 * bchunk, o.b_cols - 8 - n0));
  } else {
#pragma unroll
    for (int i = 0; i < kBBlocks; ++i)
      bvoff[i] = (uint32_t)min(8 * (i * kWaves + wave) + lrow, o.n - 1 - n0) * (uint32_t)o.b_pitch + (uint32_t)piece;
  }
  const unsigned char* abase = o.a + (int64_t)m0 * o.a_pitch;
  const unsigned char* bbase = kRowsC ? o.b + (int64_t)n0 * 2 : o.b + (int64_t)n0 * o.b_pitch;
  auto load_tile = [&](auto BUF, int KT) __attribute__((always_inline)) {
    constexpr int kBuf = decltype(BUF)::value;
    const int t = (kt_first + KT) * KS + group;
    const int at = t * kTileBytes;  // bytes into A's rows (past the last: every load is past the range)
    const int left = c_end - at;
#pragma unroll
    for (int i = 0; i < kABlocks; ++i)
      load_block(abase + at, sm.a[kBuf] + (i * kWaves + wave) * 1024, piece < left ? avoff[i] : kPast, 0);
    if constexpr (kRowsC) {
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
        load_block(bbase + at, sm.b[kBuf] + (i * kWaves + wave) * 1024, piece < left ? bvoff[i] : kPast, 0);
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
  auto mfmas = [&](const F* a, const F* b) __attribute__((always_inline)) {
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
        if constexpr (kFp8)
          acc[mt][nt] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b[nt].v, a[mt].v, acc[mt][nt], 0, 0, 0, 0x7f7f7f7f, 0,
                                                                       0x7f7f7f7f);
        else
          acc[mt][nt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(b[nt].v, a[mt].v, acc[mt][nt], 0, 0, 0);
      }
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

  // Tile kt in buffer kt & 1: its steps run their products with the next step's reads between them; before the last
  // step comes the tile's one barrier, which also waits for tile kt+1's loads, issued a tile earlier; then tile
  // kt+2's loads go out into the buffer that tile kt is done with.
  F fa[2][kMT], fb[2][kRowsC ? kSteps : 1][kNT];
  constexpr std::integral_constant<int, 0> kBuf0{};
  constexpr std::integral_constant<int, 1> kBuf1{};
  load_tile(kBuf0, 0);
  dc::dma_barrier();
  if constexpr (kRowsC) read_b_tile(kBuf0, fb[0]);
  else read_b(kBuf0, 0, fb[0][0]);
  read_a(kBuf0, 0, fa[0]);
  __builtin_amdgcn_sched_barrier(0);
  if (kAlways || kt_count > 1) load_tile(kBuf1, 1);
  // (a macro, so that the fragment arrays stay plain registers)
#define DC_TILE(BUF, KT)                                                                            \
  {                                                                                                 \
    _Pragma("unroll") for (int step = 0; step + 1 < kSteps; ++step) {                               \
      const int cur = step & 1;                                                                     \
      __builtin_amdgcn_sched_barrier(0);                                                            \
      read_a(kBuf##BUF, step + 1, fa[cur ^ 1]);                                                     \
      if constexpr (!kRowsC) read_b(kBuf##BUF, step + 1, fb[cur ^ 1][0]);                           \
      mfmas(fa[cur], kRowsC ? fb[BUF][kRowsC ? step : 0] : fb[cur][0]);                             \
      interleave();                                                                                 \
      __builtin_amdgcn_sched_barrier(0);                                                            \
    }                                                                                               \
    dc::dma_barrier();                                                                              \
    if constexpr (kRowsC) read_b_tile(kBuf##BUF##Other, fb[1 - (BUF)]);                             \
    __builtin_amdgcn_sched_barrier(0);                                                              \
    if (kAlways || (KT) + 2 < kt_count) load_tile(kBuf##BUF, (KT) + 2);                             \
    __builtin_amdgcn_sched_barrier(0);                                                              \
    read_a(kBuf##BUF##Other, 0, fa[0]);                                                             \
    if constexpr (!kRowsC) read_b(kBuf##BUF##Other, 0, fb[0][0]);                                   \
    mfmas(fa[1], kRowsC ? fb[BUF][kRowsC ? kSteps - 1 : 0] : fb[1][0]);                             \
    interleave();                                                                                   \
    __builtin_amdgcn_sched_barrier(0);                                                              \
  }
  constexpr auto kBuf0Other = kBuf1;
  constexpr auto kBuf1Other = kBuf0;
  __builtin_assume(kt_count > 0);
  int kt = 0;
  do {
    DC_TILE(0, kt);
    if (kt + 1 < kt_count) DC_TILE(1, kt + 1);
    kt += 2;
  } while (kt < kt_count);
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
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x4 v = {acc[mt][nt][4 * q], acc[mt][nt][4 * q + 1], acc[mt][nt][4 * q + 2], acc[mt][nt][4 * q + 3]};
          *reinterpret_cast<f32x4*>(own + r * kPitch + 32 * nt + 8 * q + 4 * h) = v;
        }
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

template <bool kFp8, int XB, int NB, int W, int D>
__global__ __launch_bounds__(64 * W) void few_rows_kernel(Operands o, Epilogue ep) {
  constexpr int MT = (XB + 1) / 2, kStage = (2 * NB + XB) * 1024, kLoads = 2 * NB + XB;
  static_assert((D - 1) * kLoads < 64 && W * D * kStage <= 160 * 1024 && W * NB * MT * 1024 <= W * D * kStage);
  __shared__ __align__(16) unsigned char ring[W * D * kStage];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  unsigned char* own = ring + wave * D * kStage;
  const int64_t n0 = (int64_t)blockIdx.x * 16 * NB, m0 = (int64_t)blockIdx.y * 8 * XB;
  // load side: lane -> row lane / 8 of a block of 8, slot lane % 8, which holds the piece of the swizzle
  const int piece = 16 * ((lane & 7) ^ (lane >> 4));  // of even blocks; of odd ones 64 bytes away
  uint32_t woff[2 * NB], xoff[XB];
#pragma unroll
  for (int i = 0; i < 2 * NB; ++i) {
    const int row = 8 * i + (lane >> 3);
    woff[i] = n0 + row < o.n ? (uint32_t)row * (uint32_t)o.b_pitch + (uint32_t)(piece ^ (64 * (i & 1))) : kPast;
  }
#pragma unroll
  for (int i = 0; i < XB; ++i) {
    const int row = 8 * i + (lane >> 3);
    xoff[i] = m0 + row < o.m ? (uint32_t)row * (uint32_t)o.a_pitch + (uint32_t)(piece ^ (64 * (i & 1))) : kPast;
  }
  const unsigned char *wbase = o.b + n0 * o.b_pitch, *xbase = o.a + m0 * o.a_pitch;
  const int steps = (o.c_bytes + kTileBytes - 1) / kTileBytes;
  auto load = [&](unsigned char* stage, int s) __attribute__((always_inline)) {
    const int64_t at = (int64_t)s * kTileBytes;
    const int left = o.c_bytes - s * kTileBytes;
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i)
      load_block(wbase + at, stage + i * 1024, (piece ^ (64 * (i & 1))) < left ? woff[i] : kPast, 0);
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
  auto add = [&](const unsigned char* stage) __attribute__((always_inline)) {
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
#pragma unroll
  for (int d = 0; d < D - 1; ++d)
    if (d < count) load(own + d * kStage, wave + d * W);
  // The results this thread will finish, and what they take from memory, asked for before the loop: acc[i][j][v] of lane
  // 16·g + r is output 16·i + 4·g + v of row 16·j + r of x.
  constexpr int kItems = (NB * MT + W - 1) / W;
  Columns<4> cols[kItems];
  Results<4> out[kItems];
  bool mine[kItems];
#pragma unroll
  for (int q = 0; q < kItems; ++q) {
    const int t = threadIdx.x + q * 64 * W, b = t >> 6, l = t & 63;
    const int64_t i = m0 + 16 * (b % MT) + (l & 15), j = n0 + 16 * (b / MT) + 4 * (l >> 4);
    mine[q] = b < NB * MT && 16 * (b % MT) + (l & 15) < 8 * XB && i < o.m && j < o.n;
    if (mine[q]) {
      cols[q].read(ep, j, o.n);
      out[q].read(ep, cols[q], i);
    }
  }
  int slot = 0;
  for (int t = 0; t < count; ++t) {
    const int next = t + D - 1;
    if (next < count) {
      // (its stage was read in the turn before; those reads have returned, as their products have been issued)
      load(own + (slot == 0 ? D - 1 : slot - 1) * kStage, wave + next * W);
      wait_loads<(D - 1) * kLoads>();
    } else {
      wait_loads<0>();
    }
    __builtin_amdgcn_sched_barrier(0);
    add(own + slot * kStage);
    __builtin_amdgcn_sched_barrier(0);
    slot = slot + 1 == D ? 0 : slot + 1;
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
    out[q].finish(ep, cols[q], m0 + 16 * (b % MT) + (l & 15), z);
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
  PackJob job[2];
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

// The results from the sums over `count` parts of c: a lane takes eight neighbouring columns, and adds the parts in order.
// (The parts have just been written, and come from the caches.)
struct JoinJob {
  const float* parts;  // [count][m][pitch]
  int64_t m, n, pitch;
  int32_t count;
  Epilogue ep;
};
struct JoinArgs {
  JoinJob job[2];
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
struct Product {
  Operands o;
  Epilogue ep;
  ProductPlan plan;
  float* parts(dc_hip_ctx* ctx) const { return reinterpret_cast<float*>(static_cast<unsigned char*>(ctx->partials) + plan.at); }
  int64_t pitch() const { return padded(o.n, 8); }  // of those
};

constexpr int64_t kLaunchItems = int64_t(1) << 32;  // a launch has fewer work items

template <int TM, int TN, int WM, int WN, int KS, bool kFp8, bool kRowsC>
int32_t launch_products(dc_hip_ctx* ctx, const Product* const (&p)[kJobs<kRowsC>], const ColumnParts& columns) {
  constexpr int kThr = 64 * WM * WN * KS;
  Jobs<kJobs<kRowsC>> jobs{};
  int64_t total = 0;
  for (int i = 0; i < kJobs<kRowsC>; ++i) {
    if (i == 1) jobs.first = (int32_t)total;
    if (!p[i]) continue;
    Job& j = jobs.job[i];
    j.o = p[i]->o, j.ep = p[i]->ep;
    j.tiles_m = (j.o.m + TM - 1) / TM, j.tiles_n = (j.o.n + TN - 1) / TN;
    j.parts = (int32_t)p[i]->plan.split.parts, j.turns = (int32_t)p[i]->plan.split.turns;
    if (j.parts > 1) {  // the sums alone
      j.ep = Epilogue{};
      j.ep.y = p[i]->parts(ctx), j.ep.y_stride = p[i]->pitch(), j.ep.y_f32 = 1, j.ep.part_stride = j.o.m * p[i]->pitch();
    }
    total += (int64_t)j.tiles_m * j.tiles_n * j.parts;
    if (total > INT32_MAX / 2) return DC_ERR_UNSUPPORTED;
  }
  jobs.second = (int32_t)total;
  jobs.columns = columns;
  total += (columns.n + kThr / 16 - 1) / (kThr / 16);
  for (int64_t base = 0; base < total;) {
    const int64_t count = std::min(total - base, kLaunchItems / kThr - 1);
    jobs.base = (int32_t)base;
    product_kernel<TM, TN, WM, WN, KS, kFp8, kRowsC><<<(unsigned)count, kThr, 0, ctx->stream>>>(jobs);
    DC_RETURN_IF(dc::last_launch_status());
    base += count;
  }
  return DC_OK;
}

// Adds the parts of those (at most two) products that have them, in one launch.
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
  few_rows_kernel<kFp8, XB, NB, W, kStages><<<grid, 64 * W, 0, ctx->stream>>>(o, ep);
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

// The copies of those of the (at most two) operands that have to be laid out, which are taken to be in place from here on.
struct Copies {
  PackArgs args{};
  int jobs = 0;
  int64_t groups = 0;  // of workgroups for the larger
};
Copies lay_out(dc_hip_ctx* ctx, Rows* a, Rows* b) {
  Copies c;
  for (Rows* r : {a, b}) {
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

// Bytes from row to row. (The stride of a single row says nothing, and is not looked at.)
int64_t pitch_of(int64_t stride, int64_t rows, int64_t cols, int64_t size) { return (rows > 1 ? stride : cols) * size; }

int32_t check_dims(int64_t m, int64_t n, int64_t k, int32_t act) {
  if (m < 0 || n < 0 || k < 0 || act < DC_ACT_NONE || act > DC_ACT_SILU) return DC_ERR_INVALID_ARGUMENT;
  if (m > INT32_MAX / 2) return DC_ERR_INVALID_ARGUMENT;
  return n > dc::kLinearWidth || k > dc::kLinearWidth ? DC_ERR_UNSUPPORTED : DC_OK;
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
