// dc_linear_route.hpp — which kernel of dc_linear.hip takes a shape: pure functions of the sizes and the number of
// CUs, checked on the CPU by tests/cpp/feed_forward_tests.cpp.
#pragma once

#include <cstdint>

namespace dc {

// Bytes that a direct-to-LDS load can be away from its tile's first, and the pitch with which the rows of the smallest
// tiles stay below that; rows are at most kLinearWidth elements.
constexpr int32_t kLinearRange = INT32_MAX;
constexpr int64_t kLinearPitch = (int64_t(1) << 25) - 16;
constexpr int64_t kLinearWidth = int64_t(1) << 23;
static_assert(64 * kLinearPitch < kLinearRange && 2 * kLinearWidth <= kLinearPitch);

// Tiles, square, and groups of waves that take the steps along c in turn.
enum class LinearTile { k256, k128, k128x2, k64, k64x2, k64x4 };

// By rounds of the tiles over the CUs, as dc_gemm_route.hpp's rule, measured again (results m x n, sums over c; us for
// tiles of 256 / 128 / 128x2 / 64 / 64x2 / 64x4, w by rows of c where it says so):
//   bf16: 4096x4096x1024 34.5 / 39.7 / 51.7 / 52.4 / 59.4 / 94;  5120x5120x1024 58.8 / 64.4 / 89 / 80 / 92 / 145
//   2000x3000x1000 30.5 / 21.6 / 29.4 / 27.8 / 28.7 / 41;  2048^3 44 / 25.3 / 22.7 / 25.6 / 27.4 / 38
//   2048x2048x816 25.4 / 13.3 / 13.8 / 15.2 / 16.1 / 23;  2048x2048x512 18.6 / 9.7 / 10.3 / 9.1 / 11.3 / 18
//   1537x2049x1024 27.4 / 15.2 / 14.8 / 13.8 / 17.7 / 26;  1024^3 26 / 11.7 / 11.7 / 6.9 / 6.4 / 6.5
//   rows c: 8192x2048x8192 208 / 244 / 278 / 358 / 377 / 529;  4096x1024x4096 86 / 47 / 39.9 / 49 / 52 / 73
//   2000x1000x3000 71 / 41 / 36 / 29.1 / 27.9 / 37;  3000x1000x2000 51 / 30.2 / 26.5 / 27.9 / 33.8 / 38
//   512x512x4096 83 / 34 / 29.8 / 32.6 / 24.1 / 20.2;  64x2048x8192 155 / 80 / 60 / 61 / 43.8 / 34.9
//   e4m3: 4096^3 58 / 66 / 92 / 96 / 110 / 157;  2048^3 31.6 / 15.2 / 14.6 / 13.8 / 16 / 24;  1537x2049x1024 22 / 11.2 / 11.1 / 9.0 / 11 / 19
// (Three and four stages of LDS instead of two, and tiles of 128x64, 256x128 and 128x256, were no faster on any of these but
// e4m3 2048^3, 13.5.)
inline LinearTile linear_tile(int64_t m, int64_t n, int64_t c_bytes, int64_t a_pitch, int64_t b_pitch, bool rows_c, int64_t cus) {
  auto tiles = [&](int64_t t) { return ((m + t - 1) / t) * ((n + t - 1) / t); };
  auto fits = [&](int64_t t) { return t * a_pitch < kLinearRange && (rows_c || t * b_pitch < kLinearRange); };
  const int64_t t256 = tiles(256), t128 = tiles(128), t64 = tiles(64), k = c_bytes / 2;
  const bool brief = (k <= 64 && (t256 > cus || 4 * t256 <= 3 * cus)) || (k <= 128 && t256 > 2 * cus);
  if (fits(256) && 2 * t256 > cus && (t256 <= cus || 10 * t256 > 13 * cus) && !brief) return LinearTile::k256;
  if (fits(128) && t128 > cus && !brief) return LinearTile::k128;
  if (fits(128) && 4 * t128 > 3 * cus && k >= 1536) return LinearTile::k128x2;
  if (fits(128) && 10 * t128 > 9 * cus && k >= 768) return LinearTile::k128;
  if (t64 > 2 * cus || k < 512) return LinearTile::k64;
  if (2 * t64 > cus || k < 2048) return LinearTile::k64x2;
  return LinearTile::k64x4;
}

inline int64_t linear_tile_side(LinearTile t) {
  return t == LinearTile::k256 ? 256 : t == LinearTile::k128 || t == LinearTile::k128x2 ? 128 : 64;
}
inline int64_t linear_tile_groups(LinearTile t) {
  return t == LinearTile::k64x4 ? 4 : t == LinearTile::k128x2 || t == LinearTile::k64x2 ? 2 : 1;
}

// c in `parts` of `turns` tiles a group, whose sums are added by a kernel of their own: where the tiles leave CUs idle and their
// sums are long; two workgroups a CU where they are longer still. Measured, us in one part / two workgroups a CU / four (results m x n,
// sums over c): bf16 2515x256x5120 30.2 / 21.0 / 24.9; 1024x1024x4096 22.5 / 20.3 / 26.2; 1024^3 6.4 / 13.5 / 17.4; e4m3 1024x1024x4096
// 9.7 / 16.2 / 18.4. And with many parts, before / now: 315x256x5168 27 / 11.4, 64x2048x8192 (rows c) 34.9 / 14.4.
struct LinearSplit {
  int64_t parts, turns;
};
inline LinearSplit linear_split(LinearTile tile, int64_t m, int64_t n, int64_t c_bytes, int64_t cus) {
  const int64_t side = linear_tile_side(tile), tiles = ((m + side - 1) / side) * ((n + side - 1) / side);
  const int64_t step = 128 * linear_tile_groups(tile), all = (c_bytes + step - 1) / step;
  const int64_t most = tiles > 0 ? (side == 64 && all >= 32 ? 2 : 1) * cus / tiles : 1;
  if (all < 8 || most < 2) return {1, all};
  const int64_t turns = (all + most - 1) / most < 3 ? 3 : (all + most - 1) / most;
  return {(all + turns - 1) / turns, turns};
}

// Few rows of x: kernels that read w once for up to 64 of them. Measured in bf16, us (few rows / tiles): 32×16384×2048 13.3 /
// 13.8, 64×4096×4096 10.5 / 17.9, 64×6144×4096 17.1 / 18.3, 64×8192×4096 19.7 / 18.7; so up to kLinearFewRows always, and
// beyond where every 64 rows and 16 outputs still find a CU of their own.
constexpr int64_t kLinearFewRows = 32;
inline bool linear_few_rows(int64_t m, int64_t n, int64_t cus) {
  return m <= kLinearFewRows || (m + 63) / 64 * ((n + 15) / 16) <= cus;
}
// Rows that would have to be copied for those: read as they lie, which takes a time that grows with their length, 1.5 ns a
// byte for up to 8 rows of x and 4096 outputs, where copying takes 3.5 us and 0.42 ps for each byte of w. Measured (as they
// lie / copied), us in bf16: 1×1000×333 3.7 / 7.5, 1×1024×4095 15.7 / 10.6, 1×4096×4095 15.9 / 21.0, 16×4096×1023 9.4 / 10.4,
// 16×4096×4095 27.9 / 21.3, 32×216×7977 60 / 16.8.
inline bool linear_few_rows_any(int64_t m, int64_t n, int64_t c_bytes) {
  if (m > kLinearFewRows) return false;
  const double rows = 0.3 + 0.7 * (double)((m + 7) / 8), rounds = (double)((n + 4095) / 4096);
  return 1.5 * (double)c_bytes * rows * rounds < 3500.0 + 0.42e-3 * (double)n * (double)c_bytes;
}
// 64 outputs a workgroup instead of 16, where that leaves two for a CU (8×16384×2048: 11.7 us, 12.6; 8×8192×4096: 11.7, 12.2;
// 8×4096×4096: 9.6, 7.4).
inline bool linear_wide_few_rows(int64_t m, int64_t n, int64_t cus) { return m <= kLinearFewRows && (n + 15) / 16 > 2 * cus; }

}  // namespace dc
