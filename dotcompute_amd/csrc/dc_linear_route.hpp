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
struct LinearSize {
  int64_t m, n, c_bytes;     // results, and bytes of c
  int64_t a_pitch, b_pitch;  // bytes from row to row of the operands
};
inline int64_t linear_tiles(const LinearSize& s, int64_t side) { return ((s.m + side - 1) / side) * ((s.n + side - 1) / side); }
inline bool linear_fits(const LinearSize& s, bool rows_c, int64_t side) {
  return side * s.a_pitch < kLinearRange && (rows_c || side * s.b_pitch < kLinearRange);
}
// By the numbers of tiles and the elements of c (8-bit ones count half).
inline LinearTile linear_tile_by(int64_t t256, int64_t t128, int64_t t64, int64_t k, bool fits256, bool fits128, int64_t cus) {
  const bool brief = (k <= 64 && (t256 > cus || 4 * t256 <= 3 * cus)) || (k <= 128 && t256 > 2 * cus);
  if (fits256 && 2 * t256 > cus && (t256 <= cus || 10 * t256 > 13 * cus) && !brief) return LinearTile::k256;
  if (fits128 && t128 > cus && !brief) return LinearTile::k128;
  if (fits128 && 4 * t128 > 3 * cus && k >= 1536) return LinearTile::k128x2;
  if (fits128 && 10 * t128 > 9 * cus && k >= 768) return LinearTile::k128;
  if (t64 > 2 * cus || k < 512) return LinearTile::k64;
  if (2 * t64 > cus || k < 2048) return LinearTile::k64x2;
  return LinearTile::k64x4;
}
inline LinearTile linear_tile(const LinearSize& s, bool rows_c, int64_t cus) {
  return linear_tile_by(linear_tiles(s, 256), linear_tiles(s, 128), linear_tiles(s, 64), s.c_bytes / 2, linear_fits(s, rows_c, 256),
                        linear_fits(s, rows_c, 128), cus);
}
// Two products in one launch, where their c are alike: the tile that the one with the longer c would take if it had as many
// tiles as take the time of both; 128x2, of which a CU holds one, only where the shorter ones find room beside the longer.
// Measured, both gradients of m, n, k with silu and dbias, us in two launches / in one: 2000,3000,1000 70.7 / 61.4 (128x2 71.0);
// 1024^3 26.2 / 20.7; 2048^3 61.4 / 50.5; 1000,2000,1000 38.9 / 34.4; 2048,4096,1024 68.1 / 64.7 (128 67.9); 4096,4096,1024 105 /
// 94; 8192,4096,1024 216 / 205; 8192,8192,2048 550 / 550; 200,400,512 16.8 / 13.4. Where one c is three times the other or more:
// 1000,3000,1000 49.6 / 55.4, 3000,200,2500 48.6 / 87, 64,4096,4096 32.2 / 36.6.
inline bool linear_alike(const LinearSize& a, const LinearSize& b) { return a.c_bytes <= 2 * b.c_bytes && b.c_bytes <= 2 * a.c_bytes; }
inline LinearTile linear_tile_of_two(const LinearSize& a, const LinearSize& b, bool rows_c, int64_t cus) {
  const LinearSize &l = a.c_bytes >= b.c_bytes ? a : b, &s = a.c_bytes >= b.c_bytes ? b : a;
  auto tiles = [&](int64_t side) { return linear_tiles(l, side) + (linear_tiles(s, side) * s.c_bytes + l.c_bytes - 1) / l.c_bytes; };
  auto fits = [&](int64_t side) { return linear_fits(a, rows_c, side) && linear_fits(b, rows_c, side); };
  int64_t t128 = tiles(128);
  if (t128 <= cus && 4 * t128 > 3 * cus && linear_tiles(s, 128) > (cus - linear_tiles(l, 128)) * (l.c_bytes / s.c_bytes)) t128 = cus + 1;
  return linear_tile_by(tiles(256), t128, tiles(64), l.c_bytes / 2, fits(256), fits(128), cus);
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
inline LinearSplit linear_whole(LinearTile tile, const LinearSize& s) {
  const int64_t step = 128 * linear_tile_groups(tile);
  return {1, (s.c_bytes + step - 1) / step};
}
inline LinearSplit linear_split(LinearTile tile, const LinearSize& s, int64_t cus) {
  const int64_t side = linear_tile_side(tile), tiles = linear_tiles(s, side), all = linear_whole(tile, s).turns;
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
