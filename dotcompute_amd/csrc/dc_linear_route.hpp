// dc_linear_route.hpp — which kernel of dc_linear.hip takes a shape: pure functions of the sizes and the number of
// CUs, checked on the CPU by tests/cpp/feed_forward_tests.cpp.
#pragma once

#include <cstdint>
#include <initializer_list>

namespace dc {

// Bytes that a direct-to-LDS load can be away from its tile's first, and the pitch with which the rows of the smallest
// tiles stay below that; rows are at most kLinearWidth elements.
constexpr int32_t kLinearRange = INT32_MAX;
constexpr int64_t kLinearPitch = (int64_t(1) << 25) - 16;
constexpr int64_t kLinearWidth = int64_t(1) << 23;
constexpr int64_t kGatedWidth = kLinearWidth / 2;  // outputs of a gated layer, whose gradients run along those of both projections
static_assert(64 * kLinearPitch < kLinearRange && 2 * kLinearWidth <= kLinearPitch);

// Tiles, square, and groups of waves that take the steps along c in turn.
enum class LinearTile { k256, k128, k128x2, k64, k64x2, k64x4 };
constexpr LinearTile kLinearTiles[] = {LinearTile::k256, LinearTile::k128,  LinearTile::k128x2,
                                       LinearTile::k64,  LinearTile::k64x2, LinearTile::k64x4};

inline int64_t linear_tile_side(LinearTile t) {
  return t == LinearTile::k256 ? 256 : t == LinearTile::k128 || t == LinearTile::k128x2 ? 128 : 64;
}
inline int64_t linear_tile_groups(LinearTile t) {
  return t == LinearTile::k64x4 ? 4 : t == LinearTile::k128x2 || t == LinearTile::k64x2 ? 2 : 1;
}

struct LinearSize {
  int64_t m, n, c_bytes;     // results, and bytes of c
  int64_t a_pitch, b_pitch;  // bytes from row to row of the operands
};
inline int64_t linear_tiles(const LinearSize& s, LinearTile t) {
  const int64_t side = linear_tile_side(t);
  return ((s.m + side - 1) / side) * ((s.n + side - 1) / side);
}
inline bool linear_fits(const LinearSize& s, bool rows_c, LinearTile t) {
  const int64_t side = linear_tile_side(t);
  return side * s.a_pitch < kLinearRange && (rows_c || side * s.b_pitch < kLinearRange);
}

// c in `parts` of `turns` tiles a group of waves; the sums of more than one part are added by a kernel of their own.
struct LinearSplit {
  int64_t parts, turns;
};
inline LinearSplit linear_split(LinearTile tile, const LinearSize& s, int64_t parts) {
  const int64_t step = 128 * linear_tile_groups(tile), all = (s.c_bytes + step - 1) / step, turns = (all + parts - 1) / parts;
  return {(all + turns - 1) / turns, turns};
}

// The tile, and the parts of c, are those with the least time by this estimate, in us: a CU's workgroups take turns of 128 bytes of c, each
// bound by the loads of the two operands or the matrix cores, or, where few are there to cover it, by a turn's
// latency; each workgroup has its epilogue, each round of workgroups its start, and parts of c their sums' way through memory and
// the adding kernel. The numbers were fitted to the times of all tiles with 1 to 16 parts on 200 shapes (bf16, e4m3, B by
// rows of c; 64 to 16384 results a side, c 64 to 8192): what it picks takes 1.3 % more time than the best in the mean, 18 % at most,
// where rules by the number of tiles took 6 %, and 49 % at most. Measured, us, those rules / this / the best: bf16 1500×1500×6000 67.5 / 48.9 / 48.9
// (128-tiles, 3 parts), 300×1024×1024 9.2 / 6.1 / 6.1, 2048^3 23.3 / 23.5 / 23.3, 1347×3672×5288 94 / 95 / 84; by rows of c 545×3768×5632
// 66.7 / 52.1 / 52.1 (256-tiles, 4 parts), 8192×2048×8192 220 / 211 / 211; e4m3 128×4096×4096 12.1 / 9.0 / 9.0.
struct LinearCost {
  double call, groups;            // of a launch, and more for each further group of waves
  double start, more_start;       // of a round, and for each further 64-tile's worth of loads in a turn
  double end[3];                  // of a workgroup of side 64, 128, 256
  double loads[2], cores[2];      // of a turn, by 64-tile's worths: loads of 64-tiles of small operands, and else; products of bf16, e4m3
  double latency, more_latency;   // of a turn, and for each further 64-tile's worth
  double uneven[2];               // how much a CU with more workgroups than others counts, where it holds two, five
  double join, join_bytes;        // the adding kernel, and bytes of parts a us
  double side[3], group[3];       // what is left: factors for the sides 64, 128, 256, and 1, 2, 4 groups
};
constexpr LinearCost kLinearRowsA = {2.215, 0.462, 0.497, 0.254, {0.359, 3.318, 8.063}, {0.19, 0.206}, {0.045, 0.083}, 0.625, 0.183, {1.0, 0.428},
                                     6.58, 4.56e6, {1.0, 0.812, 0.963}, {1.0, 1.118, 1.167}};
constexpr LinearCost kLinearRowsC = {2.03, 0.44, 0.374, 0.0, {0.475, 1.9, 7.6}, {0.223, 0.223}, {0.048, 0.0}, 0.432, 0.197, {0.75, 0.75},
                                     3.4, 4.9e6, {1.0, 1.04, 0.93}, {1.0, 1.0, 1.0}};
constexpr int64_t kLinearSmall = int64_t(8) << 20;  // bytes of both operands, most of which an XCD's L2 (4 MiB) holds
struct LinearKind {
  bool rows_c, fp8;
};
inline const LinearCost& linear_cost(LinearKind kind) { return kind.rows_c ? kLinearRowsC : kLinearRowsA; }
constexpr double kLinearHeld[3][3] = {{5, 2, 1}, {2, 1, 1}, {1, 1, 1}};  // workgroups that a CU holds: by side, and groups
inline int linear_side_index(LinearTile t) { return t == LinearTile::k256 ? 2 : t == LinearTile::k128 || t == LinearTile::k128x2 ? 1 : 0; }
inline int linear_group_index(LinearTile t) {
  return t == LinearTile::k64x4 ? 2 : t == LinearTile::k128x2 || t == LinearTile::k64x2 ? 1 : 0;
}
inline double linear_up(double v) { return (double)(int64_t)(v + 0.999999); }
// `groups` workgroups of at most `turns` turns; the busiest CU has as many turns as `most` of those, the mean CU as `equal`.
// `small`: the operands are.
inline double linear_time(LinearTile t, LinearKind kind, double groups, double turns, double most, double equal, double cus, bool small) {
  const LinearCost& k = linear_cost(kind);
  const int by = linear_side_index(t), waves = linear_group_index(t);
  const double held = kLinearHeld[by][waves], g = 1 << waves, units = g * (1 << by);
  const double loads = k.loads[!(small && units == 1)] * units, cores = k.cores[kind.fp8] * units * (1 << by);
  const double turn = loads > cores ? loads : cores, latency = k.latency + k.more_latency * (units - 1);
  double each = most < 1 ? 1 : most;
  const double rounds = held > 1 ? linear_up(each / held) : each;
  if (held > 1) {
    const double u = k.uneven[held > 2];
    each = u * each + (1 - u) * (equal < 1 ? 1 : equal);
  }
  const double busy = each * turns * turn, waits = rounds * turns * latency, ends = groups / cus > each ? groups / cus : each;
  return (k.call + k.groups * (g - 1) + (k.start + k.more_start * (units - 1)) * rounds + k.end[by] * ends + (busy > waits ? busy : waits)) *
         k.side[by] * k.group[waves];
}
// (Counting the mean CU's turns alone picked 276 workgroups of 256-tiles for 256 CUs: both gradients of 5368,6400,592 217 us, now 158.)
// Turns of the busiest CU, where each holds one workgroup at a time: `gl` of `tl` turns are handed out, then `gs` of `ts`.
inline double linear_last(int64_t gl, double tl, int64_t gs, double ts, int64_t cus) {
  const int64_t over = gl % cus, room = cus - over;  // CUs with one long one more than others, and those others
  const double base = (double)(gl / cus) * tl, top = over ? base + tl : base;
  const int64_t beside = over ? (int64_t)(tl / ts) : 0, left = gs - room * beside;  // short ones beside a long one, and after all those
  if (left <= 0) return top;
  if (over && left <= room && base + (double)(beside + 1) * ts > top) return base + (double)(beside + 1) * ts;
  return top + linear_up((double)left / (double)cus) * ts;
}
inline double linear_parts_time(const LinearSize& s, LinearKind kind, int64_t parts) {
  return parts > 1 ? (double)parts * (double)s.m * (double)s.n * 8.0 / linear_cost(kind).join_bytes : 0.0;
}
constexpr int64_t kLinearParts[] = {1, 2, 3, 4, 5, 6, 8, 11, 16};

struct LinearPlan {
  LinearTile tile;
  LinearSplit split;
  double time;
};
inline LinearPlan linear_plan(const LinearSize& s, LinearKind kind, int64_t cus) {
  LinearPlan best{LinearTile::k64, linear_split(LinearTile::k64, s, 1), 1e300};
  const bool small = s.c_bytes >= 1024 && (s.m + s.n) * s.c_bytes <= kLinearSmall;
  for (LinearTile t : kLinearTiles) {
    if (!linear_fits(s, kind.rows_c, t)) continue;
    const int64_t tiles = linear_tiles(s, t);
    for (int64_t parts : kLinearParts) {
      // (few steps are over before a second kernel starts, and parts beyond what the chip holds only move more)
      if (parts > 1 && (s.c_bytes < 1024 || s.c_bytes < 256 * parts * linear_tile_groups(t) || tiles * (parts - 1) > 4 * cus)) break;
      const LinearSplit split = linear_split(t, s, parts);
      const double groups = (double)(tiles * split.parts);
      const double equal = groups / (double)cus;
      const double time = linear_time(t, kind, groups, (double)split.turns, linear_up(equal), equal, (double)cus, small) +
                          linear_parts_time(s, kind, split.parts) + (split.parts > 1 ? linear_cost(kind).join : 0.0);
      if (time < best.time) best = {t, split, time};
    }
  }
  return best;
}

// Two products (B by rows of c) in one launch: the shorter c in parts of about the longer one's turns. (Tiles of which a CU holds one
// workgroup of many waves were the best for none of 60 pairs but one or two, as they leave the second product no room beside them.) On those
// 60 the pick takes 2.3 % more than the best in the mean. Measured, both gradients of m, n, k with silu and dbias, us apart / together:
// 2000,3000,1000 70.7 / 58.5; 2048^3 60.3 / 47.0; 8192,4096,1024 214 / 184; 500,1500,700 30.7 / 24.4; 64,4096,4096 36.2 / 29.4;
// 589,288,192 17.5 / 11.6; 6,200,72 12.6 / 8.6; 8192,8192,2048 545 / 540. Apart was never more than 3 % faster.
struct LinearPair {
  LinearTile tile;
  LinearSplit a, b;
  double time;
};
// `fewer` (the gradients of a gated layer, where b is both weights'): the shorter c in one part less is tried too, which leaves its workgroups longer than the longer
// one's. Both gradients of 2000,2504,1000 92 us, with it 81 (256-tiles, 3 and 1 parts).
inline LinearPair linear_plan_of_two(const LinearSize& a, const LinearSize& b, int64_t cus, bool fewer = false) {
  const bool longer = a.c_bytes >= b.c_bytes;
  const LinearSize &l = longer ? a : b, &s = longer ? b : a;
  const LinearKind kind{true, false};
  LinearPair best{LinearTile::k64, {1, 1}, {1, 1}, 1e300};
  for (LinearTile t : {LinearTile::k256, LinearTile::k128, LinearTile::k64, LinearTile::k64x2}) {
    if (!linear_fits(l, true, t) || !linear_fits(s, true, t)) continue;
    const int64_t tl = linear_tiles(l, t), ts = linear_tiles(s, t), all = linear_split(t, s, 1).turns;
    for (int64_t parts : kLinearParts) {
      if (parts > 1 && (l.c_bytes < 1024 || l.c_bytes < 256 * parts * linear_tile_groups(t) || tl * (parts - 1) > 4 * cus)) break;
      const LinearSplit sl = linear_split(t, l, parts);
      const int64_t most_parts = (all + sl.turns - 1) / sl.turns;
      for (int64_t short_parts = most_parts; short_parts >= 1 && short_parts >= most_parts - (fewer ? 1 : 0); --short_parts) {
        const LinearSplit ss = linear_split(t, s, short_parts);
        const int64_t gl = tl * sl.parts, gs = ts * ss.parts;
        const double el = (double)sl.turns, es = (double)ss.turns, turns = el > es ? el : es;
        const double equal = ((double)gl * el + (double)gs * es) / turns / (double)cus;
        const bool one = kLinearHeld[linear_side_index(t)][linear_group_index(t)] == 1;
        const double most = !one ? linear_up(equal) : (el >= es ? linear_last(gl, el, gs, es, cus) : linear_last(gs, es, gl, el, cus)) / turns;
        const double time = linear_time(t, kind, (double)(gl + gs), turns, most, equal, (double)cus, false) +
                            linear_parts_time(l, kind, sl.parts) + linear_parts_time(s, kind, ss.parts) +
                            (sl.parts > 1 || ss.parts > 1 ? kLinearRowsC.join : 0.0);
        if (time < best.time) best = longer ? LinearPair{t, sl, ss, time} : LinearPair{t, ss, sl, time};
      }
    }
  }
  return best;
}

// Few rows of x: kernels whose workgroups take 64 of them and 16 outputs, and read w once for every 64 rows. Measured in bf16, us (few rows /
// tiles): 32×16384×2048 13.3 / 13.8, 64×4096×4096 10.5 / 17.9, 64×6144×4096 17.1 / 18.3, 64×8192×4096 19.7 / 18.7; so up to
// kLinearFewRows always, and beyond where every 64 rows and 16 outputs still find a CU of their own, however many rows those are.
// More of those, bf16 and e4m3 (few rows / tiles): 100×2048×2048 6.4 / 12.6, 4.5 / 6.6; 300×300×2048 6.6 / 11.8, 4.5 / 6.9; 512×512×1024
// 4.5 / 6.4, 3.9 / 5.3; 512×512×8192 16.5 / 19.6, 10.5 / 14.8; 1024×256×4096 13.0 / 14.6, 8.1 / 14.0. It loses where outputs are fewer than a
// tile's and sums long, as c is not split over workgroups here: 64×64×8192 11.9 / 9.7, 7.7 / 9.1; 300×64×8000 15.5 / 11.0, 11.0 /
// 9.5; 4096×64×1024 7.7 / 6.2, 5.7 / 5.3; 4096×64×4096 21.0 / 14.6, 18.8 / 14.1.
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

// Workgroups of the kernels that add the sums of parts of c: a lane takes eight neighbouring results, 256 a workgroup, which walk over what is left.
// (m below 2^30 and n up to kLinearWidth are more results than 32 bits count.)
inline int64_t linear_join_groups(int64_t m, int64_t n) {
  const int64_t groups = (m * ((n + 7) / 8) + 255) / 256;
  return groups < (1 << 16) ? groups : 1 << 16;
}

}  // namespace dc
