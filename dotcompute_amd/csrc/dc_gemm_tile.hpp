// dc_gemm_tile.hpp — what the tiled matrix products share: the order of the tiles over the chip, direct-to-LDS
// loads' pointer type and barrier, and the launch grid.
//
// Tile order: consecutive workgroups are dispatched round-robin over the 8 XCDs (each with its own
// L2). Block b is mapped to tile (b % 8) * (T / 8) + b / 8, so each XCD works on a contiguous
// range of tiles, and within it tiles are walked in groups of 8 tile-rows, column by column, so
// the blocks resident on one XCD share A row-panels and B column-panels in that XCD's L2.
#pragma once

#include <hip/hip_runtime.h>

#include "dc_gemm_route.hpp"

namespace dc {

struct TileCoord {
  int tm, tn;
};

constexpr int kTileGroupM = 8;

__device__ inline TileCoord map_tile(int b, int tiles_m, int tiles_n) {
  const int total = tiles_m * tiles_n;
  const int t = (total % 8 == 0) ? (b % 8) * (total / 8) + b / 8 : b;
  const int group = kTileGroupM * tiles_n;
  const int g = t / group;
  const int first_m = g * kTileGroupM;
  const int gm = min(tiles_m - first_m, kTileGroupM);
  const int in_g = t - g * group;
  return TileCoord{first_m + in_g % gm, in_g / gm};
}
// (gemm_grid's rows; workgroups past the last tile form that one too: an early exit here costs every launch 0.1-0.2 us)
__device__ inline TileCoord map_tile(int tiles_m, int tiles_n) {
  return map_tile(min((int)(blockIdx.x + (blockIdx.y << kGemmGridRowBits)), tiles_m * tiles_n - 1), tiles_m, tiles_n);
}

typedef __attribute__((address_space(3))) void* lds_ptr_t;

// Waits until this wave's direct-to-LDS loads have landed (vmcnt(0); expcnt and lgkmcnt left
// alone), then the workgroup barrier: after it every wave's loads issued before are visible.
__device__ inline void dma_barrier() {
  __builtin_amdgcn_s_waitcnt(0x0F70);  // gfx9 encoding: vmcnt = 0, expcnt = 7, lgkmcnt = 15
  __syncthreads();
}

inline dim3 tile_grid(int tiles_m, int tiles_n, int threads) {
  const GemmGrid g = gemm_grid((int64_t)tiles_m * tiles_n, threads);
  return dim3((unsigned)g.x, (unsigned)g.rows);
}

}  // namespace dc
