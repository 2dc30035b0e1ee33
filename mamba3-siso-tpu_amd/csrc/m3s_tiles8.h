// Rules of the products in 8 bits (m3s_matmul8.hip) that a test on the host can hold: which form sizes take,
// and the tiled forms' offsets against the sizes of what they point into.
#pragma once

#include <stdint.h>

#include "../../include/m3s.h"

#ifdef __HIPCC__
#define M3S_BOTH __host__ __device__ __forceinline__
#else
#define M3S_BOTH inline
#endif

namespace m3s {

// Streaming forms of 16 and 32 rows to a workgroup, and tiles of 128 x 64, 256 x 64 and 256 x 128 packed
// outputs x rows.
enum Form8 { kFew16, kFew32, kTiles64, kTiles64Wide, kTiles128 };

// The form of rows in 8 bits by np packed outputs, by the workgroups that each makes, of 256 CUs. Few rows go to
// the streaming form, 16 and 32 rows to a workgroup, as long as a CU has one, or two, of them, and up to 16 rows
// at any width (half of a tile of 32 would be empty: 16 x 2048 x 32000 12.4 and 13.8 us, the gate of 16 x 2048 x
// 16384 13.2 and 13.9); then come the tiles, each while the CUs have one of them. us of the five, weights in
// cache: 64 x 1024 x 4480 4.8, 4.4, 8.5, 11.3, 16.3; 256 rows 9.3, 8.9, 8.9, 11.7, 16.7; 768 rows 20.6, 17.5, 11.3,
// 12.5, 17.4; 4096 rows 39.5, 41.8, 40.6 (tiles); 256 x 4096 x 4096 17.5, 14.0, 26, 35, 53; 1024 rows -, 47, 37, 39,
// 54; 4096 rows 129, 116, 104 (tiles). The same borders do for short sums: 64 x 1024 x 4480 4.4, 4.0, 5.4, 6.7,
// 9.3; 256 rows 8.2, 7.3, 5.6, 7.0, 9.8; 768 rows 18.1, 14.1, 8.1, 7.8, 10.5; 4096 rows 25, 25, 23.6 (tiles).
M3S_BOTH Form8 form8(int64_t rows, int64_t np) {
  const int64_t g64 = np / 64, g128 = (np + 127) / 128, g256 = (np + 255) / 256, r64 = (rows + 63) / 64;
  if (rows <= 16 || g64 * ((rows + 15) / 16) <= 256) return kFew16;
  if (g64 * ((rows + 31) / 32) <= 512) return kFew32;
  if (g128 * r64 <= 256) return kTiles64;
  if (g256 * r64 <= 256) return kTiles64Wide;
  return kTiles128;
}

// Whether a product rounds its float rows (k of `size` bytes) itself. Each of its workgroups, 64 outputs and 16
// rows, then rounds all that it reads, which saves a launch as long as a CU rounds little: the rows' bytes times
// the workgroups that a CU takes in turn. Up to 16 rows of bf16 or 8 of float32, whose weight is read once all the
// same, it pays up to 8 KB a row at any width. us in one launch and in two, weights in cache: bf16 16 x 1024 x
// 4480 5.0, 6.6; 112 rows (two turns) 6.8, 9.3; 160 (three) 9.1, 9.7; 192 (four) 10.9, 9.8; 48 x 2048 x 4480 (one)
// 7.5, 8.9; 96 rows (two) 10.8, 10.1; 16 x 2048 x 32000 13.6, 16.2; 1 x 4096 x 8192 10.2, 9.4 (short sums 8.2,
// 9.4), 64 rows 17.4, 12.6. float32: 48 x 1024 x 4480 5.8, 6.8; 64 rows (two) 8.1, 7.3; 8 x 2048 x 32000 13.9, 15.3;
// 1 x 2048 x 1024 6.2, 6.8; 16 rows 8.8, 7.4.
M3S_BOTH bool rounds_in_launch(int64_t rows, int64_t np, int64_t k, int size) {
  if (rows > M3S_MATMUL8_FLOAT_ROWS) return false;
  const int64_t turns = (np / 64 * ((rows + 15) / 16) + 255) / 256;
  return turns * k * size <= 6144 || (rows * size <= 32 && k * size <= 8192);
}

// A step of 64 k that lies in the operands: loads are asked for up to three steps behind the last of S,
// and go nowhere then.
M3S_BOTH int step_within(int s, int S) { return s < S ? s : 0; }

// The weight's scales are a dword for every step of 128 k, group of 64 packed outputs and lane. The byte of a
// group's dword in a step for a lane that takes entry 16 g + r (g < 2: the blocks of a step of 64 k); a group
// behind the last of `groups` reads the last one instead, as its tiles do, and is not stored.
M3S_BOTH uint32_t weight_scale_at(int group, int groups, int entry) {
  return (uint32_t)(group < groups ? group : groups - 1) * 256 + 4 * entry;
}
// ... and of step s of 64 k, for np packed outputs
M3S_BOTH uint32_t weight_scale_step(int s, int np) { return (uint32_t)(s >> 1) * (uint32_t)np * 4 + (s & 1) * 128; }

}  // namespace m3s
