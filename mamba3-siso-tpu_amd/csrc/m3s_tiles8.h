// Index rules of the tiled products in 8 bits (m3s_matmul8.hip), apart so that a test on the host can
// hold them to the sizes of what they point into.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define M3S_BOTH __host__ __device__ __forceinline__
#else
#define M3S_BOTH inline
#endif

namespace m3s {

// A step of 64 k that lies in the operands: loads are asked for up to three steps behind the last of S,
// and go nowhere then.
M3S_BOTH int step_within(int s, int S) { return s < S ? s : 0; }

// The weight's scales are a dword for every step of 128 k, group of 64 packed outputs and lane. The byte of
// a group's dword in a step for a lane that takes entry 16 g + r (g < 2: the blocks of a step of 64 k); a group behind the last of `groups` reads the
// last one instead, as its tiles do, and is not stored.
M3S_BOTH uint32_t weight_scale_at(int group, int groups, int entry) {
  return (uint32_t)(group < groups ? group : groups - 1) * 256 + 4 * entry;
}
// ... and of step s of 64 k, for np packed outputs
M3S_BOTH uint32_t weight_scale_step(int s, int np) { return (uint32_t)(s >> 1) * (uint32_t)np * 4 + (s & 1) * 128; }

}  // namespace m3s
