// A ring of loads in flight, each completing on its stage's mbarrier.  Plain arithmetic, for the device and the host.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define MSKV_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define MSKV_HOST_DEVICE inline
#endif

namespace mskv {

// Where tile number t of a warp lies: stage t % kStages, complete with phase (t / kStages) & 1 of its barrier.
template <int kStages>
struct RingPlace {
  int stage;
  uint32_t phase;

  MSKV_HOST_DEVICE explicit RingPlace(uint32_t t) : stage((int)(t % kStages)), phase((t / kStages) & 1) {}
  MSKV_HOST_DEVICE void advance() {
    if (++stage == kStages) {
      stage = 0;
      phase ^= 1;
    }
  }
  // Stage of the tile `ahead` (< kStages) further on.
  MSKV_HOST_DEVICE int stage_ahead(int ahead) const { return stage + ahead < kStages ? stage + ahead : stage + ahead - kStages; }

  // Waits for the loads that are in flight when this is the place of tile i of n: those of tile i and of the up to
  // kStages - 1 tiles after it, each with its own phase.  wait(stage, phase) is bounded; false: one ran out.
  template <typename Wait>
  MSKV_HOST_DEVICE bool drain(int i, int n, const Wait& wait) {
    bool all = true;
    for (int j = i; j < n && j < i + kStages; ++j) {
      all &= wait(stage, phase);
      advance();
    }
    return all;
  }
};

}  // namespace mskv
