// The bookkeeping of one warp's ring of load stages, apart from what a barrier and a load are: paged.cu uses it with
// mbarriers and TMA, a test on the CPU with a model of them.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define MOA_RING_FN __host__ __device__ __forceinline__
#else
#define MOA_RING_FN inline
#endif

namespace moa {

// Stages are armed (a load is asked for, the stage's barrier completes a phase when it is there) and taken, in turn: first
// all of them are armed, then each is taken and armed again, as long as there is something to load.
// `wait(stage, parity)` waits for the phase of that parity, with a limit, and is false when it ran out.  From then on the
// ring is late and stays where it is: nothing may be taken or armed any more, for a barrier whose phase is open cannot
// take another load's, nor its buffer another load.
template <int kStages>
struct Ring {
  int stage = 0;            // taken next
  uint32_t parity = 0;      // of its barrier's phase
  bool late = false;

  template <typename Wait>
  MOA_RING_FN void take(Wait wait) {
    late = !wait(stage, parity);
  }
  MOA_RING_FN void next() {
    if (!late) advance();
  }
  // At the end: a late ring's loads under way, from the one that was waited for in vain on, are waited for once more, so
  // that none of them lands in a block that has ended.  (Which stages were armed is not noted: for those that were not,
  // the wait runs out.)
  template <typename Wait>
  MOA_RING_FN void drain(Wait wait) {
#pragma unroll 1
    for (int s = 0; s < kStages; ++s) {
      wait(stage, parity);
      advance();
    }
  }

 private:
  MOA_RING_FN void advance() {
    if (++stage == kStages) {
      stage = 0;
      parity ^= 1;
    }
  }
};

}  // namespace moa
