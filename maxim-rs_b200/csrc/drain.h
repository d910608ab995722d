// What a tensor-core kernel that gives up still owes: its copies have to land
// before its shared memory goes. Plain C++ apart from the barrier operations
// that the caller passes in, so that it can be run on the CPU.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define MX_DRAIN_FN __device__ __forceinline__
#else
#define MX_DRAIN_FN inline
#endif

namespace mx {

// A ring of `stages` barriers counts copies: round i is counted on barrier i %
// stages, in its (i / stages)-th phase. A CTA has armed and issued the first
// `mine` rounds. Where a pair's copies count on one CTA's barriers, that CTA
// calls this with its own count and the `peers`, which has not armed but only
// issued; else `peers` is `mine`. Neither issues any more. Rounds that one of
// the two issued alone (at most `stages` of them: both wait for the same
// releases) are made whole: arm(stage) where only the peer's copies are on
// their way, cover(stage) for the peer's bytes that an armed round will not see.
// Then every barrier's last phase is waited for. Whether all of them ended.
template <class Arm, class Cover, class Wait>
MX_DRAIN_FN bool land_copies(uint32_t mine, uint32_t peers, uint32_t stages, Arm&& arm, Cover&& cover, Wait&& wait) {
  const uint32_t lo = mine < peers ? mine : peers, hi = mine < peers ? peers : mine;
  for (uint32_t i = lo; i < hi; ++i) {
    if (i >= mine)
      arm(i % stages);
    else
      cover(i % stages);
  }
  bool all = true;
  for (uint32_t i = hi < stages ? 0 : hi - stages; i < hi; ++i)
    if (!wait(i % stages, (i / stages) & 1)) all = false;
  return all;
}

}  // namespace mx
