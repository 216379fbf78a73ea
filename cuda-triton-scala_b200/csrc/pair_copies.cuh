// pair_copies.cuh -- the copies that a CTA pair (tcgen05 cta_group::2) has under way when it gives
// up.  Both CTAs' producers fill their own shared memory, and the even CTA's full barriers count
// the bytes of both.  Where one producer got further than the other before it stopped, a stage's
// count would never come out (the even CTA armed it for both halves), or nobody would wait for
// the half that is on its way.
#pragma once

#include <cuda_runtime.h>

#include "ptx.cuh"

namespace qg {

// Limit of the waits for a CTA's own copies and MMAs after it has given up: the device's wait limit
// may be too short for a copy to land.
constexpr unsigned long long DRAIN_NS = ptx::kWaitLimitNs;

// What a producer did, in its CTA's shared memory at the same offset in both CTAs.
struct PairCopies {
  long long stages;   // filled; written when the producer has stopped
  uint32_t half[8];   // this CTA's bytes of the stage that was last in each place (8 at most)
};

// One thread of the even CTA, after a cluster barrier behind which neither producer issues: settles
// the counts and waits for every copy.  full0: the first full barrier, S of them.  False if a
// copy did not land within DRAIN_NS.
__device__ __forceinline__ bool settle_pair_copies(uint32_t full0, int S, uint32_t copies) {
  const uint32_t here = ptx::map_to_rank(copies, 0), there = ptx::map_to_rank(copies, 1);
  const long long mine = ptx::ld_cluster_s64(here), theirs = ptx::ld_cluster_s64(there);
  const long long first = mine < theirs ? mine : theirs, end = mine < theirs ? theirs : mine;
  for (long long f = first; f < end; ++f) {
    const int at = (int)(f % S);
    const uint32_t bytes = ptx::ld_cluster_u32((mine > theirs ? here : there) + 8u + 4u * at);
    if (mine > theirs) ptx::mbar_complete_tx(full0 + 8u * at, bytes);
    else ptx::mbar_arrive_expect_tx(full0 + 8u * at, bytes);
  }
  for (long long f = end > S ? end - S : 0; f < end; ++f)
    if (!ptx::mbar_wait(full0 + 8u * (int)(f % S), (uint32_t)((f / S) & 1), nullptr, DRAIN_NS))
      return false;
  return true;
}

}  // namespace qg
