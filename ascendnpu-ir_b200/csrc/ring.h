// ring.h -- which copies of a producer's ring are still to land when its roles stop.  Plain C++ beside the kernels that
// use it, so that it can be run on a host.
//
// A ring has one barrier a slot; load number i (0, 1, ..) goes into slot i % slots and completes phase i / slots of that
// slot's barrier.  A slot is loaded again only after its last load was used, so of each slot at most the last load can be
// under way, and the parity of exactly that load's phase says when it has landed.  (Either parity of a barrier would not:
// one of the two always names a phase that is over.)
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define BSIR_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define BSIR_HOST_DEVICE inline
#endif

namespace bsir {

// Of a ring whose next load would be number round * slots + `slot`, with `phase` = round & 1: the parity of slot s's last
// load.  Where there was none yet the parity is 1, which a barrier in its first phase lets through at once.
BSIR_HOST_DEVICE uint32_t ring_last_parity(int s, int slot, uint32_t phase) { return s < slot ? phase : phase ^ 1u; }
// The slot used last, in the same terms.
BSIR_HOST_DEVICE int ring_last_slot(int slots, int slot) { return slot == 0 ? slots - 1 : slot - 1; }

// A ring that two CTAs fill: each load's barrier is the leader's, where the leader arrives and announces both CTAs' bytes,
// `bytes` each.  If one gave up, the two may have issued different numbers of loads.  On the leader, when neither issues
// any more: settles every slot's last load on what was really issued, then waits for it.  Bar is the barriers' operations:
//   complete(slot, bytes)   counts bytes that will not come as arrived
//   expect(slot, bytes)     arrives and announces
//   wait(slot, parity)
template <class Bar>
BSIR_HOST_DEVICE void ring_settle_pair(uint32_t slots, uint32_t leader, uint32_t peer, uint32_t bytes, Bar bar) {
  const uint32_t issued = leader > peer ? leader : peer;
  for (uint32_t i = issued > slots ? issued - slots : 0; i < issued; ++i) {
    const uint32_t slot = i % slots;
    if (i >= peer) bar.complete(slot, bytes);        // the leader alone issued it
    else if (i >= leader) bar.expect(slot, bytes);   // the peer alone
    bar.wait(slot, (i / slots) & 1u);
  }
}

}  // namespace bsir
