// What the kernels that read the peers' buffers share: the peers' addresses as kernel arguments
// and the handshake of the one-rank emulation.
#pragma once

#include "smr_internal.hpp"

namespace smr {

// The peers' buffer addresses as kernel arguments.  The reference's kernel reads them from a
// table in device memory (triton_one_shot_all_reduce.py:87): a dependent memory round trip
// in front of every thread's first data load, which a launch of a few microseconds notices.
// A host that knows the addresses passes them by value; all-zero = read the device table.
struct PeerPtrs {
  uint64_t p[SMR_MAX_WORLD_SIZE];
};

// blockwise_barrier for the one-rank emulation: the rank's half of block `block_id`'s handshake
// and, in the same wave and the same loop, the halves of the ws - 1 ranks that nobody runs.
// Lane = role * ws + peer.  Role 0: the rank sends to `peer` (CAS 0 -> 1 on the peer's pad);
// 1: the rank waits for `peer` (own pad); 2: `peer` sends to the rank (the rank's pad, the slot
// role 1 polls); 3: `peer` waits for the rank (the peer's pad, the slot role 0 raised).  One
// loop for all of them, as in blockwise_barrier: every wait depends on a send of a lane
// beside it.  `publish` / `acquire` as there.
template <int WS, typename Pads>
__device__ __forceinline__ bool barrier_with_stand_ins(const Pads& pads, uint32_t block_id, int rank,
                                                       uint64_t limit_ticks, uint32_t* status, bool publish,
                                                       bool acquire) {
  static_assert(4 * WS <= 64, "one wave plays all four roles");
  __syncthreads();
  const int lane = threadIdx.x;
  int bad = 0;
  if (lane < 64) {
    if (publish) __builtin_amdgcn_fence(__ATOMIC_RELEASE, "agent");
    // the consuming write of an earlier call on this slot has been performed
    else wait_stores_acknowledged();
    const int role = lane / WS, peer = lane % WS;
    if (role < 4 && !(role >= 2 && peer == rank)) {
      const bool is_send = (role & 1) == 0;
      const bool peers_pad = role == 0 || role == 3;          // else the rank's own pad
      uint32_t* pad = reinterpret_cast<uint32_t*>(pads[peers_pad ? peer : rank]);
      uint32_t* slot = pad + (size_t)block_id * WS + (peers_pad ? rank : peer);
      SpinClock clk(limit_ticks);
      uint32_t level = 0;
      bool ok = false;
      for (;;) {
        if (is_send) {
          uint32_t expected = 0u;
          ok = __hip_atomic_compare_exchange_strong(slot, &expected, 1u, __ATOMIC_RELAXED, __ATOMIC_RELAXED, kScope);
        } else {
          ok = __hip_atomic_load(slot, __ATOMIC_RELAXED, kScope) == 1u;
        }
        if (ok) break;
        backoff_sleep(level);
        if (clk.expired()) break;
      }
      if (!ok) {
        if (role < 2) report(status, is_send ? SMR_ST_SEND_TIMEOUT : SMR_ST_WAIT_TIMEOUT, rank, block_id, peer);
        else report(status, is_send ? SMR_ST_SEND_TIMEOUT : SMR_ST_WAIT_TIMEOUT, peer, block_id, rank);
        bad = 1;
      } else if (!is_send) {
        __hip_atomic_fetch_and(slot, 0u, __ATOMIC_RELAXED, kScope);       // consume: 1 -> 0
      }
    }
    if (acquire) __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
  }
  bad = __syncthreads_or(bad);
  return bad == 0;
}

}  // namespace smr
