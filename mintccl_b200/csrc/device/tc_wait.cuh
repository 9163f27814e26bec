// Bounded waits on mbarriers inside the tensor-core kernels: on expiry the CTA's abort flag is raised, which ends every
// other wait of the CTA too; the kernel then leaves its loops, frees its TMEM and reports.
#pragma once
#include "prims.cuh"
#include "tc_prims.cuh"

namespace mt {
namespace tc {

__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile int* abort_flag, uint64_t timeout_ns) {
  uint32_t spins = 0;
  uint64_t t0 = 0;
  while (!mbar_try_wait(bar, parity)) {
    if ((++spins & 0x3ffu) == 0) {
      if (*abort_flag) return false;
      const uint64_t now = globaltimer();
      if (t0 == 0) t0 = now;
      else if (now - t0 > timeout_ns) {
        *abort_flag = 1;
        return false;
      }
    }
  }
  return true;
}

// The same for a whole warp: one answer for all lanes, so that the issue loops stay warp-uniform.  CLUSTER: other CTAs
// arrive with mbar_arrive_cluster_release, and fence_acquire_cluster_smem follows.
template <bool CLUSTER>
__device__ __forceinline__ bool try_wait_scope(uint64_t* bar, uint32_t parity) {
  return CLUSTER ? mbar_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity);
}
template <bool CLUSTER>
static __device__ __noinline__ bool wait_bar_warp_slow(uint64_t* bar, uint32_t parity, volatile int* abort_flag, uint64_t timeout_ns) {
  uint32_t spins = 0;
  uint64_t t0 = 0;
  while (!__all_sync(0xffffffffu, try_wait_scope<CLUSTER>(bar, parity))) {
    if ((++spins & 0x3ffu) == 0) {
      if (__any_sync(0xffffffffu, *abort_flag != 0)) return false;
      const uint64_t now = __shfl_sync(0xffffffffu, globaltimer(), 0);
      if (t0 == 0) t0 = now;
      else if (now - t0 > timeout_ns) {
        *abort_flag = 1;
        return false;
      }
    }
  }
  return true;
}
template <bool CLUSTER = false>
__device__ __forceinline__ bool wait_bar_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag, uint64_t timeout_ns) {
  if (__all_sync(0xffffffffu, try_wait_scope<CLUSTER>(bar, parity))) return true;
  return wait_bar_warp_slow<CLUSTER>(bar, parity, abort_flag, timeout_ns);
}
__device__ __forceinline__ bool aborted_warp(volatile int* abort_flag) { return __any_sync(0xffffffffu, *abort_flag != 0); }

}  // namespace tc
}  // namespace mt
