// devword.cuh -- the device error word, and the bounded barrier waits that
// record a timeout in it.  A wait that runs out returns false, so a kernel can
// skip its remaining work, release its TMEM and exit instead of hanging the
// GPU.
#pragma once
#include "ptx.cuh"

namespace boa {

// device error word (read by the host after each synchronising call)
enum : int { BOA_ERR_NONE = 0, BOA_ERR_TIMEOUT = 1, BOA_ERR_STREAM_OVERFLOW = 2, BOA_ERR_BAD_INPUT = 3 };
// One definition: only files that are part of the main translation unit
// (csrc/boa_all.cu) include this header, so device and host code see the same
// symbol.  Files that are compiled on their own (the training operators) would
// get a word of their own that the host never reads, and do not include it.
__device__ int g_dev_error = 0;

__device__ __forceinline__ void set_dev_error(int code) { atomicCAS(&g_dev_error, 0, code); }

// Bounded wait for the phase with the given parity to complete: past the
// limit it records BOA_ERR_TIMEOUT in the device error word and returns false,
// and the caller unwinds without touching the barrier's data.
__device__ __forceinline__ bool mbar_wait_for(uint64_t* bar, uint32_t parity, uint64_t limit_ns) {
  const uint32_t a = smem_u32(bar);
  if (mbar_try_wait(a, parity)) return true;
  const uint64_t t0 = global_ns();
  while (true) {
    if (mbar_try_wait(a, parity)) return true;
    if (global_ns() - t0 > limit_ns) {
      set_dev_error(BOA_ERR_TIMEOUT);
      return false;
    }
  }
}
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity) {
  return mbar_wait_for(bar, parity, kWaitLimitNs);
}

}  // namespace boa
