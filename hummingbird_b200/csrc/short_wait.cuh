// Bounded mbarrier waits of a few instructions, for loops that are inlined into every hot path.
#pragma once
#include "hb_sm100.cuh"

namespace hb {

// The limit counts tries, not time (a loop with a clock cost the tcgen05 context kernel 10 % through its instruction
// cache). A failed try suspends the thread for 3.97 us (measured with 1 to 592 x 256 waiting threads), so this is 1.04 s,
// as kWaitLimitNs, and with the producer's sleeps 1.07 s.
constexpr uint32_t kWaitTries = 1u << 18;

// Ends early once another role has given up; else records the timeout and raises the flag itself.
template <int kSleepNs>
__device__ __forceinline__ bool slow_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
#pragma unroll 1
  for (uint32_t i = 0; i < kWaitTries && !*abort_flag; ++i) {
    if (kSleepNs) __nanosleep(kSleepNs);
    if (mbar_try_wait(bar, parity)) return true;
  }
  if (!*abort_flag) record_error(HB_ERR_TIMEOUT);
  *abort_flag = 1;
  return false;
}

}  // namespace hb
