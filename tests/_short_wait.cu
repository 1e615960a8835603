// Waits on barriers that nobody, or a late thread, arrives at: what tests/test_short_wait_gpu.py loads.
#define HB_WHOLE_PROGRAM 1
#include "short_wait.cuh"

struct Result {
  int arrived, gave_up, after_abort;
  unsigned int status;
  unsigned long long ns_never, ns_abort;
};

namespace {

template <int kSleepNs>
__global__ void wait_kernel(Result* out) {
  __shared__ uint64_t late, never;
  __shared__ int flag;
  volatile int* abort_flag = &flag;
  if (threadIdx.x == 0) {
    hb::mbar_init(&late, 1);
    hb::mbar_init(&never, 1);
    flag = 0;
    hb::fence_mbar_init();
  }
  __syncthreads();
  if (threadIdx.x == 32) {  // 2 ms later: hundreds of tries
    const uint64_t t0 = hb::globaltimer_ns();
    while (hb::globaltimer_ns() - t0 < 2000000) __nanosleep(1000);
    hb::mbar_arrive(&late);
  }
  if (threadIdx.x == 0) {
    out->arrived = hb::slow_wait<kSleepNs>(&late, 0, abort_flag) && !flag;
    uint64_t t0 = hb::globaltimer_ns();
    out->gave_up = !hb::slow_wait<kSleepNs>(&never, 0, abort_flag) && flag;
    out->ns_never = hb::globaltimer_ns() - t0;
    t0 = hb::globaltimer_ns();
    out->after_abort = !hb::slow_wait<kSleepNs>(&never, 0, abort_flag);
    out->ns_abort = hb::globaltimer_ns() - t0;
    out->status = hb::g_device_status_local;
  }
}

}  // namespace

extern "C" int short_wait_run(int sleep, Result* result) {
  Result* d = nullptr;
  if (cudaMalloc(&d, sizeof(Result)) != cudaSuccess) return 1;
  if (sleep) wait_kernel<200><<<1, 64>>>(d);
  else wait_kernel<0><<<1, 64>>>(d);
  const bool ok = cudaMemcpy(result, d, sizeof(Result), cudaMemcpyDeviceToHost) == cudaSuccess;
  cudaFree(d);
  return ok ? 0 : 1;
}
