// Library-wide C-ABI entry points: version and the device status word.
#include <cuda_runtime.h>

#include "../../include/hb_b200.h"
#include "abi_common.h"
#include "band_fused.h"
#include "band_proj.h"
#include "context_attn.h"
#include "hb_sm100.cuh"

extern "C" int hb_version(void) { return 100; }

extern "C" int hb_device_status(unsigned int* status_out, cudaStream_t stream) {
  if (!status_out) return HB_ERR_NULL;
  if (cudaStreamSynchronize(stream) != cudaSuccess) return HB_ERR_LAUNCH;
  unsigned int v = 0, vb = 0, vp = 0, vc = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, hb::g_device_status, sizeof(v)) != cudaSuccess) return HB_ERR_LAUNCH;
  if (v && cudaMemcpyToSymbol(hb::g_device_status, &zero, sizeof(zero)) != cudaSuccess) return HB_ERR_LAUNCH;
  // the units compiled as whole-program device code (the fused band kernel, the band front end, the context
  // attention's tcgen05 kernel) keep their own words
  if (hb::band_fused_take_status(&vb) != HB_OK || hb::band_proj_take_status(&vp) != HB_OK ||
      hb::ctx_tiles_take_status(&vc) != HB_OK)
    return HB_ERR_LAUNCH;
  *status_out = v ? v : (vb ? vb : (vp ? vp : vc));
  return HB_OK;
}
