// What orders the lanes of one wavefront.
#pragma once

#include "fm_device.h"

namespace fm {

// What a wavefront's lanes wrote to LDS before it, its lanes read behind it.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

}  // namespace fm
