// wave_lds.hpp -- a wave's own room in LDS.
#pragma once

#include <hip/hip_runtime.h>

namespace tsr {

// Behind a wave's writes to LDS that its other lanes read, and the other way round: a wave's operations run in order
// there, so that nothing has to be waited for.
__device__ __forceinline__ void own_room() {
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_wave_barrier();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

}  // namespace tsr
