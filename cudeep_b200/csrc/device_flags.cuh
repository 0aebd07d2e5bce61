// Flags that one kernel leaves for those behind it in the stream.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace cudeep_b200 {

// Whether any of `count` words is set; all threads of the CTA.
__device__ __forceinline__ bool any_set(const uint32_t* flags, int count) {
    uint32_t set = 0;
    for (int i = int(threadIdx.x); i < count; i += int(blockDim.x)) set |= __ldg(flags + i);
    return __syncthreads_or(int(set)) != 0;
}

}  // namespace cudeep_b200
