// Launches with programmatic stream serialization.
#pragma once

#include "runtime.h"

#include <type_traits>

namespace cudeep_b200 {

// Off when the environment variable CUDEEP_B200_PDL is "0" (read once).
bool programmatic_launch_enabled();

// A plain grid whose set-up may overlap the kernel before it (it must wait for it itself).
template <class... Params, class... Args>
void launch_dependent(void (*kernel)(Params...), dim3 grid, int threads, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(unsigned(threads), 1, 1);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = programmatic_launch_enabled() ? 1 : 0;
    CB200_CUDA(cudaLaunchKernelEx(&cfg, kernel, static_cast<std::decay_t<Params>>(args)...));
}

}  // namespace cudeep_b200
