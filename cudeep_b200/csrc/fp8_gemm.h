// Products of 8-bit matrices with block scales (see fp8_gemm.cu and fp8_gemm.cuh).
#pragma once

#include "lowp_rows.h"
#include "runtime.h"

namespace cudeep_b200 {

// y[m, n] = act(x[m, k] * w[n, k]^T + bias[n]); x_scales [k blocks][m], w_scales [n blocks][k blocks].
void fp8_nt(const uint8_t* x, const float* x_scales, const uint8_t* w, const float* w_scales, const float* bias, void* y,
            int y_type, int m, int n, int k, int act, cudaStream_t stream);
// dx[m, k] = dy[m, n] * w[n, k]; dy_scales [n blocks][m], w_scales [n blocks][k blocks].
void fp8_nn(const uint8_t* dy, const float* dy_scales, const uint8_t* w, const float* w_scales, void* dx, int dx_type, int m,
            int n, int k, cudaStream_t stream);

}  // namespace cudeep_b200
