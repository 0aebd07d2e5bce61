// Launchers of the low-precision and grouped products (additions: the reference has no counterpart).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "cudeep/kernels/matmul.cuh"

namespace cudeep {
namespace kernels {

// Element types of the operands that are passed as void pointers.
enum class ElementType : int { F32 = 0, F16 = 1, BF16 = 2 };

// Blocks of an 8-bit matrix that share a scale: 128 columns of one row (activations), or 128 rows x 128 columns
// (weights).  Scales lie [column block][row] and [row block][column block].
enum class Fp8Block : int { Row = 1, Tile = 128 };

// dst = src in another element type, rounded to nearest even.
void launch_cast(const void* src, ElementType src_type, void* dst, ElementType dst_type, long long count,
                 cudaStream_t stream = nullptr);

void launch_quantize_fp8(const void* x, ElementType type, long long rows, int cols, Fp8Block block, void* q, float* scales,
                         cudaStream_t stream = nullptr);
void launch_dequantize_fp8(const void* q, const float* scales, long long rows, int cols, Fp8Block block, void* y,
                           ElementType type, cudaStream_t stream = nullptr);

// y[M,N] = act(x * W^T + bias) and dx[M,K] = dy * W on 8-bit operands with scales per block: x and dy with row blocks, W
// with tile blocks.
void launch_linear_forward_fp8(const void* x, const float* x_scales, const void* W, const float* w_scales, const float* bias,
                               void* y, ElementType y_type, int M, int N, int K, GemmEpilogue epilogue,
                               cudaStream_t stream = nullptr);
void launch_linear_backward_data_fp8(const void* dy, const float* dy_scales, const void* W, const float* w_scales, void* dx,
                                     ElementType dx_type, int M, int N, int K, cudaStream_t stream = nullptr);

// Backward pass of y = act(z), z = x * W^T + bias from x and z kept as row blocks of 8 bits.
void launch_linear_backward_saved_fp8(const void* dy, ElementType type, const void* x8, const float* x_scales, const void* z8,
                                      const float* z_scales, GemmEpilogue epilogue, const void* W, void* dx, void* dw,
                                      ElementType dw_type, float* db, int M, int N, int K, cudaStream_t stream = nullptr);

// Products of ragged row groups; `offsets` (device) holds groups + 1 ascending row numbers in [0, rows].
void launch_grouped_matmul_nt(const void* A, const void* B, void* C, ElementType type, const int32_t* offsets, int groups,
                              int rows, int N, int K, cudaStream_t stream = nullptr);
void launch_grouped_matmul_nn(const void* A, const void* B, void* C, ElementType type, const int32_t* offsets, int groups,
                              int rows, int N, int K, cudaStream_t stream = nullptr);
void launch_grouped_matmul_tn(const void* A, const void* B, void* C, ElementType type, ElementType c_type,
                              const int32_t* offsets, int groups, int rows, int M, int N, cudaStream_t stream = nullptr);

}  // namespace kernels
}  // namespace cudeep
