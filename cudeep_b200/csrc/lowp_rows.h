// One-pass kernels around the 8-bit and the grouped products (see lowp_rows.cu).
#pragma once

#include "runtime.h"

namespace cudeep_b200 {

// Element types of the low-precision entry points; values equal CUDEEP_B200_TYPE_*.
enum ElemType : int { TYPE_F32 = 0, TYPE_F16 = 1, TYPE_BF16 = 2 };
inline int elem_bytes(int type) { return type == TYPE_F32 ? 4 : 2; }

constexpr int FP8_BLOCK = 128;      // elements along a row that share a scale

// A row-major matrix whose rows the TMA unit can read: 16-byte aligned, rows of 16-byte multiples.
struct AlignedRows {
    const void* ptr = nullptr;
    long long ld = 0;      // elements between rows
    Scratch copy;          // holds ptr where the caller's matrix had to be copied
};
// The caller's matrix itself where it qualifies, else a copy with zero-padded rows.  With `offsets` (device), rows_group rows belong
// to each of their groups, and groups without rows need not be copied.
AlignedRows aligned_rows(const void* src, long long rows, int cols, int elem_size, cudaStream_t stream,
                         const int32_t* offsets = nullptr, int rows_group = 1);

// dst = src, rounded to dst_type.
void cast(const void* src, int src_type, void* dst, int dst_type, long long count, cudaStream_t stream);

// q = e4m3(x / s), s a power of two for each block of 128 columns and block_rows (1 or 128) rows.
void quantize_fp8(const void* x, int x_type, long long rows, int cols, int block_rows, uint8_t* q, float* scales,
                  cudaStream_t stream);
// y = q * s.
void dequantize_fp8(const uint8_t* q, const float* scales, long long rows, int cols, int block_rows, void* y, int y_type,
                    cudaStream_t stream);


// dz = dy * act'(z8 * z_scales), rounded to dy's type, rows ld_dz elements apart (zeros behind cols); dz may be nullptr.
// db[cols] = column sums of dz before its rounding; db may be nullptr.  type: TYPE_F16 or TYPE_BF16.
void activation_backward_fp8(const void* dy, int type, const uint8_t* z8, const float* z_scales, int act, void* dz,
                             long long ld_dz, float* db, int rows, int cols, cudaStream_t stream);
// y = q * (s / top[b]) in a 16-bit type, rows ld_y elements apart, for blocks of 1 x 128; top[b] = the largest finite
// scale of column block b.  With top == nullptr: y = q * s.
void block_tops(const float* scales, int rows, int cols, float* top, cudaStream_t stream);
void dequantize_rows(const uint8_t* q, const float* scales, const float* top, int rows, int cols, void* y, long long ld_y,
                     int y_type, cudaStream_t stream);

// out[m, n] = sum over `parts` of part[parts][m][ld], in order, rounded to `type`.  ld is a multiple of 4.
void add_parts(const float* part, int parts, int m, int n, long long ld, void* out, int type, cudaStream_t stream);

}  // namespace cudeep_b200
