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
// A matrix that is wanted so; src may be nullptr.  With `offsets` (device), rows_group rows belong to each of their groups, and
// groups without rows need not be copied.
struct RowsRequest {
    const void* src = nullptr;
    long long rows = 0;
    int cols = 0;
    int elem_size = 1;
    long long ld = 0;      // nonzero: its rows qualify already, that many elements apart
    const int32_t* offsets = nullptr;
    int rows_group = 1;
};
// top[b] = the largest finite scale of column block b, and wide[b] = 1 where FP16 does not hold q * (s / top[b]) for all of its
// scales, 0 where it does; nothing with top == nullptr.
struct ScaleTops {
    const float* scales = nullptr;      // [block][rows]
    int rows = 0, cols = 0;
    float* top = nullptr;
    uint32_t* wide = nullptr;
    int blocks() const { return (cols + FP8_BLOCK - 1) / FP8_BLOCK; }
};
struct PreparedRows {
    AlignedRows a, b;
};
// The callers' matrices themselves where they qualify, else copies with zero-padded rows; all that is to be done in one launch.
PreparedRows prepare_rows(const RowsRequest& a, const RowsRequest& b, const ScaleTops& tops, cudaStream_t stream);

// dst = src, rounded to dst_type.
void cast(const void* src, int src_type, void* dst, int dst_type, long long count, cudaStream_t stream);

// q = e4m3(x / s), s a power of two for each block of 128 columns and block_rows (1 or 128) rows.
void quantize_fp8(const void* x, int x_type, long long rows, int cols, int block_rows, uint8_t* q, float* scales,
                  cudaStream_t stream);
// y = q * s.
void dequantize_fp8(const uint8_t* q, const float* scales, long long rows, int cols, int block_rows, void* y, int y_type,
                    cudaStream_t stream);

// Column sums on their way: of each band of rows, to be added up by finish_sums or along with dequantize_rows.
struct ColumnSums {
    Scratch partial;
    int bands = 0, cols = 0;
    float* out = nullptr;      // nullptr: nothing is left to do
};
// dz = dy * act'(z8 * z_scales), rounded to dy's type, rows ld_dz elements apart (zeros behind cols); dz may be nullptr.
// db[cols] = column sums of dz before its rounding, once the result is finished; db may be nullptr.  type: TYPE_F16 or TYPE_BF16.
ColumnSums activation_backward_fp8(const void* dy, int type, const uint8_t* z8, const float* z_scales, int act, void* dz,
                                   long long ld_dz, float* db, int rows, int cols, cudaStream_t stream);
void finish_sums(const ColumnSums& sums, cudaStream_t stream);
// An FP16 matrix as two BF16 matrices whose sum it is, one behind the other in `parts`, rows ld_parts elements apart: 8 of its 11
// bits and the other 3.  Made only where ScaleTops::wide has an entry set.
struct SplitRequest {
    const void* src = nullptr;      // rows as AlignedRows has them
    long long ld = 0;
    int cols = 0;
    void* parts = nullptr;
    long long ld_parts = 0;
};
// y = q * s in a 16-bit type, rows ld_y elements apart, for blocks of 1 x 128.  In FP16, which needs `tops` and `split`,
// q * (s / top[b]), or, where an entry of tops.wide is set, q * s in BF16, and then `split` is made.  Finishes `sums` as well.
void dequantize_rows(const uint8_t* q, const float* scales, const ScaleTops& tops, int rows, int cols, void* y, long long ld_y,
                     int y_type, const ColumnSums& sums, const SplitRequest& split, cudaStream_t stream);

// out[m, n] = sum over `parts` of part[parts][m][ld], in order, rounded to `type`.  ld is a multiple of 4.
void add_parts(const float* part, int parts, int m, int n, long long ld, void* out, int type, cudaStream_t stream);

}  // namespace cudeep_b200
