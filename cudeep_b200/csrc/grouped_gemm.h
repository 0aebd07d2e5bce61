// Products of ragged row groups (see grouped_gemm.cu and ragged_gemm.cuh).
#pragma once

#include "lowp_rows.h"
#include "runtime.h"

namespace cudeep_b200 {

// offsets: device pointer to groups + 1 row numbers; nullptr: one group of all rows.  type: TYPE_F16 or TYPE_BF16.
// c[rows, n] = a[rows, k] * w[g][n, k]^T
void grouped_nt(const void* a, const void* w, void* c, int type, const int32_t* offsets, int groups, int rows, int n, int k,
                cudaStream_t stream);
// c[rows, n] = a[rows, k] * w[g][k, n].  lda, ldw: elements between rows; 0: contiguous, of any alignment; given, the rows
// are as AlignedRows has them.
void grouped_nn(const void* a, long long lda, const void* w, long long ldw, void* c, int type, const int32_t* offsets, int groups,
                int rows, int n, int k, cudaStream_t stream);
// Where operands of the one-group product may come in another form, which the device decides: if any of `blocks` words of `wide`
// is set, b is BF16 and a the sum of two BF16 matrices [rows, m] one behind the other in `parts`, rows ld_parts (a multiple of
// 64) elements apart, and there is no col_scale.
struct WideOperands {
    const uint32_t* wide = nullptr;      // nullptr: one form only
    int blocks = 0;
    const void* parts = nullptr;
    long long ld_parts = 0;
};
// c[g][m, n] = a[rows of g, m]^T * b[rows of g, n], times col_scale[n / 128] where given.  c_type: `type` or TYPE_F32.
// lda, ldb as above.
void grouped_tn(const void* a, long long lda, const void* b, long long ldb, void* c, int type, int c_type,
                const int32_t* offsets, int groups, int rows, int m, int n, const float* col_scale, const WideOperands& wide,
                cudaStream_t stream);

}  // namespace cudeep_b200
