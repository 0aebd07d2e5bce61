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
// c[g][m, n] = a[rows of g, m]^T * b[rows of g, n], times col_scale[n / 128] where given.  c_type: `type` or TYPE_F32.
// lda, ldb as above.
void grouped_tn(const void* a, long long lda, const void* b, long long ldb, void* c, int type, int c_type,
                const int32_t* offsets, int groups, int rows, int m, int n, const float* col_scale, cudaStream_t stream);

}  // namespace cudeep_b200
