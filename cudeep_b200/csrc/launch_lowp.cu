// cudeep::kernels launchers of the low-precision and grouped products: argument checks.
#include "cudeep/kernels/lowp.cuh"

#include "grouped_gemm.h"
#include "lowp_rows.h"

namespace cudeep {
namespace kernels {

namespace {

int checked_type(ElementType type) {
    const int t = static_cast<int>(type);
    CB200_REQUIRE(t >= 0 && t <= 2, "unknown element type");
    return t;
}

int checked_half_type(ElementType type) {
    const int t = checked_type(type);
    CB200_REQUIRE(t != cudeep_b200::TYPE_F32, "16-bit operands expected (F16 or BF16)");
    return t;
}

int checked_block(Fp8Block block) {
    const int b = static_cast<int>(block);
    CB200_REQUIRE(b == 1 || b == 128, "a block has 1 or 128 rows");
    return b;
}

void check_element_address(const void* p, int bytes, const char* what) {
    CB200_REQUIRE(reinterpret_cast<uintptr_t>(p) % bytes == 0, std::string(what) + " is not aligned to its element type");
}

void check_grouped(const void* a, const void* b, const void* c, const int32_t* offsets, int groups, int rows, int n, int k) {
    CB200_REQUIRE(a != nullptr && b != nullptr && c != nullptr && offsets != nullptr, "grouped matmul: null pointer");
    CB200_REQUIRE(groups > 0 && groups <= 1024, "grouped matmul: 1 to 1024 groups");
    CB200_REQUIRE(rows >= 0 && n > 0 && k > 0, "grouped matmul: rows must not be negative, the other extents positive");
    check_element_address(a, 2, "A");
    check_element_address(b, 2, "B");
    check_element_address(offsets, 4, "offsets");
}

}  // namespace

void launch_quantize_fp8(const void* x, ElementType type, long long rows, int cols, Fp8Block block, void* q, float* scales,
                         cudaStream_t stream) {
    const int t = checked_type(type), b = checked_block(block);
    CB200_REQUIRE(x != nullptr && q != nullptr && scales != nullptr, "quantize_fp8: null pointer");
    CB200_REQUIRE(rows >= 0 && cols > 0, "quantize_fp8: rows must not be negative, cols positive");
    check_element_address(x, cudeep_b200::elem_bytes(t), "x");
    check_element_address(scales, 4, "scales");
    if (rows == 0) return;
    cudeep_b200::quantize_fp8(x, t, rows, cols, b, static_cast<uint8_t*>(q), scales, stream);
}

void launch_dequantize_fp8(const void* q, const float* scales, long long rows, int cols, Fp8Block block, void* y,
                           ElementType type, cudaStream_t stream) {
    const int t = checked_type(type), b = checked_block(block);
    CB200_REQUIRE(y != nullptr && q != nullptr && scales != nullptr, "dequantize_fp8: null pointer");
    CB200_REQUIRE(rows >= 0 && cols > 0, "dequantize_fp8: rows must not be negative, cols positive");
    check_element_address(y, cudeep_b200::elem_bytes(t), "y");
    check_element_address(scales, 4, "scales");
    if (rows == 0) return;
    cudeep_b200::dequantize_fp8(static_cast<const uint8_t*>(q), scales, rows, cols, b, y, t, stream);
}

void launch_grouped_matmul_nt(const void* A, const void* B, void* C, ElementType type, const int32_t* offsets, int groups,
                              int rows, int N, int K, cudaStream_t stream) {
    const int t = checked_half_type(type);
    check_grouped(A, B, C, offsets, groups, rows, N, K);
    check_element_address(C, 2, "C");
    if (rows == 0) return;
    cudeep_b200::grouped_nt(A, B, C, t, offsets, groups, rows, N, K, stream);
}

void launch_grouped_matmul_nn(const void* A, const void* B, void* C, ElementType type, const int32_t* offsets, int groups,
                              int rows, int N, int K, cudaStream_t stream) {
    const int t = checked_half_type(type);
    check_grouped(A, B, C, offsets, groups, rows, N, K);
    check_element_address(C, 2, "C");
    if (rows == 0) return;
    cudeep_b200::grouped_nn(A, B, C, t, offsets, groups, rows, N, K, stream);
}

void launch_grouped_matmul_tn(const void* A, const void* B, void* C, ElementType type, ElementType c_type,
                              const int32_t* offsets, int groups, int rows, int M, int N, cudaStream_t stream) {
    const int t = checked_half_type(type), ct = checked_type(c_type);
    CB200_REQUIRE(ct == cudeep_b200::TYPE_F32 || ct == t, "grouped matmul: C is F32 or of the operands' type");
    check_grouped(A, B, C, offsets, groups, rows, M, N);
    check_element_address(C, cudeep_b200::elem_bytes(ct), "C");
    if (rows == 0) {      // every group is empty
        CB200_CUDA(cudaMemsetAsync(C, 0, size_t(groups) * M * N * cudeep_b200::elem_bytes(ct), stream));
        return;
    }
    cudeep_b200::grouped_tn(A, 0, B, 0, C, t, ct, offsets, groups, rows, M, N, nullptr, stream);
}

}  // namespace kernels
}  // namespace cudeep
