// cudeep::kernels launchers of the low-precision and grouped products: argument checks.
#include "cudeep/kernels/lowp.cuh"

#include "epilogue_math.cuh"
#include "fp8_gemm.h"
#include "grouped_gemm.h"
#include "lowp_rows.h"

#include <initializer_list>

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

// The kernels add up to a tile, or a band of rows, to an extent in 32 bits.
void check_extents(std::initializer_list<int> extents) {
    for (int e : extents) CB200_REQUIRE(e <= 2147483647 - 65535, "extents are at most 2^31 - 65536");
}

void check_grouped(const void* a, const void* b, const void* c, const int32_t* offsets, int groups, int rows, int n, int k) {
    CB200_REQUIRE(a != nullptr && b != nullptr && c != nullptr && offsets != nullptr, "grouped matmul: null pointer");
    CB200_REQUIRE(groups > 0 && groups <= 1024, "grouped matmul: 1 to 1024 groups");
    CB200_REQUIRE(rows >= 0 && n > 0 && k > 0, "grouped matmul: rows must not be negative, the other extents positive");
    check_extents({rows, n, k});
    check_element_address(a, 2, "A");
    check_element_address(b, 2, "B");
    check_element_address(offsets, 4, "offsets");
}

int checked_epilogue(GemmEpilogue epilogue) {
    const int act = static_cast<int>(epilogue);
    CB200_REQUIRE(act >= 0 && act <= 4, "unknown epilogue code");
    return act;
}

}  // namespace

void launch_cast(const void* src, ElementType src_type, void* dst, ElementType dst_type, long long count, cudaStream_t stream) {
    const int st = checked_type(src_type), dt = checked_type(dst_type);
    CB200_REQUIRE(src != nullptr && dst != nullptr, "cast: null pointer");
    CB200_REQUIRE(count >= 0, "cast: count must not be negative");
    check_element_address(src, cudeep_b200::elem_bytes(st), "src");
    check_element_address(dst, cudeep_b200::elem_bytes(dt), "dst");
    if (count == 0) return;
    cudeep_b200::cast(src, st, dst, dt, count, stream);
}

void launch_quantize_fp8(const void* x, ElementType type, long long rows, int cols, Fp8Block block, void* q, float* scales,
                         cudaStream_t stream) {
    const int t = checked_type(type), b = checked_block(block);
    CB200_REQUIRE(x != nullptr && q != nullptr && scales != nullptr, "quantize_fp8: null pointer");
    CB200_REQUIRE(rows >= 0 && cols > 0, "quantize_fp8: rows must not be negative, cols positive");
    check_extents({cols});
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
    check_extents({cols});
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
    cudeep_b200::grouped_nn(A, 0, B, 0, C, t, offsets, groups, rows, N, K, stream);
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
    cudeep_b200::grouped_tn(A, 0, B, 0, C, t, ct, offsets, groups, rows, M, N, nullptr, {}, stream);
}

void launch_linear_forward_fp8(const void* x, const float* x_scales, const void* W, const float* w_scales, const float* bias,
                               void* y, ElementType y_type, int M, int N, int K, GemmEpilogue epilogue, cudaStream_t stream) {
    const int t = checked_type(y_type), act = checked_epilogue(epilogue);
    CB200_REQUIRE(x != nullptr && x_scales != nullptr && W != nullptr && w_scales != nullptr && y != nullptr,
                  "linear_fp8: null pointer");
    CB200_REQUIRE(M >= 0 && N > 0 && K > 0, "linear_fp8: M must not be negative, N and K positive");
    check_extents({M, N, K});
    check_element_address(y, cudeep_b200::elem_bytes(t), "y");
    check_element_address(x_scales, 4, "x_scales");
    check_element_address(w_scales, 4, "w_scales");
    check_element_address(bias, 4, "bias");
    if (M == 0) return;
    cudeep_b200::fp8_nt(static_cast<const uint8_t*>(x), x_scales, static_cast<const uint8_t*>(W), w_scales, bias, y, t, M, N, K,
                        act, stream);
}

void launch_linear_backward_data_fp8(const void* dy, const float* dy_scales, const void* W, const float* w_scales, void* dx,
                                     ElementType dx_type, int M, int N, int K, cudaStream_t stream) {
    const int t = checked_type(dx_type);
    CB200_REQUIRE(dy != nullptr && dy_scales != nullptr && W != nullptr && w_scales != nullptr && dx != nullptr,
                  "linear_fp8: null pointer");
    CB200_REQUIRE(M >= 0 && N > 0 && K > 0, "linear_fp8: M must not be negative, N and K positive");
    check_extents({M, N, K});
    check_element_address(dx, cudeep_b200::elem_bytes(t), "dx");
    check_element_address(dy_scales, 4, "dy_scales");
    check_element_address(w_scales, 4, "w_scales");
    if (M == 0) return;
    cudeep_b200::fp8_nn(static_cast<const uint8_t*>(dy), dy_scales, static_cast<const uint8_t*>(W), w_scales, dx, t, M, N, K,
                        stream);
}

void launch_linear_backward_saved_fp8(const void* dy, ElementType type, const void* x8, const float* x_scales, const void* z8,
                                      const float* z_scales, GemmEpilogue epilogue, const void* W, void* dx, void* dw,
                                      ElementType dw_type, float* db, int M, int N, int K, cudaStream_t stream) {
    using namespace cudeep_b200;
    const int t = checked_half_type(type), act = checked_epilogue(epilogue);
    CB200_REQUIRE(dy != nullptr, "linear_backward_saved: null dy");
    CB200_REQUIRE(dx != nullptr || dw != nullptr || db != nullptr, "linear_backward_saved: no gradient asked for");
    CB200_REQUIRE(dx == nullptr || W != nullptr, "linear_backward_saved: dx needs W");
    CB200_REQUIRE(dw == nullptr || (x8 != nullptr && x_scales != nullptr), "linear_backward_saved: dw needs x8 and its scales");
    CB200_REQUIRE(act == EPI_NONE || (z8 != nullptr && z_scales != nullptr),
                  "linear_backward_saved: an activation needs z8 and its scales");
    CB200_REQUIRE(M >= 0 && N > 0 && K > 0, "linear_backward_saved: M must not be negative, N and K positive");
    check_extents({M, N, K});
    CB200_REQUIRE(dw == nullptr || t != TYPE_F16 || M <= (1 << 29), "linear_backward_saved: at most 2^29 rows for the dw of F16 operands");
    const int wt = dw != nullptr ? checked_type(dw_type) : t;
    CB200_REQUIRE(wt == t || wt == TYPE_F32, "linear_backward_saved: dw is F32 or of dy's type");
    check_element_address(dy, 2, "dy");
    check_element_address(W, 2, "W");
    check_element_address(dx, 2, "dx");
    check_element_address(dw, elem_bytes(wt), "dw");
    check_element_address(db, 4, "db");
    check_element_address(x_scales, 4, "x_scales");
    check_element_address(z_scales, 4, "z_scales");
    if (M == 0) {
        if (dw != nullptr) CB200_CUDA(cudaMemsetAsync(dw, 0, size_t(N) * K * elem_bytes(wt), stream));
        if (db != nullptr) CB200_CUDA(cudaMemsetAsync(db, 0, size_t(N) * sizeof(float), stream));
        return;
    }
    // W, and dy where the products read it themselves, as the TMA unit reads them.  And x as a 16-bit operand: q * s is exact in
    // BF16 for the power-of-two scales of quantize_fp8.  FP16 has fewer exponents: there each column block is taken relative to
    // its largest scale, by which the result is multiplied, exact too while the scales of a block lie within 2^15 of each other.
    // Where they do not (rows of zeros, whose scale is 1, next to small values; a row far larger than the others) the device
    // takes x in BF16, and dz, rounded to FP16 as ever, as the sum of two BF16 matrices: two products, and nothing is lost.
    Scratch top_buf;
    ScaleTops tops;
    if (dw != nullptr && t == TYPE_F16) {
        tops = ScaleTops{x_scales, M, K};
        top_buf = Scratch(size_t(tops.blocks()) * (sizeof(float) + sizeof(uint32_t)), stream);
        tops.top = static_cast<float*>(top_buf.ptr);
        tops.wide = reinterpret_cast<uint32_t*>(tops.top + tops.blocks());
    }
    const bool products = dx != nullptr || dw != nullptr;
    const PreparedRows operands = prepare_rows({dx != nullptr ? W : nullptr, N, K, 2},
                                               {act == EPI_NONE && products ? dy : nullptr, M, N, 2}, tops, stream);
    // dz goes to the tensor cores in dy's type: both products take it as an operand next to 16-bit W and x.  db is summed
    // from its FP32 values.
    const void* dz = operands.b.ptr;
    long long ld_dz = operands.b.ld;
    Scratch dz_buf;
    ColumnSums sums;
    if (act != EPI_NONE) {
        if (products) {
            ld_dz = (N + 63) / 64 * 64;      // whole 128-byte rows of a box
            dz_buf = Scratch(size_t(M) * ld_dz * 2, stream);
            dz = dz_buf.ptr;
        }
        sums = activation_backward_fp8(dy, t, static_cast<const uint8_t*>(z8), z_scales, act, dz_buf.ptr, ld_dz, db, M, N, stream);
    } else if (db != nullptr) {
        sums = activation_backward_fp8(dy, t, nullptr, nullptr, act, nullptr, 0, db, M, N, stream);
    }
    if (dx != nullptr) grouped_nn(dz, ld_dz, operands.a.ptr, operands.a.ld, dx, t, nullptr, 1, M, K, N, stream);
    if (dw == nullptr) return finish_sums(sums, stream);
    const long long ld_x = (K + 63) / 64 * 64;
    const long long ld_parts = (N + 63) / 64 * 64;
    const size_t x_bytes = size_t(M) * ld_x * 2, parts_bytes = t == TYPE_F16 ? size_t(M) * ld_parts * 4 : 0;
    Scratch x_buf(x_bytes + parts_bytes, stream);
    SplitRequest split;
    WideOperands wide;
    if (t == TYPE_F16) {
        void* parts = static_cast<uint8_t*>(x_buf.ptr) + x_bytes;
        split = SplitRequest{dz, ld_dz, N, parts, ld_parts};
        wide = WideOperands{tops.wide, tops.blocks(), parts, ld_parts};
    }
    dequantize_rows(static_cast<const uint8_t*>(x8), x_scales, tops, M, K, x_buf.ptr, ld_x, t, sums, split, stream);
    grouped_tn(dz, ld_dz, x_buf.ptr, ld_x, dw, t, wt, nullptr, 1, M, N, K, tops.top, wide, stream);
}

}  // namespace kernels
}  // namespace cudeep
