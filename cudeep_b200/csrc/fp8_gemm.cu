// Launchers of the 8-bit products of fp8_gemm.cuh.
#include "fp8_gemm.h"

#include "fp8_gemm.cuh"
#include "fp8_rows.cuh"
#include "ragged_plan.h"

namespace cudeep_b200 {

namespace {

// CTAs that share a tile of 128 features: as many as the device has SMs for, while each keeps four blocks of K.
int cluster_split(int features, int k) {
    const int tiles = (features + 127) / 128, blocks = (k + FP8_BK - 1) / FP8_BK;
    int split = 1;
    while (split < 8 && tiles * split * 2 <= device_info().num_sms && blocks >= 8 * split) split *= 2;
    return split;
}

template <RaggedForm FORM, class OutT>
void launch_few(Fp8FewParams& p, cudaStream_t stream) {
    const DeviceInfo& dev = device_info();
    CB200_REQUIRE(dev.cc_major == 10, "8-bit products need an sm_100 device");
    p.split = cluster_split(p.features, p.k);
    p.stage_bytes = RAGGED_A_BYTES + uint32_t(RowMaps::loaded((p.rows + 15) / 16 * 16)) * 128u;
    const int fit = int(FP8F_SMEM_BUDGET / p.stage_bytes);
    p.stages = fit < FP8F_MAX_STAGES ? fit : FP8F_MAX_STAGES;
    p.status = dev.status_word;
    p.wait_limit_ns = 2000000000ull;
    const long long tiles = (p.features + 127) / 128;
    CB200_TRACE("fp8 %s tcgen05, features on lanes: rows=%d features=%d k=%d stages=%d tiles=%lld split=%d",
                FORM == RaggedForm::NT ? "nt" : "nn", p.rows, p.features, p.k, p.stages, tiles, p.split);
    launch_clusters(fp8_few_kernel<FORM, OutT>, p, tiles, p.split, FP8F_THREADS, uint32_t(p.stages) * p.stage_bytes + 1024,
                    FP8F_SMEM_BUDGET + 1024, stream);
}

template <RaggedForm FORM, class OutT>
void launch_by_rows(Fp8RowsParams& p, cudaStream_t stream) {
    const DeviceInfo& dev = device_info();
    CB200_REQUIRE(dev.cc_major == 10, "8-bit products need an sm_100 device");
    p.tma_store = (size_t(p.features) * sizeof(OutT)) % 16 == 0 && reinterpret_cast<uintptr_t>(p.c) % 16 == 0;
    if (p.tma_store) {
        const uint64_t dims[2] = {uint64_t(p.features), uint64_t(p.rows)};
        const uint64_t strides[1] = {uint64_t(p.features) * sizeof(OutT)};
        const uint32_t box[2] = {uint32_t(128 / sizeof(OutT)), 32};
        if (sizeof(OutT) == 4) encode_tensor_map(&p.map_c, static_cast<const float*>(p.c), 2, dims, strides, box, TmaSwizzle::B128);
        else encode_tensor_map_f16(&p.map_c, p.c, 2, dims, strides, box, TmaSwizzle::B128);
    }
    p.status = dev.status_word;
    p.wait_limit_ns = 2000000000ull;
    p.tiles_m = (p.rows + 255) / 256;
    p.tiles_n = (p.features + 255) / 256;
    const long long tiles = (long long)p.tiles_m * p.tiles_n;
    const long long clusters = tiles < dev.num_sms / 2 ? tiles : dev.num_sms / 2;
    CB200_TRACE("fp8 %s tcgen05, rows on lanes: rows=%d features=%d k=%d tile=256x256 stages=%d clusters=%lld store=%s",
                FORM == RaggedForm::NT ? "nt" : "nn", p.rows, p.features, p.k, FP8R_STAGES, clusters,
                p.tma_store ? "bulk-tensor" : "rows");
    launch_clusters(fp8_rows_kernel<FORM, OutT>, p, clusters, 2, FP8R_THREADS, FP8R_SMEM_BYTES, FP8R_SMEM_BYTES, stream);
}

// x[m, k] by w, stored [n, k] (NT: features n) or [k, n] (NN: features n).
template <RaggedForm FORM>
void product(const uint8_t* x, const float* x_scales, const uint8_t* w, const float* w_scales, const float* bias, void* y,
             int y_type, int m, int n, int k, int act, cudaStream_t stream) {
    constexpr bool nn = FORM == RaggedForm::NN;
    const int w_cols = nn ? n : k, w_rows = nn ? k : n;
    const AlignedRows xr = aligned_rows(x, m, k, 1, stream);
    const AlignedRows wr = aligned_rows(w, w_rows, w_cols, 1, stream);
    const uint32_t box[2] = {128, 128};
    const uint64_t w_dims[2] = {uint64_t(w_cols), uint64_t(w_rows)}, w_strides[1] = {uint64_t(wr.ld)};
    const uint64_t x_dims[2] = {uint64_t(k), uint64_t(m)}, x_strides[1] = {uint64_t(xr.ld)};
    const long long scale_cols = (w_cols + FP8_BLOCK - 1) / FP8_BLOCK;
    auto fill = [&](auto& p) {
        encode_tensor_map_u8(&p.map_w, wr.ptr, 2, w_dims, w_strides, box, TmaSwizzle::B128);
        p.x_scales = x_scales;
        p.w_scales = w_scales;
        p.ws_feature = nn ? 1 : scale_cols;
        p.ws_k = nn ? scale_cols : 1;
        p.bias = bias;
        p.act = act;
        p.c = y;
        p.rows = m;
        p.features = n;
        p.k = k;
    };
    if (m > FP8F_MAX_ROWS) {
        Fp8RowsParams p{};
        fill(p);
        encode_tensor_map_u8(&p.map_x, xr.ptr, 2, x_dims, x_strides, box, TmaSwizzle::B128);
        if (y_type == TYPE_F32) launch_by_rows<FORM, float>(p, stream);
        else if (y_type == TYPE_F16) launch_by_rows<FORM, __half>(p, stream);
        else launch_by_rows<FORM, __nv_bfloat16>(p, stream);
    } else {
        Fp8FewParams p{};
        fill(p);
        for (uint32_t i = 0; i < 5; ++i) {
            const uint32_t rows_box[2] = {128, i < 4 ? 32 * (i + 1) : 16};
            encode_tensor_map_u8(i < 4 ? &p.x.box[i] : &p.x.box16, xr.ptr, 2, x_dims, x_strides, rows_box, TmaSwizzle::B128);
        }
        if (y_type == TYPE_F32) launch_few<FORM, float>(p, stream);
        else if (y_type == TYPE_F16) launch_few<FORM, __half>(p, stream);
        else launch_few<FORM, __nv_bfloat16>(p, stream);
    }
}

}  // namespace

void fp8_nt(const uint8_t* x, const float* x_scales, const uint8_t* w, const float* w_scales, const float* bias, void* y,
            int y_type, int m, int n, int k, int act, cudaStream_t stream) {
    product<RaggedForm::NT>(x, x_scales, w, w_scales, bias, y, y_type, m, n, k, act, stream);
}

void fp8_nn(const uint8_t* dy, const float* dy_scales, const uint8_t* w, const float* w_scales, void* dx, int dx_type, int m,
            int n, int k, cudaStream_t stream) {
    product<RaggedForm::NN>(dy, dy_scales, w, w_scales, nullptr, dx, dx_type, m, k, n, 0, stream);
}

}  // namespace cudeep_b200
