// Launchers of the 8-bit products of fp8_gemm.cuh.
#include "fp8_gemm.h"

#include "fp8_gemm.cuh"
#include "ragged_plan.h"

namespace cudeep_b200 {

namespace {

template <RaggedForm FORM, int CTAS, class OutT>
void launch(Fp8Params& p, const RaggedPlan& plan, cudaStream_t stream) {
    const DeviceInfo& dev = device_info();
    CB200_REQUIRE(dev.cc_major == 10, "8-bit products need an sm_100 device");
    p.tile_cols = plan.tile_cols;
    p.stage_bytes = RAGGED_A_BYTES + uint32_t(plan.tile_cols / CTAS) * 128u;
    const int fit = int(FP8_SMEM_BUDGET / p.stage_bytes);
    p.stages = fit < RAGGED_MAX_STAGES ? fit : RAGGED_MAX_STAGES;
    p.status = dev.status_word;
    p.wait_limit_ns = 2000000000ull;
    long long clusters = dev.num_sms / CTAS;
    if (clusters > plan.units) clusters = plan.units;
    CB200_TRACE("fp8 %s tcgen05: rows=%d features=%d k=%d tile=%dx%d stages=%d clusters=%lld",
                FORM == RaggedForm::NT ? "nt" : "nn", p.rows, p.features, p.k, 128 * CTAS, plan.tile_cols, p.stages, clusters);
    launch_clusters(fp8_gemm_kernel<FORM, CTAS, OutT>, p, clusters, CTAS, FP8_THREADS,
                    uint32_t(p.stages) * p.stage_bytes + 1024, FP8_SMEM_BUDGET + 1024, stream);
}

template <RaggedForm FORM, class OutT>
void launch_out(Fp8Params& p, const RaggedPlan& plan, cudaStream_t stream) {
    if (plan.ctas == 2) launch<FORM, 2, OutT>(p, plan, stream);
    else launch<FORM, 1, OutT>(p, plan, stream);
}

// x[m, k] by w, stored [n, k] (NT: features n) or [k, n] (NN: features n).
template <RaggedForm FORM>
void product(const uint8_t* x, const float* x_scales, const uint8_t* w, const float* w_scales, const float* bias, void* y,
             int y_type, int m, int n, int k, int act, cudaStream_t stream) {
    constexpr bool nn = FORM == RaggedForm::NN;
    const int w_cols = nn ? n : k, w_rows = nn ? k : n;
    const AlignedRows xr = aligned_rows(x, m, k, 1, stream);
    const AlignedRows wr = aligned_rows(w, w_rows, w_cols, 1, stream);
    Fp8Params p{};
    {
        const uint64_t dims[3] = {uint64_t(w_cols), uint64_t(w_rows), 1};
        const uint64_t strides[2] = {uint64_t(wr.ld), uint64_t(wr.ld) * uint64_t(w_rows)};
        const uint32_t box[3] = {128, 128, 1};
        encode_tensor_map_u8(&p.map_a, wr.ptr, 3, dims, strides, box, TmaSwizzle::B128);
    }
    {
        const uint64_t dims[2] = {uint64_t(k), uint64_t(m)};
        const uint64_t strides[1] = {uint64_t(xr.ld)};
        const uint32_t box[2] = {128, 128}, box16[2] = {128, 16};
        encode_tensor_map_u8(&p.map_b, xr.ptr, 2, dims, strides, box, TmaSwizzle::B128);
        encode_tensor_map_u8(&p.map_b16, xr.ptr, 2, dims, strides, box16, TmaSwizzle::B128);
    }
    p.x_scales = x_scales;
    p.w_scales = w_scales;
    const long long scale_cols = (w_cols + FP8_BLOCK - 1) / FP8_BLOCK;
    p.ws_feature = nn ? 1 : scale_cols;
    p.ws_k = nn ? scale_cols : 1;
    p.bias = bias;
    p.act = act;
    p.c = y;
    p.groups = 1;
    p.rows = m;
    p.features = n;
    p.k = k;
    const RaggedPlan plan = plan_rows(1, m, n);
    if (y_type == TYPE_F32) launch_out<FORM, float>(p, plan, stream);
    else if (y_type == TYPE_F16) launch_out<FORM, __half>(p, plan, stream);
    else launch_out<FORM, __nv_bfloat16>(p, plan, stream);
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
