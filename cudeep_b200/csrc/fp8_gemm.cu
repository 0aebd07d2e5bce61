// Launchers of the 8-bit products of fp8_gemm.cuh.
#include "fp8_gemm.h"

#include "fp8_gemm.cuh"
#include "fp8_rows.cuh"
#include "fp8_scaled.cuh"
#include "ragged_plan.h"

#include <algorithm>

namespace cudeep_b200 {

namespace {

struct FewPlan {
    int step;       // features per tile
    int split;      // CTAs per tile, each with a range of K
    double cost;    // cycles
};

int few_clusters(int size) {
    return resident_clusters(reinterpret_cast<const void*>(fp8_few_kernel<RaggedForm::NT, float>), size, FP8F_THREADS,
                             FP8F_SMEM_BUDGET + 1024);
}

// The cheapest of all steps and splits by what an SM's stream of operands costs, in cycles: weights that one tile reads come
// from HBM, what several tiles read from L2; and fixed costs of a wave and of adding up a split tile.
FewPlan plan_few(int rows, int features, int k) {
    const int blocks = (k + FP8_BK - 1) / FP8_BK;
    const int row_tiles = (rows + FP8F_MAX_ROWS - 1) / FP8F_MAX_ROWS;
    const int tile_rows = rows < FP8F_MAX_ROWS ? rows : FP8F_MAX_ROWS;
    const int loaded = RowMaps::loaded((tile_rows + 15) / 16 * 16);
    FewPlan best{128, 1, 1e30};
    for (int step = 128; step >= 64; step -= 16) {
        for (int split = 1; split <= 8; split *= 2) {
            if (split > 1 && blocks < 4 * split) break;      // four blocks of K for each CTA at least
            const long long tiles = (long long)((features + step - 1) / step) * row_tiles, resident = few_clusters(split);
            const long long waves = (tiles + resident - 1) / resident;
            const double loads = step * 128 / (row_tiles == 1 ? PLAN_HBM_BYTES : PLAN_L2_BYTES) + loaded * 128 / PLAN_L2_BYTES;
            const double sums = 200.0 + 4.0 * tile_rows;      // taking a block's accumulators out
            const double cost = waves * ((blocks + split - 1) / split * std::max(loads, sums) + 4000.0 +
                                         (split > 1 ? 2000.0 + 20.0 * tile_rows : 0.0));
            if (cost < best.cost * 0.98) best = FewPlan{step, split, cost};
        }
    }
    return best;
}

template <RaggedForm FORM, class OutT>
void launch_few(Fp8FewParams& p, cudaStream_t stream) {
    const DeviceInfo& dev = device_info();
    CB200_REQUIRE(dev.cc_major == 10, "8-bit products need an sm_100 device");
    p.w_bytes = FORM == RaggedForm::NT ? uint32_t(p.step) * 128u : RAGGED_A_BYTES;
    p.tile_rows = p.rows < FP8F_MAX_ROWS ? p.rows : FP8F_MAX_ROWS;
    p.stage_bytes = RAGGED_A_BYTES + uint32_t(RowMaps::loaded((p.tile_rows + 15) / 16 * 16)) * 128u;
    const int fit = int(FP8F_SMEM_BUDGET / p.stage_bytes);
    p.stages = fit < FP8F_MAX_STAGES ? fit : FP8F_MAX_STAGES;
    p.status = dev.status_word;
    p.wait_limit_ns = 2000000000ull;
    p.f_tiles = (p.features + p.step - 1) / p.step;
    const long long tiles = (long long)p.f_tiles * ((p.rows + FP8F_MAX_ROWS - 1) / FP8F_MAX_ROWS);
    CB200_TRACE("fp8 %s tcgen05, features on lanes: rows=%d features=%d k=%d stages=%d tiles=%lld step=%d split=%d",
                FORM == RaggedForm::NT ? "nt" : "nn", p.rows, p.features, p.k, p.stages, tiles, p.step,
                p.split);
    launch_clusters(fp8_few_kernel<FORM, OutT>, p, tiles, p.split, FP8F_THREADS, uint32_t(p.stages) * p.stage_bytes + 1024,
                    FP8F_SMEM_BUDGET + 1024, stream);
}

template <class OutT, class Params>
void set_output(Params& p, uint32_t box_rows) {
    p.tma_store = (size_t(p.features) * sizeof(OutT)) % 16 == 0 && reinterpret_cast<uintptr_t>(p.c) % 16 == 0;
    if (!p.tma_store) return;
    const uint64_t dims[2] = {uint64_t(p.features), uint64_t(p.rows)};
    const uint64_t strides[1] = {uint64_t(p.features) * sizeof(OutT)};
    const uint32_t box[2] = {uint32_t(128 / sizeof(OutT)), box_rows};
    if (sizeof(OutT) == 4) encode_tensor_map(&p.map_c, static_cast<const float*>(p.c), 2, dims, strides, box, TmaSwizzle::B128);
    else encode_tensor_map_f16(&p.map_c, p.c, 2, dims, strides, box, TmaSwizzle::B128);
}

template <RaggedForm FORM, int BN, class OutT>
void launch_by_rows_bn(Fp8RowsParams& p, cudaStream_t stream) {
    const DeviceInfo& dev = device_info();
    CB200_REQUIRE(dev.cc_major == 10, "8-bit products need an sm_100 device");
    set_output<OutT>(p, 32);
    p.status = dev.status_word;
    p.wait_limit_ns = 2000000000ull;
    p.tiles_m = (p.rows + 255) / 256;
    p.tiles_n = (p.features + BN - 1) / BN;
    const long long tiles = (long long)p.tiles_m * p.tiles_n;
    const long long clusters = tiles < dev.num_sms / 2 ? tiles : dev.num_sms / 2;
    CB200_TRACE("fp8 %s tcgen05, rows on lanes: rows=%d features=%d k=%d tile=256x%d stages=%d clusters=%lld store=%s",
                FORM == RaggedForm::NT ? "nt" : "nn", p.rows, p.features, p.k, BN, FP8R_STAGES, clusters,
                p.tma_store ? "bulk-tensor" : "rows");
    launch_clusters(fp8_rows_kernel<FORM, BN, OutT>, p, clusters, 2, FP8R_THREADS, FP8R_SMEM_BYTES, FP8R_SMEM_BYTES, stream);
}

// The scales applied by the tensor core, and behind it fp8_rows.cuh's kernel, which runs if they were not all powers of two.
template <RaggedForm FORM, class OutT>
void launch_scaled(Fp8RowsParams& rows_form, cudaStream_t stream) {
    const DeviceInfo& dev = device_info();
    CB200_REQUIRE(dev.cc_major == 10, "8-bit products need an sm_100 device");
    Fp8ScaledParams p{};
    p.map_x = rows_form.map_x;
    p.map_w = rows_form.map_w;
    p.bias = rows_form.bias;
    p.act = rows_form.act;
    p.c = rows_form.c;
    p.rows = rows_form.rows;
    p.features = rows_form.features;
    p.k = rows_form.k;
    p.tiles_m = (p.rows + 255) / 256;
    p.tiles_n = (p.features + 255) / 256;
    p.chunk_blocks = sizeof(OutT) == 4 ? 2048 / FP8_BK : 16384 / FP8_BK;
    p.status = dev.status_word;
    p.wait_limit_ns = 2000000000ull;
    const int k_blocks = (p.k + FP8_BK - 1) / FP8_BK;
    const size_t x_words = size_t(k_blocks) * p.tiles_m * 2 * 128, w_words = size_t(k_blocks) * p.tiles_n * 2 * 128;
    Scratch packed((x_words + w_words + SCALE_FLAGS) * 4, stream);
    uint32_t* xs = static_cast<uint32_t*>(packed.ptr);
    uint32_t* ws = xs + x_words;
    uint32_t* odd = ws + w_words;
    p.odd_scales = rows_form.odd_scales = odd;
    const uint32_t xs_box[2] = {16, 32}, ws_box[2] = {16, 64};
    const uint64_t strides[1] = {16}, xs_dims[2] = {16, x_words / 4}, ws_dims[2] = {16, w_words / 4};
    encode_tensor_map_u8(&p.map_xs, xs, 2, xs_dims, strides, xs_box, TmaSwizzle::None);
    encode_tensor_map_u8(&p.map_ws, ws, 2, ws_dims, strides, ws_box, TmaSwizzle::None);
    launch_dependent(pack_scales_kernel, dim3(SCALE_FLAGS), 256, stream, rows_form.x_scales, p.rows, 2 * p.tiles_m,
                     rows_form.w_scales, (p.features + 127) / 128, 2 * p.tiles_n, rows_form.ws_feature, rows_form.ws_k, k_blocks, xs,
                     ws, odd);
    set_output<OutT>(p, 16);
    const long long tiles = (long long)p.tiles_m * p.tiles_n;
    const long long clusters = tiles < dev.num_sms / 2 ? tiles : dev.num_sms / 2;
    CB200_TRACE("fp8 %s tcgen05, scales in the MMA: rows=%d features=%d k=%d tile=256x256 stages=%d clusters=%lld store=%s",
                FORM == RaggedForm::NT ? "nt" : "nn", p.rows, p.features, p.k, FP8S_STAGES, clusters,
                p.tma_store ? "bulk-tensor" : "rows");
    launch_clusters(fp8_scaled_kernel<FORM, OutT>, p, clusters, 2, FP8R_THREADS, FP8S_SMEM_BYTES, FP8S_SMEM_BYTES, stream);
    launch_by_rows_bn<FORM, 256, OutT>(rows_form, stream);
}

// Tiles of 256 rows x 256 features; of 128 features where even those do not outnumber the pairs of SMs.
bool narrow_tiles(int m, int n) {
    return (long long)((m + 255) / 256) * ((n + 127) / 128) <= device_info().num_sms / 2;
}

// Cycles of the product with the rows on the lanes, as plan_few counts them: a block's 32 KB of operands, or 24 KB of a
// narrow tile's, and the sums of a finished tile, which nothing hides.
double cost_by_rows(int m, int n, int k, bool narrow) {
    const int blocks = (k + FP8_BK - 1) / FP8_BK, pairs = device_info().num_sms / 2;
    const long long tiles = (long long)((m + 255) / 256) * (narrow ? (n + 127) / 128 : (n + 255) / 256);
    const double waves = double((tiles + pairs - 1) / pairs);
    return waves * (blocks * (narrow ? 24576.0 : 32768.0) / PLAN_L2_BYTES + (narrow ? 1500.0 : 3000.0)) + 4000.0;
}

// Packing the scales and a kernel that finds nothing to do cost about 5 us, which products of an estimated 50000 cycles and more
// make good: 2048 x 4096 x 4096 (61000) takes 35.3 us so and 36.9 by rows, 4096 x 1024 -> 8192 (70000) 37.0 and 40.8, but
// 2047 x 5000 -> 1672 (39000) 38.3 and 35.0.
constexpr double SCALED_FROM_CYCLES = 50000.0;

template <RaggedForm FORM, class OutT>
void launch_by_rows(Fp8RowsParams& p, bool narrow, bool scaled, cudaStream_t stream) {
    if (scaled) return launch_scaled<FORM, OutT>(p, stream);
    if constexpr (FORM == RaggedForm::NT) {
        if (narrow) return launch_by_rows_bn<FORM, 128, OutT>(p, stream);
    }
    launch_by_rows_bn<FORM, 256, OutT>(p, stream);
}

// x[m, k] by w, stored [n, k] (NT: features n) or [k, n] (NN: features n).
template <RaggedForm FORM>
void product(const uint8_t* x, const float* x_scales, const uint8_t* w, const float* w_scales, const float* bias, void* y,
             int y_type, int m, int n, int k, int act, cudaStream_t stream) {
    constexpr bool nn = FORM == RaggedForm::NN;
    const int w_cols = nn ? n : k, w_rows = nn ? k : n;
    const PreparedRows operands = prepare_rows({x, m, k, 1}, {w, w_rows, w_cols, 1}, {}, stream);
    const AlignedRows &xr = operands.a, &wr = operands.b;
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
    const bool narrow = !nn && narrow_tiles(m, n);
    const FewPlan few = plan_few(m, n, k);
    const double rows_cost = cost_by_rows(m, n, k, narrow);
    if (m > FP8F_MAX_ROWS && rows_cost < few.cost) {
        const bool scaled = !narrow && rows_cost >= SCALED_FROM_CYCLES;
        Fp8RowsParams p{};
        fill(p);
        encode_tensor_map_u8(&p.map_x, xr.ptr, 2, x_dims, x_strides, box, TmaSwizzle::B128);
        if (narrow) {
            const uint32_t w_box[2] = {128, 64};
            encode_tensor_map_u8(&p.map_w, wr.ptr, 2, w_dims, w_strides, w_box, TmaSwizzle::B128);
        }
        if (y_type == TYPE_F32) launch_by_rows<FORM, float>(p, narrow, scaled, stream);
        else if (y_type == TYPE_F16) launch_by_rows<FORM, __half>(p, narrow, scaled, stream);
        else launch_by_rows<FORM, __nv_bfloat16>(p, narrow, scaled, stream);
    } else {
        Fp8FewParams p{};
        fill(p);
        p.step = few.step;
        p.split = few.split;
        if (!nn) {
            const uint32_t w_box[2] = {128, uint32_t(few.step)};
            encode_tensor_map_u8(&p.map_w, wr.ptr, 2, w_dims, w_strides, w_box, TmaSwizzle::B128);
        }
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
