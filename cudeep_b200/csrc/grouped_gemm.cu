// Launchers of the ragged products of ragged_gemm.cuh.
#include "grouped_gemm.h"

#include "ragged_gemm.cuh"
#include "ragged_plan.h"

#include <type_traits>

namespace cudeep_b200 {

namespace {

// Copies of two maps for each group (one warp each), cut off at the group's last row (their dimension 1).
__global__ void __launch_bounds__(32) group_maps_kernel(const __grid_constant__ CUtensorMap map_a,
                                                        const __grid_constant__ CUtensorMap map_b,
                                                        const int32_t* __restrict__ offsets, int rows, CUtensorMap* out) {
#if defined(__CUDA_ARCH_FEAT_SM100_ALL) || defined(__CUDA_ARCH_FEAT_SM101_ALL) || \
    defined(__CUDA_ARCH_FEAT_SM103_ALL)
    __shared__ __align__(128) uint32_t copy[2][32];
    const uint32_t lane = threadIdx.x;
    copy[0][lane] = reinterpret_cast<const uint32_t*>(&map_a)[lane];
    copy[1][lane] = reinterpret_cast<const uint32_t*>(&map_b)[lane];
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    __syncwarp();
    // An empty group loads nothing; its map only has to be a map.
    const uint32_t end = uint32_t(min(max(__ldg(offsets + blockIdx.x + 1), 1), rows));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (lane == 0) ptx::tensormap_replace_dim1(ptx::smem_u32(copy[i]), end);
        __syncwarp();
        ptx::tensormap_publish(out + 2 * blockIdx.x + i, ptx::smem_u32(copy[i]));
    }
#endif
}

template <RaggedForm FORM, int CTAS, bool BF16, class OutT, bool WIDE = false>
void launch(RaggedParams& p, const RaggedPlan& plan, cudaStream_t stream) {
    const DeviceInfo& dev = device_info();
    CB200_REQUIRE(dev.cc_major == 10, "grouped products need an sm_100 device");
    p.tile_cols = plan.tile_cols;
    p.atom_bytes = RAGGED_A_BYTES + uint32_t(RowMaps::loaded(plan.tile_cols / CTAS)) * 128u;
    const uint32_t fixed = (FORM == RaggedForm::TN ? RAGGED_STAGING_BYTES : 0u) + ragged_table_bytes(p.groups);
    // As many K blocks to a stage, and so to a barrier, as leave three stages; more than two gain nothing.
    p.atoms = int((RAGGED_SMEM_BUDGET - fixed) / 3 / p.atom_bytes);
    p.atoms = p.atoms < 1 ? 1 : p.atoms > 2 ? 2 : p.atoms;
    p.stage_bytes = p.atoms * p.atom_bytes;
    const int fit = int((RAGGED_SMEM_BUDGET - fixed) / p.stage_bytes);
    p.stages = fit < RAGGED_MAX_STAGES ? fit : RAGGED_MAX_STAGES;
    p.status = dev.status_word;
    p.wait_limit_ns = 2000000000ull;
    p.split = plan.split;
    p.chunk_rows = std::is_same<OutT, float>::value ? RAGGED_F32_TERMS : RAGGED_F16_TERMS;
    p.chunk_blocks = RAGGED_F16_TERMS / RAGGED_BK;
    long long clusters = plan.split > 1 ? plan.units : dev.num_sms / CTAS;
    if (clusters > plan.units) clusters = plan.units;
    const uint32_t smem_bytes = uint32_t(p.stages) * p.stage_bytes + fixed + 1024;
    const long long terms = FORM != RaggedForm::TN ? (p.k + plan.split - 1) / plan.split : WIDE ? 2ll * p.part_rows : p.rows;
    Scratch partial;
    if (sizeof(OutT) == 2 && terms > RAGGED_F16_TERMS) {
        partial = Scratch(size_t(clusters) * CTAS * plan.split * RAGGED_PARTIAL_FLOATS * sizeof(float), stream);
        p.partial = static_cast<float*>(partial.ptr);
    }
    CB200_TRACE("grouped %s %s tcgen05: rows=%d groups=%d features=%d %s=%d tile=%dx%d split=%d stages=%d clusters=%lld",
                FORM == RaggedForm::NT ? "nt" : FORM == RaggedForm::NN ? "nn" : "tn", BF16 ? "bf16" : "f16", p.rows, p.groups,
                p.features, FORM == RaggedForm::TN ? "cols" : "k", FORM == RaggedForm::TN ? p.cols : p.k, 128 * CTAS,
                plan.tile_cols, plan.split, p.stages, clusters);
    auto run = [&](auto kernel) {
        launch_clusters(kernel, p, clusters, CTAS * plan.split, RAGGED_THREADS, smem_bytes, RAGGED_SMEM_BUDGET + 1024, stream);
    };
    if constexpr (sizeof(OutT) == 2) {
        if (p.partial != nullptr) return run(ragged_gemm_kernel<FORM, CTAS, BF16, OutT, WIDE, true>);
    }
    run(ragged_gemm_kernel<FORM, CTAS, BF16, OutT, WIDE>);
}

template <RaggedForm FORM>
void launch_rows(RaggedParams& p, const RaggedPlan& plan, int type, cudaStream_t stream) {
    if (type == TYPE_BF16) {
        if (plan.ctas == 2) launch<FORM, 2, true, __nv_bfloat16>(p, plan, stream);
        else launch<FORM, 1, true, __nv_bfloat16>(p, plan, stream);
    } else {
        if (plan.ctas == 2) launch<FORM, 2, false, __half>(p, plan, stream);
        else launch<FORM, 1, false, __half>(p, plan, stream);
    }
}

void rows_by_weight(bool nn, const void* a, long long lda, const void* w, long long ldw, void* c, int type, const int32_t* offsets,
                    int groups, int rows, int n, int k, cudaStream_t stream) {
    const int w_cols = nn ? n : k, w_rows = nn ? k : n;
    const PreparedRows operands = prepare_rows({a, rows, k, 2, lda}, {w, (long long)groups * w_rows, w_cols, 2, ldw, offsets, w_rows},
                                               {}, stream);
    const AlignedRows &x = operands.a, &wt = operands.b;
    const RaggedPlan plan = plan_rows(groups, rows, n, (k + RAGGED_BK - 1) / RAGGED_BK, nn ? 128 : 64, [](int size) {
        return resident_clusters(reinterpret_cast<const void*>(ragged_gemm_kernel<RaggedForm::NT, 1, true, __nv_bfloat16>), size,
                                 RAGGED_THREADS, RAGGED_SMEM_BUDGET + 1024);
    });
    RaggedParams p{};
    p.step = plan.step;
    {
        const uint64_t row_bytes = uint64_t(wt.ld) * 2, group_bytes = row_bytes * uint64_t(w_rows);
        p.a_chunked = nn && wt.ld >= (w_cols + 63) / 64 * 64;
        if (p.a_chunked) {
            const uint64_t dims[4] = {64, uint64_t(w_rows), uint64_t((w_cols + 63) / 64), uint64_t(groups)};
            const uint64_t strides[3] = {row_bytes, 128, group_bytes};
            const uint32_t box[4] = {64, 64, 2, 1};
            encode_tensor_map_f16(&p.map_a, wt.ptr, 4, dims, strides, box, TmaSwizzle::B128);
        } else {
            const uint64_t dims[3] = {uint64_t(w_cols), uint64_t(w_rows), uint64_t(groups)};
            const uint64_t strides[2] = {row_bytes, group_bytes};
            const uint32_t box[3] = {64, nn ? 64u : uint32_t(plan.step), 1};
            encode_tensor_map_f16(&p.map_a, wt.ptr, 3, dims, strides, box, TmaSwizzle::B128);
        }
    }
    {
        const uint64_t dims[2] = {uint64_t(k), uint64_t(rows)};
        const uint64_t strides[1] = {uint64_t(x.ld) * 2};
        for (uint32_t i = 0; i < 5; ++i) {
            const uint32_t box[2] = {64, i < 4 ? 32 * (i + 1) : 16};
            encode_tensor_map_f16(i < 4 ? &p.x.box[i] : &p.x.box16, x.ptr, 2, dims, strides, box, TmaSwizzle::B128);
        }
    }
    p.c = c;
    p.offsets = offsets;
    p.groups = groups;
    p.rows = rows;
    p.share = rows;
    p.features = n;
    p.k = k;
    if (nn) launch_rows<RaggedForm::NN>(p, plan, type, stream);
    else launch_rows<RaggedForm::NT>(p, plan, type, stream);
}

// The map of load_columns; returns whether it is by chunks.
int encode_columns(CUtensorMap* map, const AlignedRows& m, int rows, int cols, int chunks) {
    const bool chunked = m.ld >= (cols + 63) / 64 * 64;
    const uint64_t dims[2] = {uint64_t(cols), uint64_t(rows)}, strides[1] = {uint64_t(m.ld) * 2};
    const uint64_t dims3[3] = {64, uint64_t(rows), uint64_t((cols + 63) / 64)}, strides3[2] = {uint64_t(m.ld) * 2, 128};
    const uint32_t box[3] = {64, 64, uint32_t(chunks)};
    if (chunked) encode_tensor_map_f16(map, m.ptr, 3, dims3, strides3, box, TmaSwizzle::B128);
    else encode_tensor_map_f16(map, m.ptr, 2, dims, strides, box, TmaSwizzle::B128);
    return chunked ? 1 : 0;
}

template <int CTAS, bool BF16, bool WIDE = false>
void launch_weight(RaggedParams& p, const RaggedPlan& plan, int c_type, cudaStream_t stream) {
    if (c_type == TYPE_F32) launch<RaggedForm::TN, CTAS, BF16, float, WIDE>(p, plan, stream);
    else if constexpr (BF16) launch<RaggedForm::TN, CTAS, BF16, __nv_bfloat16>(p, plan, stream);
    else launch<RaggedForm::TN, CTAS, BF16, __half, WIDE>(p, plan, stream);
}

}  // namespace

void grouped_nt(const void* a, const void* w, void* c, int type, const int32_t* offsets, int groups, int rows, int n, int k,
                cudaStream_t stream) {
    rows_by_weight(false, a, 0, w, 0, c, type, offsets, groups, rows, n, k, stream);
}

void grouped_nn(const void* a, long long lda, const void* w, long long ldw, void* c, int type, const int32_t* offsets, int groups,
                int rows, int n, int k, cudaStream_t stream) {
    rows_by_weight(true, a, lda, w, ldw, c, type, offsets, groups, rows, n, k, stream);
}

void grouped_tn(const void* a, long long lda, const void* b, long long ldb, void* c, int type, int c_type,
                const int32_t* offsets, int groups, int rows, int m, int n, const float* col_scale, const WideOperands& wide,
                cudaStream_t stream) {
    const PreparedRows operands = prepare_rows({a, rows, m, 2, lda}, {b, rows, n, 2, ldb}, {}, stream);
    const AlignedRows &y = operands.a, &x = operands.b;
    RaggedPlan plan = plan_weight(groups, rows, m, n, elem_bytes(c_type));
    // One gradient of few tiles and many rows: `parts` ranges of the rows as groups of their own, summed in FP32 and added up
    // in order by a pass of their own (8192 rows, 512 x 512: 50 us in one range, 18 us so).
    int parts = 1;
    if (offsets == nullptr) {
        for (int p = 2; p <= 16 && rows >= 512 * p; p *= 2) {
            RaggedPlan split = plan_weight(p, rows, m, n, 4);
            split.cost += 5000.0 + 8.0 * p * m * n / (device_info().num_sms * PLAN_HBM_BYTES);
            if (split.cost < 0.95 * plan.cost) {
                plan = split;
                parts = p;
            }
        }
    }
    Scratch sums;
    void* out = c;
    int out_type = c_type;
    long long ldc = n;
    if (parts > 1) {
        ldc = (n + 3) / 4 * 4;
        sums = Scratch(size_t(parts) * m * ldc * sizeof(float), stream);
        out = sums.ptr;
        out_type = TYPE_F32;
    }
    RaggedParams p{};
    p.groups = parts > 1 ? parts : groups;
    p.share = parts > 1 ? ((rows + parts - 1) / parts + RAGGED_BK - 1) / RAGGED_BK * RAGGED_BK : rows;
    p.step = 128;
    p.a_chunked = encode_columns(&p.map_a, y, rows, m, 2);
    p.b_chunked = encode_columns(&p.map_b, x, rows, n, plan.tile_cols / plan.ctas / 64);
    if (wide.wide != nullptr) {
        CB200_REQUIRE(type == TYPE_F16 && offsets == nullptr, "operands in two parts: FP16, one group");
        p.wide = wide.wide;
        p.wide_blocks = wide.blocks;
        p.part_rows = (rows + RAGGED_BK - 1) / RAGGED_BK * RAGGED_BK;
        p.wide_share = parts > 1 ? 2 * p.share : 2 * p.part_rows;
        const uint64_t row_bytes = uint64_t(wide.ld_parts) * 2;
        const uint64_t dims[4] = {64, uint64_t(rows), uint64_t((m + 63) / 64), 2};
        const uint64_t strides[3] = {row_bytes, 128, row_bytes * uint64_t(rows)};
        const uint32_t box[4] = {64, 64, 2, 1};
        encode_tensor_map_f16(&p.map_parts, wide.parts, 4, dims, strides, box, TmaSwizzle::B128);
    }
    const uint32_t c_bytes = uint32_t(elem_bytes(out_type));
    p.tma_store = (size_t(ldc) * c_bytes) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
    if (p.tma_store) {
        const uint64_t dims[3] = {uint64_t(n), uint64_t(m), uint64_t(p.groups)};
        const uint64_t strides[2] = {uint64_t(ldc) * c_bytes, uint64_t(ldc) * c_bytes * uint64_t(m)};
        const uint32_t box[3] = {128 / c_bytes, 32, 1};
        if (out_type == TYPE_F32) encode_tensor_map(&p.map_c, static_cast<const float*>(out), 3, dims, strides, box, TmaSwizzle::B128);
        else encode_tensor_map_f16(&p.map_c, out, 3, dims, strides, box, TmaSwizzle::B128);
    }
    Scratch maps;
    if (offsets != nullptr) {
        maps = Scratch(size_t(groups) * 2 * sizeof(CUtensorMap), stream);
        p.group_maps = static_cast<const CUtensorMap*>(maps.ptr);
        launch_dependent(group_maps_kernel, dim3(unsigned(groups)), 32, stream, p.map_a, p.map_b, offsets, rows,
                         static_cast<CUtensorMap*>(maps.ptr));
    }
    p.c = out;
    p.ldc = ldc;
    p.offsets = offsets;
    p.rows = rows;
    p.features = m;
    p.cols = n;
    p.col_scale = col_scale;
    const bool pairs = plan.ctas == 2;
    if (type == TYPE_BF16) {
        if (pairs) launch_weight<2, true>(p, plan, out_type, stream);
        else launch_weight<1, true>(p, plan, out_type, stream);
    } else if (wide.wide != nullptr) {
        if (pairs) launch_weight<2, false, true>(p, plan, out_type, stream);
        else launch_weight<1, false, true>(p, plan, out_type, stream);
    } else {
        if (pairs) launch_weight<2, false>(p, plan, out_type, stream);
        else launch_weight<1, false>(p, plan, out_type, stream);
    }
    if (parts > 1) add_parts(static_cast<const float*>(out), parts, m, n, ldc, c, c_type, stream);
}

}  // namespace cudeep_b200
