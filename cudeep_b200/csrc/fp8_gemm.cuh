// Products of 8-bit (e4m3) matrices with a scale per block of 128, FP32 accumulation (tcgen05 kind::f8f6f4).
//
//   NT  C[r, f] = sum_b xs[b][r] ws[f / 128][b] ( sum_{k in block b} X[r, k] W[f, k] )     y = x W^T
//   NN  C[r, f] = sum_b xs[b][r] ws[b][f / 128] ( sum_{k in block b} X[r, k] W[k, f] )     dx = dy W
//
// A scale changes with every block of 128 along the sum, so the tensor core may only sum within one block: each K block
// (128 bytes per row, four MMAs of K = 32) is multiplied into a fresh TMEM accumulator, and eight epilogue warps take it
// out and add it, scaled, to sums that they hold in registers (two FP32 lanes per fma.rn.f32x2).  Those sums round to
// nearest, so the length of K costs no accuracy beyond FP32's.  Two accumulators alternate: while one is drained, the
// tensor core fills the other.
//
// As in the ragged products the FEATURES lie on the 128 lanes of a CTA and the rows on the columns: a CTA's features
// are one block of W's scales, a scalar, and the width of the MMA follows the number of rows, so that a handful of
// rows costs the weight's bytes and little else.
#pragma once

#include "ragged_gemm.cuh"

namespace cudeep_b200 {

constexpr int FP8_BK = 128;                     // elements per K block = one 128-byte swizzle row = one scale
constexpr int FP8_EPI_WARPS = 8;
constexpr int FP8_THREADS = 64 + 32 * FP8_EPI_WARPS;
constexpr uint32_t FP8_SMEM_BUDGET = 232448 - 1024 - 22 * 1024;   // minus alignment slack, group tables, scales, barriers

struct Fp8Params {
    CUtensorMap map_a;       // NT {K, F, G} box {128, 128, 1}; NN {F, K, G} box {128, 128, 1}
    RowMaps x;               // {K, rows}
    const float* x_scales;   // [K blocks][rows]
    const float* w_scales;   // + group * ws_group + feature block * ws_feature + K block * ws_k
    long long ws_group, ws_feature, ws_k;
    const float* bias;       // [F] or nullptr
    int act;
    void* c;
    const int32_t* offsets;
    int groups;
    int rows;
    int features;
    int k;
    int tile_cols;
    int stages;
    uint32_t stage_bytes;
    uint32_t* status;
    unsigned long long wait_limit_ns;
};

// (d0, d1) += (a0, a1) * (s0, s1)
__device__ __forceinline__ void fma2(float& d0, float& d1, uint32_t a0, uint32_t a1, float s0, float s1) {
    asm("{\n\t"
        ".reg .b64 a, s, d;\n\t"
        "mov.b64 a, {%2, %3};\n\t"
        "mov.b64 s, {%4, %5};\n\t"
        "mov.b64 d, {%0, %1};\n\t"
        "fma.rn.f32x2 d, a, s, d;\n\t"
        "mov.b64 {%0, %1}, d;\n\t"
        "}\n"
        : "+f"(d0), "+f"(d1) : "r"(a0), "r"(a1), "f"(s0), "f"(s1));
}

// The epilogue's activations as one formula, y = g * sigmoid(a z + b z^3), g = z (GELU in its tanh form, SiLU) or 1
// (sigmoid), with log2(e) folded into a and b.  Two values share one reciprocal, 1 / d0 = d1 / (d0 d1): the SFU is what bounds
// an epilogue that activates 128 values a thread, and this takes three of its operations per pair instead of four.  The
// exponents are held below 60 so that d0 d1 stays finite (sigmoid = 2^-60 there instead of less).
struct Fp8Activation {
    int act;
    float a, b;
    __device__ __forceinline__ explicit Fp8Activation(int act_) : act(act_) {
        const float c = act == EPI_GELU ? 2.0f * 0.7978845608028654f : 1.0f;
        a = -1.4426950408889634f * c;
        b = act == EPI_GELU ? a * 0.044715f : 0.0f;
    }
};

__device__ __forceinline__ void fp8_activation(float (&v)[32], const Fp8Activation& f) {
    if (f.act == EPI_NONE) return;
    if (f.act == EPI_RELU) {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = fmaxf(v[j], 0.0f);
        return;
    }
    const bool gate = f.act != EPI_SIGMOID;
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
        const float x0 = v[j], x1 = v[j + 1];
        const float d0 = 1.0f + sfu_ex2(fminf(x0 * fmaf(f.b, x0 * x0, f.a), 60.0f));
        const float d1 = 1.0f + sfu_ex2(fminf(x1 * fmaf(f.b, x1 * x1, f.a), 60.0f));
        const float r = sfu_rcp(d0 * d1);
        v[j] = (gate ? x0 : 1.0f) * (d1 * r);
        v[j + 1] = (gate ? x1 : 1.0f) * (d0 * r);
    }
}

template <RaggedForm FORM, int CTAS, class OutT>
__global__ void __launch_bounds__(FP8_THREADS, 1) fp8_gemm_kernel(const __grid_constant__ Fp8Params p) {
#if defined(__CUDA_ARCH_FEAT_SM100_ALL) || defined(__CUDA_ARCH_FEAT_SM101_ALL) || \
    defined(__CUDA_ARCH_FEAT_SM103_ALL)
    static_assert(FORM != RaggedForm::TN, "rows are not summed over in 8 bits");
    constexpr bool A_MN = FORM == RaggedForm::NN;

    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bar_full[RAGGED_MAX_STAGES];
    __shared__ __align__(8) uint64_t bar_empty[RAGGED_MAX_STAGES];
    __shared__ __align__(8) uint64_t bar_acc_full[2];
    __shared__ __align__(8) uint64_t bar_acc_empty[2];
    __shared__ __align__(16) float scale_buf[FP8_EPI_WARPS][2][128];
    __shared__ uint32_t tmem_base_holder;
    __shared__ uint32_t abort_flag;
    __shared__ int group_rows[2 * RAGGED_MAX_GROUPS];
    __shared__ int group_start[RAGGED_MAX_GROUPS + 1];

    const uint32_t warp = threadIdx.x >> 5;
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t cta_rank = CTAS == 2 ? ptx::cluster_ctarank() : 0u;
    const bool is_leader = cta_rank == 0;
    const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    ptx::WaitCtx wctx{&abort_flag, p.status, p.wait_limit_ns};

    if (threadIdx.x == 0) {
        abort_flag = 0;
        ptx::prefetch_tensormap(&p.map_a);
        p.x.prefetch();
        for (int s = 0; s < RAGGED_MAX_STAGES; ++s) {
            ptx::mbar_init(ptx::smem_u32(&bar_full[s]), CTAS);
            ptx::mbar_init(ptx::smem_u32(&bar_empty[s]), 1);
        }
        for (int a = 0; a < 2; ++a) {
            ptx::mbar_init(ptx::smem_u32(&bar_acc_full[a]), 1);
            ptx::mbar_init(ptx::smem_u32(&bar_acc_empty[a]), FP8_EPI_WARPS * CTAS);
        }
        ptx::fence_mbar_init();
    }
    if (warp == 1) {
        ptx::tmem_alloc<CTAS>(ptx::smem_u32(&tmem_base_holder), 512);
        ptx::tmem_relinquish<CTAS>();
    }
    ptx::grid_dependency_wait();
    const int f_tiles = (p.features + 128 * CTAS - 1) / (128 * CTAS);
    if (warp == 0) group_tables(p.offsets, p.groups, p.rows, f_tiles, -p.tile_cols, group_rows, group_start, p.status);
    ptx::tc_fence_before();
    __syncthreads();
    if (CTAS == 2) {
        ptx::cluster_arrive();
        ptx::cluster_wait();
    }
    ptx::tc_fence_after();
    const uint32_t tmem_base = tmem_base_holder;
    ptx::grid_launch_dependents();

    const int unit_stride = gridDim.x / CTAS;
    const int first_unit = blockIdx.x / CTAS;
    RaggedWalk<FORM, CTAS> walk{group_rows, group_start, p.groups, f_tiles, 0, p.tile_cols, p.features, 0};
    const int num_units = walk.total();
    const int k_blocks = (p.k + FP8_BK - 1) / FP8_BK;

    if (warp == 0) {
        // ------------------------------------------------------------ producer
        if (lane == 0) {
            uint32_t stage = 0, phase = 0;
            for (int u = first_unit; u < num_units; u += unit_stride) {
                const RaggedTile t = walk.at(u);
                const int per = t.umma_n / CTAS;
                const int feature = t.feature0 + int(cta_rank) * 128;
                const int col = t.col0 + int(cta_rank) * per;
                const uint32_t bytes = RAGGED_A_BYTES + uint32_t(RowMaps::loaded(per)) * 128u;
                for (int kb = 0; kb < k_blocks; ++kb) {
                    if (!ptx::mbar_wait(ptx::smem_u32(&bar_empty[stage]), phase ^ 1u, wctx, UMMA_TIMEOUT_PRODUCER))
                        goto producer_done;
                    const uint32_t a_smem = smem_base + stage * p.stage_bytes;
                    const uint32_t b_smem = a_smem + RAGGED_A_BYTES;
                    const uint32_t full_local = ptx::smem_u32(&bar_full[stage]);
                    const uint32_t full = CTAS == 2 ? ptx::mapa(full_local, 0) : full_local;
                    if (is_leader) ptx::mbar_arrive_expect_tx(full_local, bytes);
                    else ptx::mbar_arrive_expect_tx_cluster_relaxed(full, bytes);
                    const int k0 = kb * FP8_BK;
                    const int ax = A_MN ? feature : k0, ay = A_MN ? k0 : feature;
                    if constexpr (CTAS == 2) ptx::tma_load_3d_pair(a_smem, &p.map_a, full, ax, ay, t.group);
                    else ptx::tma_load_3d(a_smem, &p.map_a, full, ax, ay, t.group);
                    p.x.template load<CTAS>(b_smem, full, k0, col, per);
                    if (++stage == uint32_t(p.stages)) { stage = 0; phase ^= 1u; }
                }
            }
        }
    producer_done:
        __syncwarp();
        if (CTAS == 2) ptx::cluster_arrive();
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer
        if (is_leader) {
            // K-major: one MMA (K = 32) is 32 bytes along the row.  Features along the row (NN): 32 rows of 128 bytes.
            constexpr uint32_t A_KSTEP = A_MN ? 4096u : 32u;
            const uint64_t a_desc0 = ptx::smem_desc_at(ptx::smem_desc(A_MN ? 16384 : 16, 1024, ptx::SMEM_LAYOUT_SW128), smem_base);
            const uint64_t b_desc0 =
                ptx::smem_desc_at(ptx::smem_desc(16, 1024, ptx::SMEM_LAYOUT_SW128), smem_base + RAGGED_A_BYTES);
            uint32_t stage = 0, phase = 0;
            uint32_t it = 0;
            for (int u = first_unit; u < num_units; u += unit_stride) {
                const RaggedTile t = walk.at(u);
                const uint32_t idesc = ptx::idesc_e4m3(128 * CTAS, t.umma_n, A_MN ? 1 : 0, 0);
                bool ready = __all_sync(0xffffffffu, ptx::mbar_test(ptx::smem_u32(&bar_full[stage]), phase));
                for (int kb = 0; kb < k_blocks; ++kb, ++it) {
                    const uint32_t acc = it & 1;
                    if (!__all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&bar_acc_empty[acc]), ((it >> 1) & 1) ^ 1u,
                                                                wctx, UMMA_TIMEOUT_MMA_ACC)))
                        goto mma_done;
                    if (!ready && !__all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&bar_full[stage]), phase, wctx,
                                                                          UMMA_TIMEOUT_MMA_FULL)))
                        goto mma_done;
                    ptx::tc_fence_after();
                    uint32_t next_stage = stage + 1, next_phase = phase;
                    if (next_stage == uint32_t(p.stages)) { next_stage = 0; next_phase ^= 1u; }
                    ready = __all_sync(0xffffffffu, ptx::mbar_test(ptx::smem_u32(&bar_full[next_stage]), next_phase));
                    if (ptx::elect_one()) {
                        const uint32_t d_tmem = tmem_base + acc * 256u;
                        const uint64_t a_stage = a_desc0 + ((stage * p.stage_bytes) >> 4);
                        const uint64_t b_stage = b_desc0 + ((stage * p.stage_bytes) >> 4);
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            ptx::umma_f8<CTAS>(d_tmem, a_stage + ((kk * A_KSTEP) >> 4), b_stage + ((kk * 32u) >> 4), idesc,
                                               kk != 0);
                        const uint32_t empty_local = ptx::smem_u32(&bar_empty[stage]);
                        ptx::umma_commit<CTAS>(empty_local);
                        if constexpr (CTAS == 2) ptx::umma_commit<CTAS>(ptx::mapa(empty_local, 1));
                        const uint32_t accf_local = ptx::smem_u32(&bar_acc_full[acc]);
                        ptx::umma_commit<CTAS>(accf_local);
                        if constexpr (CTAS == 2) ptx::umma_commit<CTAS>(ptx::mapa(accf_local, 1));
                    }
                    __syncwarp();
                    stage = next_stage;
                    phase = next_phase;
                }
            }
        }
    mma_done:
        __syncwarp();
        if (CTAS == 2) ptx::cluster_arrive();
    } else {
        // ------------------------------------------------------------ sums and epilogue
        // Warps 2..5 take the first half of the columns, 6..9 the second; each its quarter of the lanes.
        const uint32_t quarter = warp & 3u;
        const int half = int(warp - 2) >> 2;
        float* my_scales = &scale_buf[warp - 2][0][0];
        uint32_t it = 0;
        for (int u = first_unit; u < num_units; u += unit_stride) {
            const RaggedTile t = walk.at(u);
            const int cta_feature = t.feature0 + int(cta_rank) * 128;
            const int feature = cta_feature + int(quarter) * 32 + int(lane);
            const int half_cols = (t.umma_n / 2 + 15) / 16 * 16;
            const int c_begin = half * half_cols;
            const int c_count = min(half_cols, t.umma_n - c_begin);
            const float* xs = p.x_scales + t.col0 + c_begin;
            // A CTA of a pair whose features all lie outside has no block of scales.
            const float* ws = p.w_scales + t.group * p.ws_group + (cta_feature < p.features ? cta_feature / 128 : 0) * p.ws_feature;
            float pre[4], pre_w;
            auto fetch = [&](int kb) {
                pre_w = __ldg(ws + kb * p.ws_k);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int c = int(lane) + 32 * i;
                    pre[i] = c < c_count && t.col0 + c_begin + c < p.rows ? __ldg(xs + (long long)kb * p.rows + c) : 0.0f;
                }
            };
            float acc[4][32];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 32; ++j) acc[i][j] = 0.0f;
            fetch(0);
            for (int kb = 0; kb < k_blocks; ++kb, ++it) {
                float* s = my_scales + (kb & 1) * 128;
#pragma unroll
                for (int i = 0; i < 4; ++i) s[lane + 32 * i] = pre[i] * pre_w;
                __syncwarp();
                if (kb + 1 < k_blocks) fetch(kb + 1);
                const uint32_t buf = it & 1;
                const bool ok = ptx::mbar_wait(ptx::smem_u32(&bar_acc_full[buf]), (it >> 1) & 1, wctx, UMMA_TIMEOUT_EPILOGUE);
                if (!__all_sync(0xffffffffu, ok)) goto epilogue_done;
                ptx::tc_fence_after();
                const uint32_t t_row = tmem_base + buf * 256u + uint32_t(c_begin) + ((quarter * 32u) << 16);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (32 * i < c_count) {
                        uint32_t r[32];
                        ptx::tmem_ld_32x32(t_row + 32 * i, r);
                        ptx::tmem_ld_wait();
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            const float4 sc = *reinterpret_cast<const float4*>(s + 32 * i + j);
                            fma2(acc[i][j], acc[i][j + 1], r[j], r[j + 1], sc.x, sc.y);
                            fma2(acc[i][j + 2], acc[i][j + 3], r[j + 2], r[j + 3], sc.z, sc.w);
                        }
                    }
                }
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    const uint32_t e = ptx::smem_u32(&bar_acc_empty[buf]);
                    if (CTAS == 2 && !is_leader) ptx::mbar_arrive_cluster_relaxed(ptx::mapa(e, 0));
                    else ptx::mbar_arrive(e);
                }
            }
            const Fp8Activation act(p.act);
            if (feature < p.features) {
                const float bias = p.bias != nullptr ? __ldg(p.bias + feature) : 0.0f;
                OutT* dst = static_cast<OutT*>(p.c) + (long long)(t.col0 + c_begin) * p.features + feature;
                const int stored = min(c_count, t.col_count - c_begin);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (32 * i < stored) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) acc[i][j] += bias;
                        fp8_activation(acc[i], act);
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (32 * i + j < stored) dst[(long long)(32 * i + j) * p.features] = round_to<OutT>(acc[i][j]);
                    }
                }
            }
        }
    epilogue_done:
        __syncwarp();
        if (CTAS == 2) ptx::cluster_arrive();
    }

    // ---------------------------------------------------------------- teardown
    ptx::tc_fence_before();
    __syncthreads();
    if (abort_flag) {
        const uint64_t t0 = ptx::globaltimer_ns();
        while (ptx::globaltimer_ns() - t0 < 2000000ull) { }
        __syncthreads();
    }
    if (CTAS == 2) ptx::cluster_wait();
    if (warp == 1) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc<CTAS>(tmem_base, 512);
    }
#else
    if (threadIdx.x == 0 && blockIdx.x == 0) atomicCAS(p.status, 0u, 0xdeadu);
#endif
}

}  // namespace cudeep_b200
