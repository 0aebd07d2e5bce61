// Products of 8-bit (e4m3) matrices with a scale per block of 128, FP32 accumulation (tcgen05 kind::f8f6f4).
//
//   NT  C[r, f] = sum_b xs[b][r] ws[f / 128][b] ( sum_{k in block b} X[r, k] W[f, k] )     y = x W^T
//   NN  C[r, f] = sum_b xs[b][r] ws[b][f / 128] ( sum_{k in block b} X[r, k] W[k, f] )     dx = dy W
//
// A scale changes with every block of 128 along the sum, so the tensor core may only sum within one block: each K block
// (128 bytes per row, four MMAs of K = 32) is multiplied into a fresh TMEM accumulator, and eight epilogue warps take it
// out and add it, scaled, to sums that they hold in registers (two FP32 lanes per fma.rn.f32x2).  Those sums round to
// nearest, so the length of K costs no accuracy beyond FP32's.  While one accumulator is drained the tensor core fills
// the next.  Two orientations: many rows (fp8_rows.cuh) and few (below).
#pragma once

#include "ragged_gemm.cuh"

namespace cudeep_b200 {

constexpr int FP8_BK = 128;                     // elements per K block = one 128-byte swizzle row = one scale

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

// The epilogue's activations as one formula, y = g * sigmoid(t), g = z (GELU in its tanh form, SiLU) or 1 (sigmoid), with
// -t log2(e) = u = z (a + b z^2).  sigmoid = 1 / d, d = 1 + 2^u, and two values share one reciprocal, 1 / d0 = d1 / (d0 d1): the
// SFU is what bounds an epilogue that activates 128 values a thread, and this takes three of its operations per pair instead
// of four.  u is held below 126, where sigmoid is FP32's least normal number, 2^-126, and so that d0 d1 stays finite d1 is
// taken times 2^-126: the product then lies between 2^-126 and 2^126, and one more multiplication per pair takes that out of
// 1 / d1: 8192 x 4096 -> 16384 with GELU 469.3 us in bursts, 467.6 us with u held below 60 and no factors.  (The sign of u
// instead, sigmoid = 2^-u / (1 + 2^-u) for positive u, costs three operations a value, 482 us.)  g is held above -128, so that no z however low makes more of 2^-126 than 2^-119.
// fminf also keeps a NaN from its neighbour, and the factor g carries it on.  Where the formula has no cubic term b is a
// negligible number of the right sign instead of 0: 0 * Inf is NaN.
struct Fp8Activation {
    int act;
    float a, b;
    float g_lo, g_hi;
    __device__ __forceinline__ explicit Fp8Activation(int act_) : act(act_) {
        const float c = act == EPI_GELU ? 2.0f * 0.7978845608028654f : 1.0f;
        a = -1.4426950408889634f * c;
        b = act == EPI_GELU ? a * 0.044715f : -1e-37f;
        g_lo = act == EPI_SIGMOID ? 1.0f : -128.0f;
        g_hi = act == EPI_SIGMOID ? 1.0f : __int_as_float(0x7f800000);
    }
};

template <int N>
__device__ __forceinline__ void fp8_activation(float (&v)[N], const Fp8Activation& f) {
    static_assert(N % 2 == 0, "values are activated in pairs");
    if (f.act == EPI_NONE) return;
    if (f.act == EPI_RELU) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = fmaxf(v[j], 0.0f);      // as the other epilogues' ReLU, which drops NaN
        return;
    }
    constexpr float least = 1.17549435e-38f;      // 2^-126
#pragma unroll
    for (int j = 0; j < N; j += 2) {
        const float x0 = v[j], x1 = v[j + 1];
        const float d0 = 1.0f + sfu_ex2(fminf(x0 * fmaf(f.b * x0, x0, f.a), 126.0f));
        const float d1 = fmaf(sfu_ex2(fminf(x1 * fmaf(f.b * x1, x1, f.a), 126.0f)), least, least);
        const float r = sfu_rcp(d0 * d1);
        v[j] = clamp_nan(x0, f.g_lo, f.g_hi) * (d1 * r);
        v[j + 1] = clamp_nan(x1, f.g_lo, f.g_hi) * ((d0 * r) * least);
    }
}

// ---- few tiles ----------------------------------------------------------------------------------------------------------------

// For few rows (and for few features, whatever the rows) the FEATURES lie on the 128 lanes and up to 128 rows on the
// columns: the width of the MMA follows the number of rows, and a CTA streams its features' weights once, which is all that
// a product of a few rows costs.  One tile per CTA; where there are fewer tiles than the device has SMs, a cluster of up to
// eight CTAs shares a tile, each with a range of K, and adds the parts up through distributed shared memory in rank order.
// A tile may take fewer than 128 features (the last lanes then idle), so that the tiles fill the SMs: 16384 features are 128
// tiles of 128, but 147 of 112.
//
// The factors xs * ws change along the columns here: each epilogue warp fetches those of its columns four blocks ahead and
// reads them back from shared memory.  With so few columns TMEM holds up to eight accumulators, so the tensor core runs
// ahead of the sums by that many blocks (two accumulators and factors one block ahead: 16 rows, 4096 -> 16384 took 35 us,
// every block waiting for its factors; now 17 us).
constexpr int FP8F_MAX_ROWS = 128;
constexpr int FP8F_EPI_WARPS = 8;
constexpr int FP8F_THREADS = 64 + 32 * FP8F_EPI_WARPS;
constexpr int FP8F_MAX_STAGES = 12;
constexpr int FP8F_MAX_BUFFERS = 8;
constexpr uint32_t FP8F_SMEM_BUDGET = 232448 - 1024 - 6 * 1024;   // minus alignment slack, factors and barriers

struct Fp8FewParams {
    CUtensorMap map_w;       // NT {K, F} box {128, step}; NN {F, K} box {128, 128}
    RowMaps x;               // {K, rows}
    const float* x_scales;   // [K blocks][rows]
    const float* w_scales;   // + feature block * ws_feature + K block * ws_k
    long long ws_feature, ws_k;
    const float* bias;
    int act;
    void* c;
    int rows;
    int tile_rows;           // rows per tile, up to 128
    int features;
    int f_tiles;
    int k;
    int split;               // CTAs per tile
    int step;                // features per tile, a multiple of 16 up to 128
    uint32_t w_bytes;        // of a stage
    int stages;
    uint32_t stage_bytes;
    uint32_t* status;
    unsigned long long wait_limit_ns;
};

template <RaggedForm FORM, class OutT>
__global__ void __launch_bounds__(FP8F_THREADS, 1) fp8_few_kernel(const __grid_constant__ Fp8FewParams p) {
#if defined(__CUDA_ARCH_FEAT_SM100_ALL) || defined(__CUDA_ARCH_FEAT_SM101_ALL) || \
    defined(__CUDA_ARCH_FEAT_SM103_ALL)
    constexpr bool A_MN = FORM == RaggedForm::NN;

    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bar_full[FP8F_MAX_STAGES];
    __shared__ __align__(8) uint64_t bar_empty[FP8F_MAX_STAGES];
    __shared__ __align__(8) uint64_t bar_acc_full[FP8F_MAX_BUFFERS];
    __shared__ __align__(8) uint64_t bar_acc_empty[FP8F_MAX_BUFFERS];
    __shared__ __align__(16) float factors[FP8F_EPI_WARPS][2][64];
    __shared__ uint32_t tmem_base_holder;
    __shared__ uint32_t abort_flag;

    const uint32_t warp = threadIdx.x >> 5;
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    ptx::WaitCtx wctx{&abort_flag, p.status, p.wait_limit_ns};

    const int split = p.split;
    const uint32_t rank = split > 1 ? ptx::cluster_ctarank() : 0u;
    const int tile = int(blockIdx.x) / split;
    const int feature0 = tile % p.f_tiles * p.step;
    const int row0 = tile / p.f_tiles * p.tile_rows;
    const int rows = min(p.tile_rows, p.rows - row0);      // of this tile
    const int f_end = min(p.features, feature0 + p.step);
    const int umma_n = (rows + 15) / 16 * 16;
    const int buf_cols = (rows + 31) / 32 * 32;
    const int buffers = min(FP8F_MAX_BUFFERS, 512 / buf_cols);
    const int all_blocks = (p.k + FP8_BK - 1) / FP8_BK;
    const int share = (all_blocks + split - 1) / split;
    const int kb0 = min(all_blocks, int(rank) * share);
    const int blocks = min(share, all_blocks - kb0);      // may be none for the last ranks

    if (threadIdx.x == 0) {
        abort_flag = 0;
        ptx::prefetch_tensormap(&p.map_w);
        p.x.prefetch();
        for (int s = 0; s < FP8F_MAX_STAGES; ++s) {
            ptx::mbar_init(ptx::smem_u32(&bar_full[s]), 1);
            ptx::mbar_init(ptx::smem_u32(&bar_empty[s]), 1);
        }
        for (int a = 0; a < FP8F_MAX_BUFFERS; ++a) {
            ptx::mbar_init(ptx::smem_u32(&bar_acc_full[a]), 1);
            ptx::mbar_init(ptx::smem_u32(&bar_acc_empty[a]), FP8F_EPI_WARPS);
        }
        ptx::fence_mbar_init();
    }
    if (warp == 1) {
        ptx::tmem_alloc<1>(ptx::smem_u32(&tmem_base_holder), 512);
        ptx::tmem_relinquish<1>();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem_base = tmem_base_holder;
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();

    // Epilogue warps 2..5 take the first half of the columns, 6..9 the second; each its quarter of the lanes.
    const uint32_t quarter = warp & 3u;
    const int half = int(warp - 2) >> 2;
    const int half_cols = (umma_n / 2 + 15) / 16 * 16;
    const int c_begin = half * half_cols;
    const int c_count = min(half_cols, umma_n - c_begin);
    const int feature = feature0 + int(quarter) * 32 + int(lane);
    float acc[4][16];

    if (warp == 0) {
        // ------------------------------------------------------------ producer
        if (lane == 0) {
            uint32_t stage = 0, phase = 0;
            const uint32_t bytes = p.w_bytes + uint32_t(RowMaps::loaded(umma_n)) * 128u;
            for (int kb = 0; kb < blocks; ++kb) {
                if (!ptx::mbar_wait(ptx::smem_u32(&bar_empty[stage]), phase ^ 1u, wctx, UMMA_TIMEOUT_PRODUCER)) break;
                const uint32_t a_smem = smem_base + stage * p.stage_bytes;
                const uint32_t full = ptx::smem_u32(&bar_full[stage]);
                ptx::mbar_arrive_expect_tx(full, bytes);
                const int k0 = (kb0 + kb) * FP8_BK;
                ptx::tma_load_2d(a_smem, &p.map_w, full, A_MN ? feature0 : k0, A_MN ? k0 : feature0);
                p.x.template load<1>(a_smem + RAGGED_A_BYTES, full, k0, row0, umma_n);
                if (++stage == uint32_t(p.stages)) { stage = 0; phase ^= 1u; }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer
        constexpr uint32_t A_KSTEP = A_MN ? 4096u : 32u;
        const uint32_t idesc = ptx::idesc_e4m3(128, umma_n, A_MN ? 1 : 0, 0);
        const uint64_t a_desc0 = ptx::smem_desc_at(ptx::smem_desc(A_MN ? 16384 : 16, 1024, ptx::SMEM_LAYOUT_SW128), smem_base);
        const uint64_t b_desc0 =
            ptx::smem_desc_at(ptx::smem_desc(16, 1024, ptx::SMEM_LAYOUT_SW128), smem_base + RAGGED_A_BYTES);
        uint32_t stage = 0, phase = 0, buf = 0, buf_phase = 0;
        for (int kb = 0; kb < blocks; ++kb) {
            if (!__all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&bar_acc_empty[buf]), buf_phase ^ 1u, wctx,
                                                        UMMA_TIMEOUT_MMA_ACC)))
                break;
            if (!__all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&bar_full[stage]), phase, wctx, UMMA_TIMEOUT_MMA_FULL)))
                break;
            ptx::tc_fence_after();
            if (ptx::elect_one()) {
                const uint64_t a_stage = a_desc0 + ((stage * p.stage_bytes) >> 4);
                const uint64_t b_stage = b_desc0 + ((stage * p.stage_bytes) >> 4);
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                    ptx::umma_f8<1>(tmem_base + buf * uint32_t(buf_cols), a_stage + ((kk * A_KSTEP) >> 4),
                                    b_stage + ((kk * 32u) >> 4), idesc, kk != 0);
                ptx::umma_commit<1>(ptx::smem_u32(&bar_acc_full[buf]));
                ptx::umma_commit<1>(ptx::smem_u32(&bar_empty[stage]));
            }
            __syncwarp();
            if (++stage == uint32_t(p.stages)) { stage = 0; phase ^= 1u; }
            if (++buf == uint32_t(buffers)) { buf = 0; buf_phase ^= 1u; }
        }
    } else {
        // ------------------------------------------------------------ sums
        float* mine = &factors[warp - 2][0][0];
        const float* xs = p.x_scales + (long long)kb0 * p.rows + row0 + c_begin;
        // A tile's features may belong to two blocks of scales; lanes behind the last feature take some that exist.
        const float* ws = p.w_scales + (min(feature, p.features - 1) / 128) * p.ws_feature + kb0 * p.ws_k;
        float px[4][2], pw[4];
        auto fetch = [&](int kb, float (&x)[2], float& w) {
            w = kb < blocks ? __ldg(ws + kb * p.ws_k) : 0.0f;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int c = int(lane) + 32 * i;
                x[i] = kb < blocks && c < c_count && c_begin + c < rows ? __ldg(xs + (long long)kb * p.rows + c) : 0.0f;
            }
        };
#pragma unroll
        for (int d = 0; d < 4; ++d) fetch(d, px[d], pw[d]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) acc[i][j] = 0.0f;
        uint32_t buf = 0, buf_phase = 0;
        bool ok = true;
#pragma unroll 1
        for (int kb4 = 0; kb4 < blocks && ok; kb4 += 4) {
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const int kb = kb4 + d;
                if (kb >= blocks) break;
                float* f = mine + (d & 1) * 64;
                const float w = pw[d];
                f[lane] = px[d][0];
                f[lane + 32] = px[d][1];
                __syncwarp();
                fetch(kb + 4, px[d], pw[d]);
                ok = ptx::mbar_wait(ptx::smem_u32(&bar_acc_full[buf]), buf_phase, wctx, UMMA_TIMEOUT_EPILOGUE);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                ptx::tc_fence_after();
                const uint32_t t_row = tmem_base + buf * uint32_t(buf_cols) + uint32_t(c_begin) + ((quarter * 32u) << 16);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (16 * i < c_count) {
                        uint32_t r[16];
                        ptx::tmem_ld_32x16(t_row + 16 * i, r);
                        ptx::tmem_ld_wait(r);
#pragma unroll
                        for (int j = 0; j < 16; j += 4) {
                            const float4 sc = *reinterpret_cast<const float4*>(f + 16 * i + j);
                            fma2(acc[i][j], acc[i][j + 1], r[j], r[j + 1], sc.x * w, sc.y * w);
                            fma2(acc[i][j + 2], acc[i][j + 3], r[j + 2], r[j + 3], sc.z * w, sc.w * w);
                        }
                    }
                }
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&bar_acc_empty[buf]));
                if (++buf == uint32_t(buffers)) { buf = 0; buf_phase ^= 1u; }
            }
        }
        const Fp8Activation act(p.act);
        const int stored = min(c_count, rows - c_begin);
        if (split == 1) {
            if (feature < f_end) {
                const float bias = p.bias != nullptr ? __ldg(p.bias + feature) : 0.0f;
                OutT* dst = static_cast<OutT*>(p.c) + (long long)(row0 + c_begin) * p.features + feature;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (16 * i < stored) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) acc[i][j] += bias;
                        fp8_activation(acc[i], act);
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            if (16 * i + j < stored) dst[(long long)(16 * i + j) * p.features] = round_to<OutT>(acc[i][j]);
                    }
                }
            }
        } else {
            // The stage ring is idle (every load was consumed by an MMA whose sums were taken out): it takes this CTA's part,
            // [column][128 features].
            const uint32_t part = smem_base + (uint32_t(c_begin) * 128u + quarter * 32u + lane) * 4u;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (16 * i + j < c_count) ptx::st_shared_f32(part + uint32_t(16 * i + j) * 512u, acc[i][j]);
        }
    }
    __syncwarp();
    if (split > 1) {
        ptx::cluster_arrive();
        ptx::cluster_wait();
        if (warp >= 2) {
            // Rank r finishes columns r, r + split, ...: a warp takes a column, four features a lane, and reads the parts of
            // all ranks of two columns at once.
            const Fp8Activation act(p.act);
            const int f_in = 4 * int(lane), f = feature0 + f_in;
            float bias[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) bias[j] = p.bias != nullptr && f + j < f_end ? __ldg(p.bias + f + j) : 0.0f;
            const int step = split * FP8F_EPI_WARPS;
            for (int c = int(rank) + split * int(warp - 2); c < rows; c += 2 * step) {
                float v[2][4] = {};
                for (int s = 0; s < split; ++s) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int cc = c + i * step < rows ? c + i * step : c;
                        const float4 q = ptx::ld_cluster_v4(
                            ptx::mapa(smem_base + (uint32_t(cc) * 128u + uint32_t(f_in)) * 4u, uint32_t(s)));
                        v[i][0] += q.x;
                        v[i][1] += q.y;
                        v[i][2] += q.z;
                        v[i][3] += q.w;
                    }
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (c + i * step >= rows) break;
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[i][j] += bias[j];
                    fp8_activation(v[i], act);
                    OutT* dst = static_cast<OutT*>(p.c) + (long long)(row0 + c + i * step) * p.features + f;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (f + j < f_end) dst[j] = round_to<OutT>(v[i][j]);
                }
            }
        }
        __syncwarp();
        ptx::cluster_arrive();      // nobody leaves while its part may still be read
        ptx::cluster_wait();
    }

    // ---------------------------------------------------------------- teardown
    ptx::tc_fence_before();
    __syncthreads();
    if (abort_flag) {
        const uint64_t t0 = ptx::globaltimer_ns();
        while (ptx::globaltimer_ns() - t0 < 2000000ull) { }
        __syncthreads();
    }
    if (warp == 1) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc<1>(tmem_base, 512);
    }
#else
    if (threadIdx.x == 0 && blockIdx.x == 0) atomicCAS(p.status, 0u, 0xdeadu);
#endif
}

}  // namespace cudeep_b200
