// The 8-bit products of fp8_gemm.cuh with the ROWS on the accumulator's lanes, for matrices of many rows.
//
//   NT  C[r, f] = sum_b xs[b][r] ws[f / 128][b] ( sum_{k in block b} X[r, k] W[f, k] )
//   NN  C[r, f] = sum_b xs[b][r] ws[b][f / 128] ( sum_{k in block b} X[r, k] W[k, f] )
//
// A thread then owns one row and 128 consecutive features, which share one scale of W: a K block's sum is added with a
// single factor per thread, xs * ws, that waits in a register, where the other orientation reads a factor per column from
// shared memory.  What bounds the kernel is taking the accumulators out of TMEM: each block of 128 (512 cycles of MMAs on
// a 256 x 256 tile of a CTA pair) hands 128 x 256 sums to eight warps, 64 packed multiply-adds a thread.  To hold
// 128 sums, two sets of 16 values on their way out of TMEM and the rest, those warps take the registers that the first four
// warps (producer, MMA issuer, two that only wait) give up.  (With sets of 32 the compiler spilled in this loop: 8192 x 4096 x
// 16384 took 778 us, with sets of 16 it takes 491 us; without any sums taken out, 448 us.)
#pragma once

#include "fp8_gemm.cuh"

namespace cudeep_b200 {

constexpr int FP8R_THREADS = 384;               // three groups of four warps
// Registers per thread: 384 * 168 at launch; 128 * 56 + 256 * 216 = 62464 <= 64512 afterwards.
constexpr int FP8R_REGS_FEW = 56;
constexpr int FP8R_REGS_MANY = 216;
constexpr int FP8R_ATOMS = 2;                     // K blocks per stage
constexpr uint32_t FP8R_ATOM_BYTES = 2 * 128 * 128;
constexpr uint32_t FP8R_STAGE_BYTES = FP8R_ATOMS * FP8R_ATOM_BYTES;
constexpr uint32_t FP8R_STAGING_BYTES = 8 * 4096;      // 32 rows x 128 bytes per epilogue warp
constexpr int FP8R_STAGES = 3;
constexpr uint32_t FP8R_SMEM_BYTES = FP8R_STAGES * FP8R_STAGE_BYTES + FP8R_STAGING_BYTES + 1024;

constexpr int SCALE_FLAGS = 256;      // CTAs of pack_scales_kernel (fp8_scaled.cuh), each with a word of its own

// Whether any word is set; all threads of the CTA.
__device__ __forceinline__ bool any_odd_scales(const uint32_t* flags) {
    return __syncthreads_or(threadIdx.x < SCALE_FLAGS ? int(__ldg(flags + threadIdx.x)) : 0) != 0;
}

struct Fp8RowsParams {
    CUtensorMap map_x;       // {K, rows} box {128, 128}
    CUtensorMap map_w;       // NT {K, F} box {128, BN / 2}; NN {F, K} box {128, 128}
    CUtensorMap map_c;       // {F, rows} box {128 bytes, 32}; used when `tma_store`
    const float* x_scales;   // [K blocks][rows]
    const float* w_scales;   // + feature block * ws_feature + K block * ws_k
    long long ws_feature, ws_k;
    const float* bias;
    int act;
    void* c;
    int tma_store;
    int rows;
    int features;
    int k;
    int tiles_m, tiles_n;
    const uint32_t* odd_scales;      // nullptr, or SCALE_FLAGS words: run only if one of them is set
    uint32_t* status;
    unsigned long long wait_limit_ns;
};

template <int REGS>
__device__ __forceinline__ void take_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS)); }
template <int REGS>
__device__ __forceinline__ void give_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS)); }

// A warp's 32 rows x BN / 2 features: bias, activation, and out through its staging block of ROWS x 128 bytes (the box of map_c).
template <int BN, class OutT, int ROWS, class Params>
__device__ __forceinline__ void store_tile(const Params& p, float (&acc)[BN / 64][32], const Fp8Activation& act, uint32_t staging,
                                           uint32_t lane, int row0, int feature0) {
    constexpr int COLS = 128 / sizeof(OutT);          // columns of a staged block
    constexpr int CHUNKS = COLS / 32;                 // of 32 columns
#pragma unroll
    for (int i0 = 0; i0 < BN / 64; i0 += CHUNKS) {
        const int f0 = feature0 + 32 * i0;
#pragma unroll
        for (int i = i0; i < i0 + CHUNKS; ++i) {
            if (p.bias != nullptr) {
#pragma unroll
                for (int j = 0; j < 32; ++j) acc[i][j] += __ldg(p.bias + min(feature0 + 32 * i + j, p.features - 1));
            }
            fp8_activation(acc[i], act);
        }
#pragma unroll
        for (int r0 = 0; r0 < 32; r0 += ROWS) {
            if (lane == 0) ptx::bulk_wait_group_read<0>();      // the block's last store has read it
            __syncwarp();
            if (ROWS == 32 || int(lane) / ROWS == r0 / ROWS) {
#pragma unroll
                for (int i = i0; i < i0 + CHUNKS; ++i) stage_block<OutT>(staging, lane % ROWS, 32 * (i - i0), acc[i]);
            }
            if (p.tma_store) {
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0 && row0 + r0 < p.rows && f0 < p.features) {
                    ptx::tma_store_2d(&p.map_c, staging, f0, row0 + r0);
                    ptx::bulk_commit_group();
                }
            } else {
                // Rows of C that are no 16-byte multiples: the warp writes them one by one.
                __syncwarp();
                OutT* dst = static_cast<OutT*>(p.c) + (long long)(row0 + r0) * p.features + f0;
                write_block<OutT>(staging, lane, dst, p.features, min(ROWS, p.rows - row0 - r0), p.features - f0, false);
            }
        }
    }
}

template <RaggedForm FORM, int BN, class OutT>
__global__ void __launch_bounds__(FP8R_THREADS, 1) fp8_rows_kernel(const __grid_constant__ Fp8RowsParams p) {
#if defined(__CUDA_ARCH_FEAT_SM100_ALL) || defined(__CUDA_ARCH_FEAT_SM101_ALL) || \
    defined(__CUDA_ARCH_FEAT_SM103_ALL)
    constexpr bool B_MN = FORM == RaggedForm::NN;
    static_assert(BN == 256 || (BN == 128 && !B_MN), "a row of features in a box is one 128-byte swizzle row");
    constexpr int CHUNKS = BN / 32;      // of 16 columns, per epilogue warp (half of the tile's columns)
    constexpr uint32_t TX_BYTES = FP8R_ATOMS * (2 * 16384 + BN * 128);

    if (p.odd_scales != nullptr) {
        ptx::grid_dependency_wait();
        if (!any_odd_scales(p.odd_scales)) return;      // the tensor core has applied these scales itself
    }
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bar_full[FP8R_STAGES];
    __shared__ __align__(8) uint64_t bar_empty[FP8R_STAGES];
    __shared__ __align__(8) uint64_t bar_acc_full[2];
    __shared__ __align__(8) uint64_t bar_acc_empty[2];
    __shared__ uint32_t tmem_base_holder;
    __shared__ uint32_t abort_flag;

    const uint32_t warp = threadIdx.x >> 5;
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t cta_rank = ptx::cluster_ctarank();
    const bool is_leader = cta_rank == 0;
    const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    ptx::WaitCtx wctx{&abort_flag, p.status, p.wait_limit_ns};

    if (threadIdx.x == 0) {
        abort_flag = 0;
        ptx::prefetch_tensormap(&p.map_x);
        ptx::prefetch_tensormap(&p.map_w);
        ptx::prefetch_tensormap(&p.map_c);
        for (int s = 0; s < FP8R_STAGES; ++s) {
            ptx::mbar_init(ptx::smem_u32(&bar_full[s]), 1);
            ptx::mbar_init(ptx::smem_u32(&bar_empty[s]), 1);
        }
        for (int a = 0; a < 2; ++a) {
            ptx::mbar_init(ptx::smem_u32(&bar_acc_full[a]), 1);
            ptx::mbar_init(ptx::smem_u32(&bar_acc_empty[a]), 8 * 2);
        }
        ptx::fence_mbar_init();
    }
    if (warp == 1) {
        ptx::tmem_alloc<2>(ptx::smem_u32(&tmem_base_holder), 512);
        ptx::tmem_relinquish<2>();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::cluster_arrive();
    ptx::cluster_wait();
    ptx::tc_fence_after();
    const uint32_t tmem_base = tmem_base_holder;
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();

    const int unit_stride = gridDim.x / 2;
    const int first_unit = blockIdx.x / 2;
    const int num_units = p.tiles_m * p.tiles_n;
    const int k_blocks = (p.k + FP8_BK - 1) / FP8_BK;

    if (warp < 4) {
        give_registers<FP8R_REGS_FEW>();
        if (warp == 0) {
            // -------------------------------------------------------- producer
            if (lane == 0) {
                uint32_t stage = 0, phase = 0;
                for (int u = first_unit; u < num_units; u += unit_stride) {
                    int tm, tn;
                    raster_coords(u, p.tiles_m, p.tiles_n, 8, tm, tn);
                    const int row = (tm * 2 + int(cta_rank)) * 128;
                    const int feature = tn * BN + int(cta_rank) * (BN / 2);
                    for (int kb = 0; kb < k_blocks; kb += FP8R_ATOMS) {
                        if (!ptx::mbar_wait(ptx::smem_u32(&bar_empty[stage]), phase ^ 1u, wctx, UMMA_TIMEOUT_PRODUCER))
                            goto producer_done;
                        const uint32_t full_local = ptx::smem_u32(&bar_full[stage]);
                        if (is_leader) ptx::mbar_arrive_expect_tx(full_local, TX_BYTES);
                        const uint32_t full = ptx::mapa(full_local, 0);
#pragma unroll
                        for (int a = 0; a < FP8R_ATOMS; ++a) {      // a block behind the last one loads as zeros
                            const uint32_t a_smem = smem_base + stage * FP8R_STAGE_BYTES + a * FP8R_ATOM_BYTES;
                            const int k0 = (kb + a) * FP8_BK;
                            ptx::tma_load_2d_pair(a_smem, &p.map_x, full, k0, row);
                            ptx::tma_load_2d_pair(a_smem + 16384, &p.map_w, full, B_MN ? feature : k0, B_MN ? k0 : feature);
                        }
                        if (++stage == FP8R_STAGES) { stage = 0; phase ^= 1u; }
                    }
                }
            }
        producer_done:
            __syncwarp();
        } else if (warp == 1 && is_leader) {
            // -------------------------------------------------------- MMA issuer
            constexpr uint32_t B_KSTEP = B_MN ? 4096u : 32u;
            constexpr uint32_t idesc = ptx::idesc_e4m3(256, BN, 0, B_MN ? 1 : 0);
            const uint64_t a_desc0 = ptx::smem_desc_at(ptx::smem_desc(16, 1024, ptx::SMEM_LAYOUT_SW128), smem_base);
            const uint64_t b_desc0 =
                ptx::smem_desc_at(ptx::smem_desc(B_MN ? 16384 : 16, 1024, ptx::SMEM_LAYOUT_SW128), smem_base + 16384);
            uint32_t stage = 0, phase = 0, it = 0;
            for (int u = first_unit; u < num_units; u += unit_stride) {
                for (int kb = 0; kb < k_blocks; ++kb, ++it) {
                    const uint32_t acc = it & 1;
                    const uint32_t atom = uint32_t(kb) % FP8R_ATOMS;
                    if (atom == 0 && !__all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&bar_full[stage]), phase, wctx,
                                                                             UMMA_TIMEOUT_MMA_FULL)))
                        goto mma_done;
                    if (!__all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&bar_acc_empty[acc]), ((it >> 1) & 1) ^ 1u,
                                                                wctx, UMMA_TIMEOUT_MMA_ACC)))
                        goto mma_done;
                    ptx::tc_fence_after();
                    const bool stage_done = atom + 1 == FP8R_ATOMS || kb + 1 == k_blocks;
                    if (ptx::elect_one()) {
                        const uint64_t offset = (stage * FP8R_STAGE_BYTES + atom * FP8R_ATOM_BYTES) >> 4;
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            ptx::umma_f8<2>(tmem_base + acc * 256u, a_desc0 + offset + ((kk * 32u) >> 4),
                                            b_desc0 + offset + ((kk * B_KSTEP) >> 4), idesc, kk != 0);
                        const uint32_t accf_local = ptx::smem_u32(&bar_acc_full[acc]);
                        ptx::umma_commit<2>(accf_local);
                        ptx::umma_commit<2>(ptx::mapa(accf_local, 1));
                        if (stage_done) {
                            const uint32_t empty_local = ptx::smem_u32(&bar_empty[stage]);
                            ptx::umma_commit<2>(empty_local);
                            ptx::umma_commit<2>(ptx::mapa(empty_local, 1));
                        }
                    }
                    __syncwarp();
                    if (stage_done && ++stage == FP8R_STAGES) { stage = 0; phase ^= 1u; }
                }
            }
        mma_done:
            __syncwarp();
        }
        ptx::cluster_arrive();
    } else {
        take_registers<FP8R_REGS_MANY>();
        // ------------------------------------------------------------ sums and epilogue
        const uint32_t quarter = warp & 3u;
        const int half = int(warp - 4) >> 2;
        const uint32_t staging = smem_base + FP8R_STAGES * FP8R_STAGE_BYTES + (warp - 4) * 4096u;
        const Fp8Activation act(p.act);
        uint32_t it = 0;
        for (int u = first_unit; u < num_units; u += unit_stride) {
            int tm, tn;
            raster_coords(u, p.tiles_m, p.tiles_n, 8, tm, tn);
            const int row0 = (tm * 2 + int(cta_rank)) * 128 + int(quarter) * 32;
            const int row = row0 + int(lane);
            const int feature0 = tn * BN + half * (BN / 2);
            // Rows and features outside the matrices take some factor that exists; what it makes is not stored.
            const float* xs = p.x_scales + (row < p.rows ? row : 0);
            const float* ws = p.w_scales + (feature0 < p.features ? feature0 / 128 : 0) * p.ws_feature;
            float acc[BN / 64][32];
#pragma unroll
            for (int i = 0; i < BN / 64; ++i)
#pragma unroll
                for (int j = 0; j < 32; ++j) acc[i][j] = 0.0f;
            // The factors come four blocks ahead: a block takes 500 cycles and a load from L2 under this traffic longer.
            float px[4], pw[4];
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                px[d] = d < k_blocks ? __ldg(xs + (long long)d * p.rows) : 0.0f;
                pw[d] = d < k_blocks ? __ldg(ws + d * p.ws_k) : 0.0f;
            }
#pragma unroll 1
            for (int kb4 = 0; kb4 < k_blocks; kb4 += 4) {
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    const int kb = kb4 + d;
                    if (kb >= k_blocks) break;
                    const float s = px[d] * pw[d];
                    if (kb + 4 < k_blocks) {
                        px[d] = __ldg(xs + (long long)(kb + 4) * p.rows);
                        pw[d] = __ldg(ws + (kb + 4) * p.ws_k);
                    }
                    const uint32_t buf = it & 1;
                    const bool ok = ptx::mbar_wait(ptx::smem_u32(&bar_acc_full[buf]), (it >> 1) & 1, wctx, UMMA_TIMEOUT_EPILOGUE);
                    if (!__all_sync(0xffffffffu, ok)) goto epilogue_done;
                    ptx::tc_fence_after();
                    const uint32_t t_row = tmem_base + buf * 256u + uint32_t(half) * uint32_t(BN / 2) + ((quarter * 32u) << 16);
                    uint32_t r[2][16];
                    ptx::tmem_ld_32x16(t_row, r[0]);
#pragma unroll
                    for (int i = 0; i < CHUNKS; ++i) {
                        ptx::tmem_ld_wait(r[i & 1]);
                        if (i + 1 < CHUNKS) {
                            ptx::tmem_ld_32x16(t_row + 16 * (i + 1), r[(i + 1) & 1]);
                        } else {
                            ptx::tc_fence_before();
                            __syncwarp();
                            if (lane == 0) {
                                const uint32_t e = ptx::smem_u32(&bar_acc_empty[buf]);
                                if (is_leader) ptx::mbar_arrive(e);
                                else ptx::mbar_arrive_cluster_relaxed(ptx::mapa(e, 0));
                            }
                        }
#pragma unroll
                        for (int j = 0; j < 16; j += 2) {
                            float* sum = &acc[i >> 1][(i & 1) * 16 + j];
                            fma2(sum[0], sum[1], r[i & 1][j], r[i & 1][j + 1], s, s);
                        }
                    }
                    ++it;
                }
            }
            store_tile<BN, OutT, 32>(p, acc, act, staging, lane, row0, feature0);
        }
    epilogue_done:
        __syncwarp();
        ptx::cluster_arrive();
        if (lane == 0) ptx::bulk_wait_group_read<0>();
        __syncwarp();
    }

    // ---------------------------------------------------------------- teardown
    ptx::tc_fence_before();
    __syncthreads();
    if (abort_flag) {
        const uint64_t t0 = ptx::globaltimer_ns();
        while (ptx::globaltimer_ns() - t0 < 2000000ull) { }
        __syncthreads();
    }
    ptx::cluster_wait();
    if (warp == 1) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc<2>(tmem_base, 512);
    }
#else
    if (threadIdx.x == 0 && blockIdx.x == 0) atomicCAS(p.status, 0u, 0xdeadu);
#endif
}

}  // namespace cudeep_b200
