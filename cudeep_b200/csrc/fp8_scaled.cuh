// The 8-bit products of fp8_rows.cuh with the scales applied by the tensor core (tcgen05 kind::mxf8f6f4), for scales that are powers
// of two, as quantize_fp8 makes them.
//
// That MMA takes a scale of 8 exponent bits for each row and 32 elements of K from tensor memory.  A block of 128 elements is
// four of them with one scale, so a word of four equal bytes per row and K block is all it needs, and sums may stay in the
// accumulator over many blocks: nothing has to be taken out of TMEM for each of them, which is what bounds fp8_rows.cuh.
// pack_scales_kernel writes those words, 128 rows of a K block to 512 bytes in the order that tcgen05.cp spreads over the lanes
// (row r in word 4 (r % 32) + r / 32), and notes whether a scale was not a power of two; then this kernel leaves the product to
// the one behind it.
//
// The accumulator of 256 columns leaves TMEM no room for a second next to the scales, so the epilogue warps take a finished tile into
// registers at once and the next tile's MMAs begin while they store it.  The tensor core truncates as it sums; products of e4m3
// values have few bits to lose (FP32 results of up to 16384 elements of K, 2048 in the accumulator at a time: no mean loss above
// 3e-8), but as scales differ an FP32 result is taken out and added up every 2048 elements of K, a 16-bit one every 16384.
#pragma once

#include "fp8_rows.cuh"

namespace cudeep_b200 {

constexpr int FP8S_STAGES = 3;
constexpr uint32_t FP8S_SCALE_BYTES = 3 * 512;         // of a K block: 128 rows, 256 features
constexpr uint32_t FP8S_STAGING_BYTES = 8 * 2048;      // 16 rows x 128 bytes per epilogue warp: what three stages of two blocks leave
constexpr uint32_t FP8S_SMEM_BYTES =
    FP8S_STAGES * (FP8R_STAGE_BYTES + FP8R_ATOMS * FP8S_SCALE_BYTES) + FP8S_STAGING_BYTES + 1024;

struct Fp8ScaledParams {
    CUtensorMap map_x;       // {K, rows} box {128, 128}
    CUtensorMap map_w;       // NT {K, F}, NN {F, K}: box {128, 128}
    CUtensorMap map_xs;      // packed scales {16, 32 * tiles of 128 rows * K blocks}, box {16, 32}
    CUtensorMap map_ws;      // ... of W, box {16, 64}
    CUtensorMap map_c;       // {F, rows} box {128 bytes, 16}
    const float* bias;
    int act;
    void* c;
    int tma_store;
    int rows;
    int features;
    int k;
    int chunk_blocks;        // K blocks summed in the accumulator
    int tiles_m, tiles_n;
    const uint32_t* odd_scales;
    uint32_t* status;
    unsigned long long wait_limit_ns;
};

// Packed scales [K block][tile of 128][512 bytes] of x (rows of its own) and of w (one scale for 128 features), and a word per
// CTA that says whether any was not a positive power of two.
__global__ void __launch_bounds__(256) pack_scales_kernel(const float* __restrict__ x_scales, int rows, int row_tiles,
                                                          const float* __restrict__ w_scales, int feature_blocks, int feature_tiles,
                                                          long long ws_feature, long long ws_k, int k_blocks,
                                                          uint32_t* __restrict__ packed_x, uint32_t* __restrict__ packed_w,
                                                          uint32_t* __restrict__ odd) {
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    bool bad = false;
    auto pack = [&](float s) {
        const uint32_t bits = __float_as_uint(s);
        bad = bad || (bits & 0x807fffffu) != 0 || bits == 0 || bits == 0x7f800000u;
        return (bits >> 23) * 0x01010101u;
    };
    const int words_x = k_blocks * row_tiles * 128, words_w = k_blocks * feature_tiles * 128;
    for (int i = blockIdx.x * 256 + threadIdx.x; i < words_x; i += gridDim.x * 256) {
        // Neighbouring threads take neighbouring rows; their words lie 16 bytes apart.
        const int r = i & 127, tile = (i >> 7) % row_tiles, kb = (i >> 7) / row_tiles;
        const int row = tile * 128 + r;
        packed_x[(i & ~127) + 4 * (r & 31) + (r >> 5)] =
            row < rows ? pack(__ldg(x_scales + (long long)kb * rows + row)) : 0x7f7f7f7fu;
    }
    for (int i = blockIdx.x * 256 + threadIdx.x; i < words_w; i += gridDim.x * 256) {
        const int block = (i >> 7) % feature_tiles, kb = (i >> 7) / feature_tiles;
        packed_w[i] = block < feature_blocks ? pack(__ldg(w_scales + block * ws_feature + kb * ws_k)) : 0x7f7f7f7fu;
    }
    const int any = __syncthreads_or(bad ? 1 : 0);
    if (threadIdx.x == 0) odd[blockIdx.x] = any ? 1u : 0u;
}

template <RaggedForm FORM, class OutT>
__global__ void __launch_bounds__(FP8R_THREADS, 1) fp8_scaled_kernel(const __grid_constant__ Fp8ScaledParams p) {
#if defined(__CUDA_ARCH_FEAT_SM100_ALL) || defined(__CUDA_ARCH_FEAT_SM101_ALL) || \
    defined(__CUDA_ARCH_FEAT_SM103_ALL)
    constexpr bool B_MN = FORM == RaggedForm::NN;

    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bar_full[FP8S_STAGES];
    __shared__ __align__(8) uint64_t bar_empty[FP8S_STAGES];
    __shared__ __align__(8) uint64_t bar_acc_full;
    __shared__ __align__(8) uint64_t bar_acc_empty;
    __shared__ uint32_t tmem_base_holder;
    __shared__ uint32_t abort_flag;

    ptx::grid_dependency_wait();
    if (any_odd_scales(p.odd_scales)) return;
    const uint32_t warp = threadIdx.x >> 5;
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t cta_rank = ptx::cluster_ctarank();
    const bool is_leader = cta_rank == 0;
    const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t smem_staging = smem_base + FP8S_STAGES * FP8R_STAGE_BYTES;      // swizzled blocks: 1024-byte aligned
    const uint32_t smem_scales = smem_staging + FP8S_STAGING_BYTES;
    ptx::WaitCtx wctx{&abort_flag, p.status, p.wait_limit_ns};

    if (threadIdx.x == 0) {
        abort_flag = 0;
        ptx::prefetch_tensormap(&p.map_x);
        ptx::prefetch_tensormap(&p.map_w);
        ptx::prefetch_tensormap(&p.map_xs);
        ptx::prefetch_tensormap(&p.map_ws);
        ptx::prefetch_tensormap(&p.map_c);
        for (int s = 0; s < FP8S_STAGES; ++s) {
            ptx::mbar_init(ptx::smem_u32(&bar_full[s]), 1);
            ptx::mbar_init(ptx::smem_u32(&bar_empty[s]), 1);
        }
        ptx::mbar_init(ptx::smem_u32(&bar_acc_full), 1);
        ptx::mbar_init(ptx::smem_u32(&bar_acc_empty), 8 * 2);
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
                    const int feature = tn * 256 + int(cta_rank) * 128;
                    for (int kb = 0; kb < k_blocks; kb += FP8R_ATOMS) {
                        if (!ptx::mbar_wait(ptx::smem_u32(&bar_empty[stage]), phase ^ 1u, wctx, UMMA_TIMEOUT_PRODUCER))
                            goto producer_done;
                        const uint32_t full_local = ptx::smem_u32(&bar_full[stage]);
                        if (is_leader)
                            ptx::mbar_arrive_expect_tx(full_local, 2 * (FP8R_STAGE_BYTES + FP8R_ATOMS * FP8S_SCALE_BYTES));
                        const uint32_t full = ptx::mapa(full_local, 0);
#pragma unroll
                        for (int a = 0; a < FP8R_ATOMS; ++a) {      // a block behind the last one loads as zeros
                            const uint32_t a_smem = smem_base + stage * FP8R_STAGE_BYTES + a * FP8R_ATOM_BYTES;
                            const uint32_t s_smem = smem_scales + (stage * FP8R_ATOMS + a) * FP8S_SCALE_BYTES;
                            const int k0 = (kb + a) * FP8_BK;
                            ptx::tma_load_2d_pair(a_smem, &p.map_x, full, k0, row);
                            ptx::tma_load_2d_pair(a_smem + 16384, &p.map_w, full, B_MN ? feature : k0, B_MN ? k0 : feature);
                            // Each CTA needs the scales of its own rows and of all 256 features.
                            ptx::tma_load_2d_pair(s_smem, &p.map_xs, full, 0,
                                                  ((kb + a) * 2 * p.tiles_m + tm * 2 + int(cta_rank)) * 32);
                            ptx::tma_load_2d_pair(s_smem + 512, &p.map_ws, full, 0, ((kb + a) * 2 * p.tiles_n + tn * 2) * 32);
                        }
                        if (++stage == FP8S_STAGES) { stage = 0; phase ^= 1u; }
                    }
                }
            }
        producer_done:
            __syncwarp();
        } else if (warp == 1 && is_leader) {
            // -------------------------------------------------------- MMA issuer
            constexpr uint32_t B_KSTEP = B_MN ? 4096u : 32u;
            constexpr uint32_t idesc = ptx::idesc_mxf8(256, 256, 0, B_MN ? 1 : 0);
            const uint64_t a_desc0 = ptx::smem_desc_at(ptx::smem_desc(16, 1024, ptx::SMEM_LAYOUT_SW128), smem_base);
            const uint64_t b_desc0 =
                ptx::smem_desc_at(ptx::smem_desc(B_MN ? 16384 : 16, 1024, ptx::SMEM_LAYOUT_SW128), smem_base + 16384);
            const uint64_t s_desc0 = ptx::smem_desc_at(ptx::smem_desc(0, 128, 0), smem_scales);
            uint32_t stage = 0, phase = 0, it = 0;
            for (int u = first_unit; u < num_units; u += unit_stride) {
                for (int kb = 0; kb < k_blocks; ++kb) {
                    const bool first = kb % p.chunk_blocks == 0;
                    const bool last = kb + 1 == k_blocks || (kb + 1) % p.chunk_blocks == 0;
                    const uint32_t atom = uint32_t(kb) % FP8R_ATOMS;
                    const bool stage_done = atom + 1 == FP8R_ATOMS || kb + 1 == k_blocks;
                    if (atom == 0 && !__all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&bar_full[stage]), phase, wctx,
                                                                             UMMA_TIMEOUT_MMA_FULL)))
                        goto mma_done;
                    if (first && !__all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&bar_acc_empty), (it & 1) ^ 1u, wctx,
                                                                         UMMA_TIMEOUT_MMA_ACC)))
                        goto mma_done;
                    ptx::tc_fence_after();
                    if (ptx::elect_one()) {
                        const uint64_t offset = (stage * FP8R_STAGE_BYTES + atom * FP8R_ATOM_BYTES) >> 4;
                        const uint64_t s_block = s_desc0 + (((stage * FP8R_ATOMS + atom) * FP8S_SCALE_BYTES) >> 4);
                        // Columns 256 on: 4 for the scales of the rows, 8 for those of the features; each block of the ring its own.
                        const uint32_t s_tmem = tmem_base + 256u + (stage * FP8R_ATOMS + atom) * 16u;
                        ptx::tmem_cp_32x128b_pair(s_tmem, s_block);
                        ptx::tmem_cp_32x128b_pair(s_tmem + 4, s_block + (512u >> 4));
                        ptx::tmem_cp_32x128b_pair(s_tmem + 8, s_block + (1024u >> 4));
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            ptx::umma_mxf8<2>(tmem_base, a_desc0 + offset + ((kk * 32u) >> 4),
                                              b_desc0 + offset + ((kk * B_KSTEP) >> 4), idesc, s_tmem, s_tmem + 4,
                                              !(first && kk == 0));
                        if (last) {
                            const uint32_t accf_local = ptx::smem_u32(&bar_acc_full);
                            ptx::umma_commit<2>(accf_local);
                            ptx::umma_commit<2>(ptx::mapa(accf_local, 1));
                        }
                        if (stage_done) {
                            const uint32_t empty_local = ptx::smem_u32(&bar_empty[stage]);
                            ptx::umma_commit<2>(empty_local);
                            ptx::umma_commit<2>(ptx::mapa(empty_local, 1));
                        }
                    }
                    __syncwarp();
                    if (last) ++it;
                    if (stage_done && ++stage == FP8S_STAGES) { stage = 0; phase ^= 1u; }
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
        const uint32_t staging = smem_staging + (warp - 4) * 2048u;
        const uint32_t t_row = tmem_base + uint32_t(half) * 128u + ((quarter * 32u) << 16);
        const Fp8Activation act(p.act);
        uint32_t it = 0;
        for (int u = first_unit; u < num_units; u += unit_stride) {
            int tm, tn;
            raster_coords(u, p.tiles_m, p.tiles_n, 8, tm, tn);
            const int row0 = (tm * 2 + int(cta_rank)) * 128 + int(quarter) * 32;
            const int feature0 = tn * 256 + half * 128;
            float acc[4][32];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 32; ++j) acc[i][j] = 0.0f;
#pragma unroll 1
            for (int kb = 0; kb < k_blocks; kb += p.chunk_blocks, ++it) {
                const bool ok = ptx::mbar_wait(ptx::smem_u32(&bar_acc_full), it & 1, wctx, UMMA_TIMEOUT_EPILOGUE);
                if (!__all_sync(0xffffffffu, ok)) goto epilogue_done;
                ptx::tc_fence_after();
                uint32_t r[2][16];
                ptx::tmem_ld_32x16(t_row, r[0]);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    ptx::tmem_ld_wait(r[i & 1]);
                    if (i < 7) {
                        ptx::tmem_ld_32x16(t_row + 16 * (i + 1), r[(i + 1) & 1]);
                    } else {
                        ptx::tc_fence_before();
                        __syncwarp();
                        if (lane == 0) {
                            const uint32_t e = ptx::smem_u32(&bar_acc_empty);
                            if (is_leader) ptx::mbar_arrive(e);
                            else ptx::mbar_arrive_cluster_relaxed(ptx::mapa(e, 0));
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j) acc[i >> 1][(i & 1) * 16 + j] += __uint_as_float(r[i & 1][j]);
                }
            }
            store_tile<256, OutT, 16>(p, acc, act, staging, lane, row0, feature0);
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
