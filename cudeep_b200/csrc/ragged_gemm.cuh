// Products of ragged row groups with a weight per group, 16-bit operands, FP32 accumulation (tcgen05 kind::f16).
//
// Rows [offsets[g], offsets[g+1]) of a [rows, ...] matrix form group g.  Three products, with W[g] as Linear stores it:
//   NT  C[r, f] = sum_k X[r, k] W[g][f, k]        forward
//   NN  C[r, f] = sum_k X[r, k] W[g][k, f]        gradient of the rows
//   TN  C[g][f, c] = sum_{r in g} Y[r, f] X[r, c]  gradient of the weight
//
// The group sizes are known on the device only, so every CTA (or CTA pair) reads the offsets, makes the running
// count of tiles and walks its share of them; the grid never depends on the sizes and nothing is read back.
//
// NT and NN put the FEATURES on the accumulator's 128 (256 for a pair) lanes and the ROWS of the group on its
// columns.  The number of columns of one MMA is free (any multiple of 16 per CTA), so a group's ragged end costs at most
// 31 columns and a group of a few rows costs a narrow MMA, where lanes come in 128s only.  Rows behind a group's
// end that fall into its last columns are computed and not stored: they cannot reach another row's result.
//
// TN sums over the rows, so a row behind the group's end must not be multiplied at all (a zero on one side does not
// do: 0 * Inf = NaN).  Each group therefore has tensor maps of its own whose rows end with the group, made on the device by
// group_maps_kernel just before, and the TMA unit fills what lies behind with zeros in both operands.  (Bringing the last
// 16 rows with ordinary loads instead cost a cluster-scope release and acquire per tile: 8192 rows in 16 groups, 2048 x 2048,
// 129 us; 86 us this way.)
#pragma once

#include "device_flags.cuh"
#include "runtime.h"
#include "sm100_ptx.cuh"
#include "umma_gemm.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace cudeep_b200 {

enum class RaggedForm { NT, NN, TN };

constexpr int RAGGED_MAX_GROUPS = 1024;
constexpr int RAGGED_BK = 64;                        // 16-bit elements per K block = one 128-byte swizzle row
// With four epilogue warps a gradient tile of 512 summed rows took longer to leave than to compute.
constexpr int RAGGED_EPI_WARPS = 8;
constexpr int RAGGED_THREADS = 64 + 32 * RAGGED_EPI_WARPS;
// TN: a block of 32 rows x 128 bytes for each epilogue warp.  A second one would cost the third stage of two K blocks (8192 x
// 4096 x 4096: 232 us instead of 211).
constexpr uint32_t RAGGED_STAGING_BYTES = 8 * 4096;
// First and last row of each group, and the tiles before it, behind everything else in shared memory.
__host__ __device__ constexpr uint32_t ragged_table_bytes(int groups) { return uint32_t(3 * groups + 1) * 4u; }
constexpr uint32_t RAGGED_A_BYTES = 128 * 128;       // one CTA's features of a K block
constexpr int RAGGED_MAX_STAGES = 12;
constexpr uint32_t RAGGED_SMEM_BUDGET = 232448 - 1024 - 512;   // minus alignment slack and barriers
// The tensor core truncates as it adds: sums of positive FP16 products come out about 6e-9 of themselves too low per term (measured:
// 1.2e-5 after 2048 rows, 1.0e-4 after 16384; BF16, whose products have fewer bits to lose, 2.5e-6 after 2048).  So an FP32 result
// is summed over 2048 terms at a time, a 16-bit one over 16384, a fifth of FP16's half step, and such parts are added up in
// FP32 with rounding.
constexpr int RAGGED_F32_TERMS = 2048, RAGGED_F16_TERMS = 16384;
// The parts of a 16-bit result so far, of one CTA's tile: 128 columns x 32 lanes for each epilogue warp, in global memory.
constexpr size_t RAGGED_PARTIAL_FLOATS = RAGGED_EPI_WARPS * 128 * 32;
constexpr uint32_t UMMA_BAD_OFFSETS = 6;             // status word: the offsets decrease or leave [0, rows]

// Rows of a matrix as K blocks of 128 bytes.  One box brings all rows that a CTA stages for a tile, up to 128, rounded up to a
// size there is a map for: the TMA unit spends about 130 cycles on a box however small (2 KB boxes of 16 rows loaded
// a 112-row operand at a third of one 16 KB box's rate: 16384 x 4096 x 2048 in 224-row tiles 335 us, in 256-row tiles 183 us).
struct RowMaps {
    CUtensorMap box16;
    CUtensorMap box[4];      // 32, 64, 96, 128 rows
    __device__ __forceinline__ void prefetch() const {
        ptx::prefetch_tensormap(&box16);
        ptx::prefetch_tensormap(&box[3]);
    }
    // Rows that loads of `per` rows bring.
    __host__ __device__ static constexpr int loaded(int per) { return per <= 16 ? 16 : (per + 31) / 32 * 32; }
    template <int CTAS>
    __device__ __forceinline__ void load(uint32_t dst, uint32_t bar, int k0, int row, int per) const {
        for (int left = loaded(per); left > 0; left -= 128, row += 128, dst += 128 * 128) {
            const CUtensorMap* map = left == 16 ? &box16 : &box[left >= 128 ? 3 : left / 32 - 1];
            if constexpr (CTAS == 2) ptx::tma_load_2d_pair(dst, map, bar, k0, row);
            else ptx::tma_load_2d(dst, map, bar, k0, row);
        }
    }
};

struct RaggedParams {
    CUtensorMap map_a;       // NT {K, F, G} box {64, 128, 1}; NN as load_columns, and G; TN load_columns
    RowMaps x;               // NT, NN {K, rows}
    CUtensorMap map_b;       // TN see load_columns
    int a_chunked, b_chunked;
    CUtensorMap map_c;       // TN: {C, F, G} box {128 bytes, 32, 1}, where rows of C are 16-byte multiples
    int tma_store;           // ... and whether it is so
    const CUtensorMap* group_maps;      // TN: map_a and map_b of each group; nullptr: one group of all rows
    void* c;
    long long ldc;           // TN: elements between rows of C
    const int32_t* offsets;  // [groups + 1], or nullptr: `share` rows each, a multiple of 64 unless there is one group
    int share;
    int groups;
    int rows;                // rows of X (and of Y)
    int features;            // F
    int cols;                // TN: C
    int k;                   // NT, NN: length of the sums
    // NT, NN of single CTAs: CTAs per tile, a cluster, each with a range of the sums' blocks.  More than one only where every
    // cluster has one tile at most.
    int split;
    int step;                // features of a CTA's tile: 128; NT of single CTAs 64 to 128 (the last lanes then idle)
    int tile_cols;           // columns of a tile at most: rows of a group (NT, NN) or C (TN); <= 256
    int stages;
    uint32_t stage_bytes;
    // K blocks per stage, atom_bytes apart.  Two to a barrier instead of one: 8192 x 4096 x 4096 nt 214 -> 187 us.
    int atoms;
    uint32_t atom_bytes;
    int chunk_rows;          // TN: rows summed in the tensor core's accumulator before they are added into C or `partial`
    int chunk_blocks;        // NT, NN: K blocks likewise, a multiple of `atoms`
    float* partial;          // RAGGED_PARTIAL_FLOATS for each CTA, where a 16-bit result may take more than one chunk
    const float* col_scale;  // TN: nullptr, or a factor for each 128 columns of C
    // TN of one group, WIDE: if any of these words is set, X is BF16 and Y two BF16 matrices whose sum it is (WideOperands).  The sums
    // then run over 2 * part_rows rows, part_rows being `rows` rounded up to whole K blocks: those of the first part and those of
    // the second, each with the rows of X again.  wide_share takes the place of `share`.
    const uint32_t* wide;
    int wide_blocks;
    int part_rows;
    int wide_share;
    CUtensorMap map_parts;   // {64, rows, F / 64, 2} box {64, 64, 2, 1}
    uint32_t* status;
    unsigned long long wait_limit_ns;
};

// One tile: which group, its first feature and column, how many columns, and what it sums over.
struct RaggedTile {
    int group;
    int feature0;      // of the whole CTA group
    int col0;          // NT, NN: first row of X; TN: first column of C
    int col_count;     // real columns
    int umma_n;        // columns of the MMA
    int row0, row1;    // TN: rows of the group
};

template <RaggedForm FORM, int CTAS>
struct RaggedWalk {
    const int* off;
    const int* start;
    int groups, f_tiles, c_tiles_tn, tile_cols, features, cols, step;
    int g = 0;

    __device__ __forceinline__ int total() const { return start[groups]; }
    __device__ __forceinline__ RaggedTile at(int u) {
        while (u >= start[g + 1]) ++g;
        RaggedTile t;
        t.group = g;
        t.row0 = off[2 * g];
        t.row1 = off[2 * g + 1];
        const int in_group = u - start[g];
        int ct, ft;
        if (FORM == RaggedForm::TN) {
            raster_coords(in_group, f_tiles, c_tiles_tn, 8, ft, ct);
            t.col0 = ct * tile_cols;
            t.col_count = min(tile_cols, cols - t.col0);
            t.umma_n = tile_cols;
        } else {
            // Equal shares of the group's rows, so that no tile of it is much shorter than the others.
            const int size = t.row1 - t.row0;
            const int c_tiles = (size + tile_cols - 1) / tile_cols;
            constexpr int unit = 16 * CTAS;
            const int share = ((size + c_tiles - 1) / c_tiles + unit - 1) / unit * unit;
            raster_coords(in_group, c_tiles, f_tiles, 8, ct, ft);
            t.col0 = t.row0 + ct * share;
            t.col_count = min(share, t.row1 - t.col0);
            t.umma_n = max(unit, (t.col_count + unit - 1) / unit * unit);
        }
        t.feature0 = ft * step * CTAS;
        return t;
    }
};

template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// A warp's block of 32 rows x 128 bytes in shared memory, 16-byte unit q of row r at q ^ (r & 7) (the 128-byte swizzle of a
// tensor map): lane `lane` writes 32 values of its row from column `col` of the block on, rounded to T.
template <class T>
__device__ __forceinline__ void stage_block(uint32_t block, uint32_t lane, int col, const float (&v)[32]) {
    constexpr int V = 16 / sizeof(T);
#pragma unroll
    for (int j = 0; j < 32; j += V) {
        const uint32_t dst = block + lane * 128u + (((uint32_t(col + j) / V) ^ (lane & 7u)) << 4);
        if constexpr (sizeof(T) == 4)
            ptx::st_shared_v4(dst, v[j], v[j + 1], v[j + 2], v[j + 3]);
        else
            ptx::st_shared_u4(dst, pack2<T>(v[j], v[j + 1]), pack2<T>(v[j + 2], v[j + 3]), pack2<T>(v[j + 4], v[j + 5]),
                              pack2<T>(v[j + 6], v[j + 7]));
    }
}

// Writes (or adds: FP32) the first `rows` rows and `cols` columns of such a block to dst, whole warp, row by row.
template <class T>
__device__ __forceinline__ void write_block(uint32_t block, uint32_t lane, T* dst, long long ld, int rows, int cols, bool add) {
    for (int r = 0; r < rows; ++r, dst += ld) {
#pragma unroll
        for (int h = 0; h < int(128 / sizeof(T)) / 32; ++h) {
            const int c = int(lane) + 32 * h;
            const uint32_t byte = uint32_t(c) * sizeof(T);
            const uint32_t at = block + uint32_t(r) * 128u + (((byte >> 4) ^ (uint32_t(r) & 7u)) << 4) + (byte & 15u);
            if (c < cols) {
                if constexpr (sizeof(T) == 4) {
                    const float v = ptx::ld_shared_f32(at);
                    dst[c] = add ? dst[c] + v : v;
                } else {
                    reinterpret_cast<uint16_t*>(dst)[c] = ptx::ld_shared_u16(at);
                }
            }
        }
    }
    __syncwarp();
}

// One warp: the row range of each group, brought into [0, rows] (without offsets: `share` rows each), and the number of tiles
// before it.  col_tiles >= 0: column tiles of every group (TN); otherwise -col_tiles is the number of a group's rows that a
// tile takes.
__device__ __forceinline__ void group_tables(const int32_t* offsets, int groups, int rows, int share, int f_tiles, int col_tiles,
                                             int* group_rows, int* group_start, uint32_t* status) {
    const int lane = int(threadIdx.x & 31);
    int carry = 0;
    bool bad = false;
    for (int base = 0; base < groups; base += 32) {
        const int g = base + lane;
        int tiles = 0;
        if (g < groups) {
            int lo, hi;
            if (offsets != nullptr) {
                lo = __ldg(offsets + g);
                hi = __ldg(offsets + g + 1);
            } else {
                lo = int(min((long long)rows, (long long)g * share));
                hi = int(min((long long)rows, (long long)(g + 1) * share));
            }
            const int lo_in = min(max(lo, 0), rows), hi_in = min(max(hi, lo_in), rows);
            bad = bad || lo_in != lo || hi_in != hi;      // nothing is read or written outside the matrices
            group_rows[2 * g] = lo_in;
            group_rows[2 * g + 1] = hi_in;
            tiles = f_tiles * (col_tiles >= 0 ? col_tiles : (hi_in - lo_in - col_tiles - 1) / -col_tiles);
        }
        int sum = tiles;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int other = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d) sum += other;
        }
        if (g < groups) group_start[g + 1] = carry + sum;
        carry += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) group_start[0] = 0;
    if (__any_sync(0xffffffffu, bad) && lane == 0) atomicCAS(status, 0u, UMMA_BAD_OFFSETS);
}

template <class T>
__device__ __forceinline__ T round_to(float v);
template <>
__device__ __forceinline__ float round_to<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half round_to<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 round_to<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 64 rows of `chunks` times 64 columns, each chunk 64 rows of 128 bytes.  Where the rows hold whole chunks the map is
// {64, rows, columns / 64} with all chunks in one box; otherwise {columns, rows} with one chunk per box (a map by chunks would
// read past the last row's end).
template <int CTAS>
__device__ __forceinline__ void load_columns(uint32_t dst, const CUtensorMap* map, int chunked, int chunks, uint32_t bar, int col,
                                             int row) {
    if (chunked) {
        if constexpr (CTAS == 2) ptx::tma_load_3d_pair(dst, map, bar, 0, row, col / 64);
        else ptx::tma_load_3d(dst, map, bar, 0, row, col / 64);
        return;
    }
    for (int j = 0; j < chunks; ++j) {
        if constexpr (CTAS == 2) ptx::tma_load_2d_pair(dst + j * 8192, map, bar, col + j * 64, row);
        else ptx::tma_load_2d(dst + j * 8192, map, bar, col + j * 64, row);
    }
}

// 32 columns of a chunk's sums: with those of the chunks before it (`add`), kept for the next chunk unless this is the last one.
// `part` is the lane's place in the CTA's partial sums; a lane meets only what it wrote itself.
__device__ __forceinline__ void join_chunks(float* part, uint32_t (&r)[32], bool add, bool last) {
    if (add) {
#pragma unroll
        for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) + part[32 * j]);
    }
    if (!last) {
#pragma unroll
        for (int j = 0; j < 32; ++j) part[32 * j] = __uint_as_float(r[j]);
    }
}

// WIDE: the operands may come in the form of RaggedParams::wide.  A kernel of its own, as reading the flags and the test in the
// producer's loop cost 3.5 us of 195 in 8192 x 4096 x 4096.  LONG: 16-bit results of more than one chunk, which a kernel that
// has the code for them pays with 0.2 us even where it is not reached (7.8 us for 300 rows, 1024 -> 640).
template <RaggedForm FORM, int CTAS, bool BF16, class OutT, bool WIDE = false, bool LONG = false>
__global__ void __launch_bounds__(RAGGED_THREADS, 1) ragged_gemm_kernel(const __grid_constant__ RaggedParams p) {
#if defined(__CUDA_ARCH_FEAT_SM100_ALL) || defined(__CUDA_ARCH_FEAT_SM101_ALL) || \
    defined(__CUDA_ARCH_FEAT_SM103_ALL)
    constexpr bool A_MN = FORM != RaggedForm::NT;
    constexpr bool B_MN = FORM == RaggedForm::TN;

    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bar_full[RAGGED_MAX_STAGES];
    __shared__ __align__(8) uint64_t bar_empty[RAGGED_MAX_STAGES];
    __shared__ __align__(8) uint64_t bar_acc_full[2];
    __shared__ __align__(8) uint64_t bar_acc_empty[2];
    __shared__ uint32_t tmem_base_holder;
    __shared__ uint32_t abort_flag;

    const uint32_t warp = threadIdx.x >> 5;
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t cta_rank = CTAS == 2 ? ptx::cluster_ctarank() : 0u;
    const bool is_leader = cta_rank == 0;
    const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    int* group_rows = reinterpret_cast<int*>(smem_raw + (smem_base - ptx::smem_u32(smem_raw)) +
                                             uint32_t(p.stages) * p.stage_bytes + (FORM == RaggedForm::TN ? RAGGED_STAGING_BYTES : 0u));
    int* group_start = group_rows + 2 * p.groups;
    ptx::WaitCtx wctx{&abort_flag, p.status, p.wait_limit_ns};

    if (threadIdx.x == 0) {
        abort_flag = 0;
        ptx::prefetch_tensormap(&p.map_a);
        if constexpr (FORM == RaggedForm::TN) {
            ptx::prefetch_tensormap(&p.map_b);
            ptx::prefetch_tensormap(&p.map_c);
        } else {
            p.x.prefetch();
        }
        for (int s = 0; s < RAGGED_MAX_STAGES; ++s) {
            ptx::mbar_init(ptx::smem_u32(&bar_full[s]), CTAS);      // each CTA's producer arrives with its bytes
            ptx::mbar_init(ptx::smem_u32(&bar_empty[s]), 1);
        }
        for (int a = 0; a < 2; ++a) {
            ptx::mbar_init(ptx::smem_u32(&bar_acc_full[a]), 1);
            ptx::mbar_init(ptx::smem_u32(&bar_acc_empty[a]), RAGGED_EPI_WARPS * CTAS);
        }
        ptx::fence_mbar_init();
    }
    if (warp == 1) {
        ptx::tmem_alloc<CTAS>(ptx::smem_u32(&tmem_base_holder), 512);
        ptx::tmem_relinquish<CTAS>();
    }
    constexpr bool SPLITS = FORM != RaggedForm::TN && CTAS == 1;
    const int split = SPLITS ? p.split : 1;
    const int split_rank = SPLITS && split > 1 ? int(ptx::cluster_ctarank()) : 0;
    ptx::grid_dependency_wait();      // the offsets may come from the kernel before
    bool wide = false;
    if constexpr (WIDE) wide = any_set(p.wide, p.wide_blocks);
    constexpr bool STEPS = FORM == RaggedForm::NT && CTAS == 1;
    const int step = STEPS ? p.step : 128;
    const int f_tiles = (p.features + step * CTAS - 1) / (step * CTAS);
    const int c_tiles_tn = FORM == RaggedForm::TN ? (p.cols + p.tile_cols - 1) / p.tile_cols : 0;
    if (warp == 0)
        group_tables(p.offsets, p.groups, WIDE && wide ? 2 * p.part_rows : p.rows, WIDE && wide ? p.wide_share : p.share, f_tiles, FORM == RaggedForm::TN ? c_tiles_tn : -p.tile_cols, group_rows,
                     group_start, p.status);
    ptx::tc_fence_before();
    __syncthreads();
    if (CTAS == 2) {
        ptx::cluster_arrive();
        ptx::cluster_wait();
    }
    ptx::tc_fence_after();
    const uint32_t tmem_base = tmem_base_holder;
    ptx::grid_launch_dependents();

    const int first_unit = int(blockIdx.x) / (CTAS * split);
    RaggedWalk<FORM, CTAS> walk{group_rows, group_start, p.groups, f_tiles, c_tiles_tn, p.tile_cols, p.features, p.cols, step};
    const int num_units = walk.total();
    // A split tile is its cluster's only one (with bad offsets there may be more tiles: those are left out).
    const int unit_stride = split > 1 ? num_units : int(gridDim.x) / CTAS;
    // Blocks of this CTA's sums, k_first on; a split tile's last CTAs may have none.
    const int k_blocks_all = FORM == RaggedForm::TN ? 0 : (p.k + RAGGED_BK - 1) / RAGGED_BK;
    const int k_share = split > 1 ? ((k_blocks_all + split - 1) / split + p.atoms - 1) / p.atoms * p.atoms : k_blocks_all;
    const int k_first = min(k_blocks_all, split_rank * k_share);
    const int k_blocks_row = min(k_share, k_blocks_all - k_first);
    // TN: blocks of a chunk of the group's rows that starts at `row`.
    auto chunk_blocks = [&](const RaggedTile& t, int row) {
        return (min(p.chunk_rows, t.row1 - row) + RAGGED_BK - 1) / RAGGED_BK;
    };

    if (warp == 0) {
        // ------------------------------------------------------------ producer
        uint32_t stage = 0, phase = 0;
        for (int u = first_unit; u < num_units; u += unit_stride) {
            const RaggedTile t = walk.at(u);
            const int per = t.umma_n / CTAS;                               // columns this CTA stages
            const int feature = t.feature0 + int(cta_rank) * 128;
            const int col = t.col0 + int(cta_rank) * per;
            const int blocks = FORM == RaggedForm::TN ? (t.row1 - t.row0 + RAGGED_BK - 1) / RAGGED_BK : k_blocks_row;
            const CUtensorMap* map_a = &p.map_a;
            const CUtensorMap* map_b = &p.map_b;
            if (FORM == RaggedForm::TN && p.group_maps != nullptr) {
                map_a = p.group_maps + 2 * t.group;
                map_b = map_a + 1;
                if (lane == 0) {
                    ptx::tensormap_acquire(map_a);
                    ptx::tensormap_acquire(map_b);
                }
            }
            for (int kb = 0; kb < blocks; kb += p.atoms) {
                const bool ok = ptx::mbar_wait(ptx::smem_u32(&bar_empty[stage]), phase ^ 1u, wctx, UMMA_TIMEOUT_PRODUCER);
                if (!__all_sync(0xffffffffu, ok)) goto producer_done;
                const uint32_t full_local = ptx::smem_u32(&bar_full[stage]);
                const uint32_t full = CTAS == 2 ? ptx::mapa(full_local, 0) : full_local;
                const uint32_t atom = (STEPS ? uint32_t(step) * 128u : RAGGED_A_BYTES) + uint32_t(FORM == RaggedForm::TN ? per : RowMaps::loaded(per)) * 128u;
                if (lane == 0) {
                    // Blocks behind the last one load as zeros or are not multiplied.
                    for (int a = 0; a < p.atoms; ++a) {
                        const uint32_t a_smem = smem_base + stage * p.stage_bytes + a * p.atom_bytes;
                        const uint32_t b_smem = a_smem + RAGGED_A_BYTES;
                        const int k0 = (k_first + kb + a) * RAGGED_BK;
                        if constexpr (FORM == RaggedForm::NT) {
                            if constexpr (CTAS == 2) ptx::tma_load_3d_pair(a_smem, &p.map_a, full, k0, feature, t.group);
                            else ptx::tma_load_3d(a_smem, &p.map_a, full, k0, feature, t.group);
                        } else if constexpr (FORM == RaggedForm::NN) {
                            if (p.a_chunked) {
                                if constexpr (CTAS == 2)
                                    ptx::tma_load_4d_pair(a_smem, &p.map_a, full, 0, k0, feature / 64, t.group);
                                else
                                    ptx::tma_load_4d(a_smem, &p.map_a, full, 0, k0, feature / 64, t.group);
                            } else {
#pragma unroll
                                for (int j = 0; j < 2; ++j) {
                                    if constexpr (CTAS == 2)
                                        ptx::tma_load_3d_pair(a_smem + j * 8192, &p.map_a, full, feature + j * 64, k0, t.group);
                                    else
                                        ptx::tma_load_3d(a_smem + j * 8192, &p.map_a, full, feature + j * 64, k0, t.group);
                                }
                            }
                        } else {
                            int row = t.row0 + k0;
                            if (WIDE && wide) {
                                const int part = row >= p.part_rows ? 1 : 0;
                                row -= part * p.part_rows;
                                if constexpr (CTAS == 2) ptx::tma_load_4d_pair(a_smem, &p.map_parts, full, 0, row, feature / 64, part);
                                else ptx::tma_load_4d(a_smem, &p.map_parts, full, 0, row, feature / 64, part);
                            } else {
                                load_columns<CTAS>(a_smem, map_a, p.a_chunked, 2, full, feature, row);
                            }
                            load_columns<CTAS>(b_smem, map_b, p.b_chunked, per / 64, full, col, row);
                        }
                        if constexpr (FORM != RaggedForm::TN) p.x.template load<CTAS>(b_smem, full, k0, col, per);
                    }
                    const uint32_t bytes = uint32_t(p.atoms) * atom;
                    if (is_leader) ptx::mbar_arrive_expect_tx(full_local, bytes);
                    else ptx::mbar_arrive_expect_tx_cluster_relaxed(full, bytes);
                }
                __syncwarp();
                if (++stage == uint32_t(p.stages)) { stage = 0; phase ^= 1u; }
            }
        }
    producer_done:
        __syncwarp();
        if (CTAS == 2) ptx::cluster_arrive();
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer
        if (is_leader) {
            constexpr uint32_t KSTEP_MN = 2048u, KSTEP_K = 32u;
            const uint64_t a_desc0 = ptx::smem_desc_at(
                A_MN ? ptx::smem_desc(8192, 1024, ptx::SMEM_LAYOUT_SW128) : ptx::smem_desc(16, 1024, ptx::SMEM_LAYOUT_SW128),
                smem_base);
            const uint64_t b_desc0 = ptx::smem_desc_at(
                B_MN ? ptx::smem_desc(8192, 1024, ptx::SMEM_LAYOUT_SW128) : ptx::smem_desc(16, 1024, ptx::SMEM_LAYOUT_SW128),
                smem_base + RAGGED_A_BYTES);
            uint32_t stage = 0, phase = 0;
            int it = 0;      // accumulators handed over
            for (int u = first_unit; u < num_units; u += unit_stride) {
                const RaggedTile t = walk.at(u);
                const uint32_t idesc = ptx::idesc_f16(128 * CTAS, t.umma_n, A_MN ? 1 : 0, B_MN ? 1 : 0, BF16 || (WIDE && wide) ? 1 : 0);
                int row = t.row0, k_done = 0;
                do {
                    const int blocks = FORM == RaggedForm::TN ? chunk_blocks(t, row) : LONG ? min(p.chunk_blocks, k_blocks_row - k_done) : k_blocks_row;
                    if (blocks <= 0) break;
                    const uint32_t acc = it & 1;
                    const uint32_t acc_phase = (it >> 1) & 1;
                    if (!__all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&bar_acc_empty[acc]), acc_phase ^ 1u, wctx,
                                                                UMMA_TIMEOUT_MMA_ACC)))
                        goto mma_done;
                    ptx::tc_fence_after();
                    const uint32_t d_tmem = tmem_base + acc * 256u;
                    bool ready = __all_sync(0xffffffffu, ptx::mbar_test(ptx::smem_u32(&bar_full[stage]), phase));
                    for (int kb = 0; kb < blocks; kb += p.atoms) {
                        if (!ready &&
                            !__all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&bar_full[stage]), phase, wctx,
                                                                    UMMA_TIMEOUT_MMA_FULL)))
                            goto mma_done;
                        ptx::tc_fence_after();
                        uint32_t next_stage = stage + 1, next_phase = phase;
                        if (next_stage == uint32_t(p.stages)) { next_stage = 0; next_phase ^= 1u; }
                        ready = __all_sync(0xffffffffu, ptx::mbar_test(ptx::smem_u32(&bar_full[next_stage]), next_phase));
                        if (ptx::elect_one()) {
                            const uint64_t a_stage = a_desc0 + ((stage * p.stage_bytes) >> 4);
                            const uint64_t b_stage = b_desc0 + ((stage * p.stage_bytes) >> 4);
                            for (int a = 0; a < p.atoms; ++a) {
                                int steps = kb + a < blocks ? 4 : 0;
                                if (FORM == RaggedForm::TN)
                                    steps = max(0, min(steps, (t.row1 - row - (kb + a) * RAGGED_BK + 15) / 16));
                                const uint64_t offset = (a * p.atom_bytes) >> 4;
#pragma unroll
                                for (int kk = 0; kk < 4; ++kk)
                                    if (kk < steps)
                                        ptx::umma_f16<CTAS>(d_tmem, a_stage + offset + ((kk * (A_MN ? KSTEP_MN : KSTEP_K)) >> 4),
                                                            b_stage + offset + ((kk * (B_MN ? KSTEP_MN : KSTEP_K)) >> 4), idesc,
                                                            (kb | a | kk) != 0);
                            }
                            const uint32_t empty_local = ptx::smem_u32(&bar_empty[stage]);
                            ptx::umma_commit<CTAS>(empty_local);
                            if constexpr (CTAS == 2) ptx::umma_commit<CTAS>(ptx::mapa(empty_local, 1));
                            if (kb + p.atoms >= blocks) {
                                const uint32_t accf_local = ptx::smem_u32(&bar_acc_full[acc]);
                                ptx::umma_commit<CTAS>(accf_local);
                                if constexpr (CTAS == 2) ptx::umma_commit<CTAS>(ptx::mapa(accf_local, 1));
                            }
                        }
                        __syncwarp();
                        stage = next_stage;
                        phase = next_phase;
                    }
                    ++it;
                    row += p.chunk_rows;
                    k_done += p.chunk_blocks;
                } while (FORM == RaggedForm::TN ? row < t.row1 : LONG && k_done < k_blocks_row);
            }
        }
    mma_done:
        __syncwarp();
        if (CTAS == 2) ptx::cluster_arrive();
    } else {
        // ------------------------------------------------------------ epilogue
        const uint32_t quarter = warp & 3u;
        float* partial = p.partial + (size_t(blockIdx.x) * RAGGED_EPI_WARPS + (warp - 2)) * (128 * 32) + lane;
        int it = 0;
        for (int u = first_unit; u < num_units; u += unit_stride) {
            const RaggedTile t = walk.at(u);
            if constexpr (FORM == RaggedForm::TN) {
                // A chunk's sums leave as blocks of 32 features x 128 bytes, staged in shared memory: by a tensor store (the
                // later chunks of an FP32 gradient by a tensor reduction, an FP32 addition in L2; each element has this one
                // writer, in order), or, where rows of C are no 16-byte multiples, row by row.
                const int feature_w = t.feature0 + int(cta_rank) * 128 + int(quarter) * 32;
                const uint32_t staging =
                    smem_base + uint32_t(p.stages) * p.stage_bytes + (warp - 2) * 4096u;
                constexpr int COLS = 128 / sizeof(OutT);
                const int c_begin = (int(warp - 2) >> 2) * (t.umma_n / 2);      // warps 6..9 take the second half of the columns
                const int c_end = min(t.col_count, c_begin + t.umma_n / 2);
                int row = t.row0;
                do {
                    const bool any = chunk_blocks(t, row) > 0;       // an empty group's gradient is zero
                    const bool first = row == t.row0, last = !LONG || t.row1 - row <= p.chunk_rows;
                    const bool add = sizeof(OutT) == 4 && !first;      // into C
                    const uint32_t acc = it & 1;
                    if (any) {
                        const bool ok = ptx::mbar_wait(ptx::smem_u32(&bar_acc_full[acc]), (it >> 1) & 1, wctx, UMMA_TIMEOUT_EPILOGUE);
                        if (!__all_sync(0xffffffffu, ok)) goto epilogue_done;
                        ptx::tc_fence_after();
                    }
                    if (add && lane == 0) ptx::bulk_wait_group<0>();      // the chunk before has arrived in C
                    __syncwarp();
                    const uint32_t t_row = tmem_base + acc * 256u + ((quarter * 32u) << 16);
                    for (int c = c_begin; c < c_end; c += 32) {
                        uint32_t r[32];
                        if (any) {
                            ptx::tmem_ld_32x32(t_row + c, r);
                            ptx::tmem_ld_wait(r);
                        } else {
#pragma unroll
                            for (int j = 0; j < 32; ++j) r[j] = 0u;
                        }
                        if (LONG && !(first && last)) {
                            join_chunks(partial + (c - c_begin) * 32, r, !first, last);
                            if (!last) continue;
                        }
                        const float scale = p.col_scale != nullptr && !(WIDE && wide) ? __ldg(p.col_scale + (t.col0 + c) / 128) : 1.0f;
                        const int c0 = c / COLS * COLS;
                        if (c == c0) {      // the last store has read the block
                            if (lane == 0) ptx::bulk_wait_group_read<0>();
                            __syncwarp();
                        }
                        float v[32];
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]) * scale;
                        stage_block<OutT>(staging, lane, c - c0, v);
                        if (c + 32 - c0 == COLS || c + 32 >= c_end) {
                            if (p.tma_store) {
                                ptx::fence_proxy_async_smem();
                                __syncwarp();
                                if (lane == 0 && feature_w < p.features) {
                                    if (add) ptx::tma_reduce_add_3d(&p.map_c, staging, t.col0 + c0, feature_w, t.group);
                                    else ptx::tma_store_3d(&p.map_c, staging, t.col0 + c0, feature_w, t.group);
                                    ptx::bulk_commit_group();
                                }
                            } else {
                                __syncwarp();
                                OutT* dst = static_cast<OutT*>(p.c) +
                                            ((long long)t.group * p.features + feature_w) * p.ldc + t.col0 + c0;
                                write_block<OutT>(staging, lane, dst, p.ldc, min(32, p.features - feature_w), c_end - c0, add);
                            }
                        }
                    }
                    if (any) {
                        ptx::tc_fence_before();
                        __syncwarp();
                        if (lane == 0) {
                            const uint32_t e = ptx::smem_u32(&bar_acc_empty[acc]);
                            if (CTAS == 2 && !is_leader) ptx::mbar_arrive_cluster_relaxed(ptx::mapa(e, 0));
                            else ptx::mbar_arrive(e);
                        }
                        ++it;
                    }
                    row += p.chunk_rows;
                } while (row < t.row1);
            } else {
                const int feature = t.feature0 + int(cta_rank) * 128 + int(quarter) * 32 + int(lane);
                const int f_end = STEPS ? min(p.features, t.feature0 + step) : p.features;
                const int c_half = (t.umma_n / 2 + 31) / 32 * 32;      // warps 6..9 take the second half of the columns
                const int c_begin = (int(warp - 2) >> 2) * c_half, c_end = min(t.col_count, c_begin + c_half);
                const bool shared = SPLITS && split > 1;
                // The stage ring is idle once the last MMA is done: it takes this CTA's part, [column][128 features].
                const uint32_t part = smem_base + (quarter * 32u + lane) * 4u;
                OutT* dst = static_cast<OutT*>(p.c) + (long long)t.col0 * p.features + feature;
                int k_done = 0;
                do {
                    const bool any = k_blocks_row > 0;      // a split tile's last CTAs may have nothing to sum
                    const bool first = k_done == 0, last = !LONG || k_blocks_row - k_done <= p.chunk_blocks;
                    const uint32_t acc = it & 1;
                    if (any) {
                        const bool ok = ptx::mbar_wait(ptx::smem_u32(&bar_acc_full[acc]), (it >> 1) & 1, wctx, UMMA_TIMEOUT_EPILOGUE);
                        if (!__all_sync(0xffffffffu, ok)) goto epilogue_done;
                        ptx::tc_fence_after();
                    }
                    const uint32_t t_row = tmem_base + acc * 256u + ((quarter * 32u) << 16);
                    for (int c = c_begin; c < c_end; c += 32) {
                        uint32_t r[32];
                        if (any) {
                            ptx::tmem_ld_32x32(t_row + c, r);
                            ptx::tmem_ld_wait(r);
                        } else {
#pragma unroll
                            for (int j = 0; j < 32; ++j) r[j] = 0u;
                        }
                        if (LONG && !(first && last)) {
                            join_chunks(partial + (c - c_begin) * 32, r, !first, last);
                            if (!last) continue;
                        }
                        if (shared) {
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (c + j < c_end) ptx::st_shared_f32(part + uint32_t(c + j) * 512u, __uint_as_float(r[j]));
                        } else if (feature < f_end) {
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (c + j < c_end)
                                    dst[(long long)(c + j) * p.features] = round_to<OutT>(__uint_as_float(r[j]));
                        }
                    }
                    ptx::tc_fence_before();
                    __syncwarp();
                    if (any && lane == 0) {
                        const uint32_t e = ptx::smem_u32(&bar_acc_empty[acc]);
                        if (CTAS == 2 && !is_leader) ptx::mbar_arrive_cluster_relaxed(ptx::mapa(e, 0));
                        else ptx::mbar_arrive(e);
                    }
                    ++it;
                    k_done += p.chunk_blocks;
                } while (LONG && k_done < k_blocks_row);
            }
        }
    epilogue_done:
        __syncwarp();
        if (CTAS == 2) ptx::cluster_arrive();
        if (FORM == RaggedForm::TN && lane == 0) ptx::bulk_wait_group_read<0>();      // bulk stores still read shared memory
        __syncwarp();
    }

    if constexpr (SPLITS) {
        if (split > 1) {
            __syncwarp();
            ptx::cluster_arrive();
            ptx::cluster_wait();
            if (warp >= 2 && first_unit < num_units) {
                // Rank r finishes columns r, r + split, ...: a warp a column, four features a lane, the parts in rank order.
                const RaggedTile t = walk.at(first_unit);
                const int f = t.feature0 + 4 * int(lane), f_end = STEPS ? min(p.features, t.feature0 + step) : p.features;
                for (int c = split_rank + split * int(warp - 2); c < t.col_count; c += split * RAGGED_EPI_WARPS) {
                    float v[4] = {};
                    for (int r = 0; r < split; ++r) {
                        const float4 q = ptx::ld_cluster_v4(ptx::mapa(smem_base + uint32_t(c) * 512u + lane * 16u, uint32_t(r)));
                        v[0] += q.x;
                        v[1] += q.y;
                        v[2] += q.z;
                        v[3] += q.w;
                    }
                    OutT* dst = static_cast<OutT*>(p.c) + (long long)(t.col0 + c) * p.features + f;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (f + j < f_end) dst[j] = round_to<OutT>(v[j]);
                }
            }
            __syncwarp();
            ptx::cluster_arrive();      // nobody leaves while its part may still be read
            ptx::cluster_wait();
        }
    }

    // ---------------------------------------------------------------- teardown
    ptx::tc_fence_before();
    __syncthreads();
    if (abort_flag) {
        // A wait ran out: copies still in flight get a bounded time to land before the shared memory goes.
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
