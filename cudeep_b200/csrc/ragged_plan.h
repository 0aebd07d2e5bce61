// Tile choice and launch shared by the ragged and the 8-bit products.
#pragma once

#include "umma_gemm.cuh"

namespace cudeep_b200 {

struct RaggedPlan {
    int ctas;             // CTAs per tile
    int tile_cols;        // columns of a tile at most
    long long units;      // most tiles there can be, whatever the group sizes
};

// Rows of `groups` groups, `rows` in all, on the columns of the tiles.
inline RaggedPlan plan_rows(int groups, int rows, int features) {
    const int sms = device_info().num_sms;
    RaggedPlan plan{features <= 128 ? 1 : 2, 256, 0};
    const long long f_tiles = (features + 128 * plan.ctas - 1) / (128 * plan.ctas);
    const int used = groups < rows ? groups : rows;
    for (int tile = 256; tile >= 32; tile /= 2) {
        plan.tile_cols = tile;
        // Each group that has rows ends in a partial tile: half a tile on average.
        const long long expected = f_tiles * (rows / tile + (used + 1) / 2);
        if (expected * plan.ctas >= sms) break;
    }
    const int most = (rows + 31) / 32 * 32;
    if (plan.tile_cols > most) plan.tile_cols = most;
    plan.units = f_tiles * (rows / plan.tile_cols + used);
    return plan;
}

template <class Kernel, class Params>
void launch_clusters(Kernel kernel, const Params& p, long long clusters, int cluster_size, int threads, uint32_t smem_bytes,
                     uint32_t smem_limit, cudaStream_t stream) {
    ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem_limit);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(clusters * cluster_size), 1, 1);
    cfg.blockDim = dim3(unsigned(threads), 1, 1);
    cfg.dynamicSmemBytes = smem_bytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int count = 0;
    if (cluster_size > 1) {
        attr[count].id = cudaLaunchAttributeClusterDimension;
        attr[count].val.clusterDim.x = unsigned(cluster_size);
        attr[count].val.clusterDim.y = 1;
        attr[count].val.clusterDim.z = 1;
        ++count;
    }
    if (programmatic_launch_enabled()) {
        attr[count].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[count].val.programmaticStreamSerializationAllowed = 1;
        ++count;
    }
    cfg.attrs = attr;
    cfg.numAttrs = unsigned(count);
    CB200_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
}

// A plain grid whose set-up may overlap the kernel before it (it must wait for it itself).
template <class... Params, class... Args>
void launch_dependent(void (*kernel)(Params...), dim3 grid, int threads, cudaStream_t stream, const Args&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(unsigned(threads), 1, 1);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = programmatic_launch_enabled() ? 1 : 0;
    CB200_CUDA(cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...));
}

}  // namespace cudeep_b200
