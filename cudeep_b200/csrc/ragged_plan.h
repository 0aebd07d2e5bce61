// Tile choice and launch shared by the ragged and the 8-bit products.
#pragma once

#include "launch_dependent.h"
#include "umma_gemm.cuh"

#include <algorithm>
#include <cmath>
#include <map>
#include <mutex>
#include <tuple>

namespace cudeep_b200 {

struct RaggedPlan {
    int ctas;             // CTAs per tile
    int tile_cols;        // columns of a tile at most
    long long units;      // most tiles there can be, whatever the group sizes
    double cost;          // estimate in cycles
    int split = 1;        // CTAs that share a tile of one CTA, each with a range of the sums
    int step = 128;       // features of a CTA's tile
};

// An SM takes in about 41 bytes of operands a cycle from L2, 20 from HBM (measured: 16 KB boxes, all SMs loading), and a K
// block of 128 bytes per row costs two cycles of MMAs per column on 128 lanes.
constexpr double PLAN_L2_BYTES = 41.0, PLAN_HBM_BYTES = 20.0, PLAN_MMA_CYCLES = 2.0;

// Clusters of `size` CTAs of a kernel, an SM each, that the device runs at once: fewer than SMs / size, as a cluster lies within
// one part of the chip.  (148 CTAs as 37 clusters of four took two turns: 1 row, 4096 -> 4096 in 8 bits 13.2 us, 128 CTAs
// 8.1 us.)
inline int resident_clusters(const void* kernel, int size, int threads, size_t smem_bytes) {
    static std::mutex mu;
    static std::map<std::tuple<int, const void*, int>, int> known;
    const DeviceInfo& dev = device_info();
    if (size == 1) return dev.num_sms;
    std::lock_guard<std::mutex> lock(mu);
    const auto key = std::make_tuple(dev.device, kernel, size);
    const auto at = known.find(key);
    if (at != known.end()) return at->second;
    ensure_dynamic_smem(kernel, int(smem_bytes));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(size), 1, 1);
    cfg.blockDim = dim3(unsigned(threads), 1, 1);
    cfg.dynamicSmemBytes = smem_bytes;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(size);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int count = 0;
    CB200_CUDA(cudaOccupancyMaxActiveClusters(&count, kernel, &cfg));
    return known[key] = count < 1 ? 1 : count;
}

// Rows of `groups` groups, `rows` in all, on the columns of the tiles; `blocks` K blocks.  Sizes of the groups are not known
// here, so the cost of each choice is that of groups of equal size: waves of tiles, each its K blocks at the slower of
// loads and MMAs and a start and an end that nothing hides.  Weights that only one tile of a group reads come from HBM.
//
// Where there are few tiles (a token or two for each expert), clusters share them, if each cluster then has one at most
// (7 rows of 31 groups, 4096 -> 208: 23.4 us with a CTA to a tile, 7.8 us with eight; 1 row, 4096 -> 4096: 23.1 and 10.0 us).
// clusters(size): how many the device runs at once.
//
// Tiles of a single CTA that take all rows of a group may have fewer than 128 features, least_step at least, where that makes
// fuller waves (64 rows of 16 groups, 1024 -> 4096: 512 tiles of 128 are four waves on 148 SMs, and so are 592 of 112: 27.2 us
// and 26.0 us).
template <class Clusters>
RaggedPlan plan_rows(int groups, int rows, int features, int blocks, int least_step, Clusters clusters) {
    const int sms = device_info().num_sms;
    const int used = groups < rows ? groups : rows;
    const double size = double(rows) / used;
    const int most = (rows + 31) / 32 * 32;
    RaggedPlan best{2, 256, 0, 1e30};
    int fit[3] = {-1, -1, -1};
    auto consider = [&](int ctas, int step, int tile) {
        const long long f_tiles = (features + (long long)step * ctas - 1) / (step * ctas);
        const int per_group = int((size + tile - 1) / tile);
        const int width = int((size / per_group + 16 * ctas - 1) / (16 * ctas)) * 16 * ctas;
        // Uneven groups: the last tile of a group is half empty on average.
        const double tiles = double(f_tiles) * (groups == 1 ? per_group : used * (size / tile > 1 ? size / tile + 0.5 : 1.0));
        const double waves = std::ceil(tiles * ctas / sms);
        const double loads = step * 128 / (per_group == 1 ? PLAN_HBM_BYTES : PLAN_L2_BYTES) + width / ctas * 128 / PLAN_L2_BYTES;
        const double cost = waves * (blocks * std::max(loads, PLAN_MMA_CYCLES * width) + 2500.0 + 8.0 * width);
        if (cost < 0.97 * best.cost) best = RaggedPlan{ctas, tile, 0, cost, 1, step};
        if (ctas == 2 || tile > 128) return;      // the parts of a tile lie in the stages' memory
        for (int split = 2; split <= 8 && blocks >= 4 * split; split *= 2) {
            int& count = fit[split == 2 ? 0 : split == 4 ? 1 : 2];
            if (count < 0) count = clusters(split);
            if (f_tiles * (rows / std::min(tile, most) + used) > count) break;
            const double shared = (blocks + split - 1) / split * std::max(loads, PLAN_MMA_CYCLES * width) + 4500.0 + 28.0 * width;
            if (shared < 0.97 * best.cost) best = RaggedPlan{ctas, tile, 0, shared, split, step};
        }
    };
    for (int tile = 256; tile >= 32; tile /= 2) consider(2, 128, tile);
    for (int step = 128; step >= least_step; step -= 16)
        for (int tile = 256; tile >= 32 && (step == 128 || tile >= size); tile /= 2) consider(1, step, tile);
    if (best.tile_cols > most) best.tile_cols = most;
    best.units = (features + (long long)best.step * best.ctas - 1) / (best.step * best.ctas) * (rows / best.tile_cols + used);
    return best;
}

// Gradients of `groups` matrices: tiles of features x cols, summed over `rows` rows of all groups.  C leaves while the next
// tile is summed, at about 30 bytes a cycle and SM.
inline RaggedPlan plan_weight(int groups, int rows, int features, int cols, int c_bytes) {
    const int sms = device_info().num_sms;
    const double blocks = std::ceil(double(rows) / groups / 64);
    RaggedPlan best{2, 256, 0, 1e30};
    for (int ctas = 2; ctas >= 1; --ctas) {
        for (int tile = 256; tile >= 128; tile /= 2) {
            const long long tiles = (features + 128ll * ctas - 1) / (128 * ctas) * ((cols + tile - 1) / tile) * groups;
            const double waves = std::ceil(double(tiles) * ctas / sms);
            const double loads = (16384.0 + tile / ctas * 128) / PLAN_L2_BYTES;
            const double sums = blocks * std::max(loads, PLAN_MMA_CYCLES * tile), out = 128.0 * tile * c_bytes / 30.0;
            const double cost = waves * std::max(sums + 500.0, out) + std::min(sums, out) + 2500.0;
            if (cost < 0.97 * best.cost) best = RaggedPlan{ctas, tile, tiles, cost};
        }
    }
    return best;
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

}  // namespace cudeep_b200
