// Host side of what the kernels over a paged cache have in common.
#pragma once

#include "dsdpa_cache_launch.h"
#include "dsdpa_share.cuh"

namespace dsdpa {

inline TreeSplit tree_split(const TreePlan& t, void* workspace) {
    char* at = (char*)workspace;
    return TreeSplit{ t.whole, t.row_tiles, t.part_rows, (long long*)at, (float*)(at + t.part), (float*)(at + t.part_lse), t.parts * t.part_rows };
}

// The second kernel's blocks are in place when the first one's end, and wait for its results there.
template <typename T, typename Tile>
cudaError_t launch_combine(const CacheParams& p, const TreePlan& t, const TreeSplit& sp, cudaStream_t s) {
    cudaLaunchConfig_t cfg{};
    const long long rows = (long long)p.B * p.Hq * p.T;
    // parts of a row on average, from the workers of the first kernel: above a warp's 32 a block takes them together
    const bool spread = (long long)t.blocks * Tile::kWorkers > 32ll * p.B * p.Hkv * t.row_tiles;
    cfg.gridDim = dim3((unsigned)(spread ? rows : (rows + kCombineWarps - 1) / kCombineWarps));
    cfg.blockDim = dim3(kCombineWarps * 32);
    cfg.stream = s;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    const cudaError_t e = spread ? cudaLaunchKernelEx(&cfg, tree_combine_kernel<T, Tile, kCombineWarps>, p, sp) : cudaLaunchKernelEx(&cfg, tree_combine_kernel<T, Tile, 1>, p, sp);
    count_launches(1);
    return e;
}

}  // namespace dsdpa
