// Host side of the tensor-core kernels of the paged cache.
#pragma once

#include "dsdpa_host.h"
#include "dsdpa_cache.cuh"

namespace dsdpa {

// A call's work, as far as the host can know it (the lengths are on the device).
struct TreePlan {
    bool whole;              // units are not cut
    int row_tiles, part_rows, blocks;
    size_t part, part_lse, bytes;      // workspace: the table of starts at 0
};
inline TreePlan plan_tree(const dsdpa_cache_problem& p) {
    TreePlan t{};
    const long long room = (long long)p.table_width * p.page_size;
    const int rows = p.T * (p.Hq / p.Hkv);
    t.row_tiles = (rows + 127) / 128;
    t.part_rows = rows < 128 ? rows : 128;
    const long long units = (long long)p.B * p.Hkv * t.row_tiles, tiles = units * ((room + 127) / 128);
    // A cache of up to four key tiles is not worth a second kernel: a block goes through it while the launch
    // of one would take.
    t.whole = room <= 512;
    const long long most = t.whole ? units : (tiles + 1) / 2;     // a share has two key tiles at least
    t.blocks = (int)(most < kSMs ? most : kSMs);
    if (!t.whole) {
        auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
        t.part_lse = up(((size_t)p.B + 2) * 8);
        t.part = t.part_lse + up((size_t)t.blocks * 2 * t.part_rows * 4);
        t.bytes = t.part + (size_t)t.blocks * 2 * t.part_rows * p.D * 4;
    }
    return t;
}

template <typename T> cudaError_t launch_tree_tc(const CacheParams& p, const TreePlan& t, void* workspace, cudaStream_t s);
template <typename T> cudaError_t launch_weights_tc(const CacheParams& p, cudaStream_t s);

}  // namespace dsdpa
