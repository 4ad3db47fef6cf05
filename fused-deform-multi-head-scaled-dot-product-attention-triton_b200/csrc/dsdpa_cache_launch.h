// Host side of the kernels over a paged cache.
#pragma once

#include "dsdpa_host.h"
#include "dsdpa_cache.cuh"

namespace dsdpa {

// The tensor-core kernels take 16-bit storage with up to 128 elements a row; fp32 arithmetic the rest.
inline bool cache_on_tensor_cores(const dsdpa_cache_problem& p) { return p.dtype != DSDPA_F32 && p.D <= 128; }

// A call's work, as far as the host can know it (the lengths are on the device).
struct TreePlan {
    bool whole;              // units are not cut
    int row_unit, row_tiles, part_rows, blocks, weight_blocks;
    size_t part, part_lse, bytes;      // workspace: the table of starts at 0
};
inline TreePlan plan_tree(const dsdpa_cache_problem& p) {
    TreePlan t{};
    const bool tc = cache_on_tensor_cores(p);
    const long long room = (long long)p.table_width * p.page_size;
    const int rows = p.T * (p.Hq / p.Hkv), keys = tc ? 128 : 64;
    t.row_unit = tc ? 128 : rows <= 16 ? 16 : p.D <= 128 ? 64 : 32;
    t.row_tiles = (rows + t.row_unit - 1) / t.row_unit;
    t.part_rows = rows < t.row_unit ? rows : t.row_unit;
    const long long units = (long long)p.B * p.Hkv * t.row_tiles, tiles = (room + keys - 1) / keys;
    // A cache of up to four key tiles is not worth a second kernel: a block goes through it while the launch
    // of one would take.
    t.whole = tiles <= 4;
    // as many blocks as stay on the SMs at once, but no share below two key tiles
    const long long stay = tc ? kSMs : p.D <= 64 ? 3 * kSMs : p.D <= 128 ? 2 * kSMs : kSMs;
    const long long most = t.whole ? units : (units * tiles + 1) / 2, most_weights = ((long long)p.B * p.Hkv * tiles + 1) / 2;
    t.blocks = (int)(most < stay ? most : stay);
    t.weight_blocks = (int)(most_weights < stay ? most_weights : stay);
    if (!t.whole) {
        auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
        t.part_lse = up(((size_t)p.B + 2) * 8);
        t.part = t.part_lse + up((size_t)t.blocks * 2 * t.part_rows * 4);
        t.bytes = t.part + (size_t)t.blocks * 2 * t.part_rows * p.D * 4;
    }
    return t;
}

template <typename T> cudaError_t launch_tree_tc(const CacheParams& p, const TreePlan& t, void* workspace, cudaStream_t s);
template <typename T> cudaError_t launch_tree_simt(const CacheParams& p, const TreePlan& t, void* workspace, cudaStream_t s);
template <typename T> cudaError_t launch_weights_tc(const CacheParams& p, const TreePlan& t, cudaStream_t s);
template <typename T> cudaError_t launch_weights_simt(const CacheParams& p, const TreePlan& t, cudaStream_t s);

}  // namespace dsdpa
