// Host side of the tensor-core kernels of the paged cache.
#pragma once

#include "dsdpa_host.h"
#include "dsdpa_cache.cuh"

namespace dsdpa {

// How a call's keys are split: chunks of `chunk` keys, of which the longest sequence that the table holds has `chunks`.
struct TreePlan {
    int chunk, chunks, row_tiles, items;
    size_t part, bytes;      // workspace: chunk lse at 0, chunk results at `part`
};
inline TreePlan plan_tree(const dsdpa_cache_problem& p) {
    TreePlan t{};
    const long long room = (long long)p.table_width * p.page_size;
    const int rows = p.T * (p.Hq / p.Hkv);
    t.row_tiles = (rows + 127) / 128;
    const long long units = (long long)p.B * p.Hkv * t.row_tiles;
    // A chunk's results (4 D bytes a row, written and read) stay below a sixteenth of its keys and values (4 D bytes a
    // key); chunks get shorter as long as there are fewer than two for every SM; a cache of one or two tiles is
    // not worth a second kernel.
    long long chunk = (32ll * (rows < 128 ? rows : 128) + 255) / 256 * 256;
    if (chunk < 1024) chunk = 1024;
    while (chunk > 256 && units * ((room + chunk - 1) / chunk) < 2 * 148) chunk = (chunk / 2 + 255) / 256 * 256;
    if (room <= 512) chunk = 512;
    t.chunk = (int)chunk;
    t.chunks = (int)((room + chunk - 1) / chunk);
    t.items = (int)(units * t.chunks < (1ll << 31) - 1 ? units * t.chunks : 0);
    if (t.chunks > 1) {
        const size_t n = (size_t)p.B * p.Hq * p.T * t.chunks;
        t.part = (n * 4 + 255) & ~(size_t)255;
        t.bytes = t.part + n * p.D * 4;
    }
    return t;
}

template <typename T> cudaError_t launch_tree_tc(const CacheParams& p, const TreePlan& t, void* workspace, cudaStream_t s);

}  // namespace dsdpa
