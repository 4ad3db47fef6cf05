// Host side of the kernels over a paged cache.
#pragma once

#include "dsdpa_host.h"
#include "dsdpa_cache.cuh"

namespace dsdpa {

// The tensor-core kernels take 16-bit storage with up to 128 elements a row; fp32 arithmetic the rest.
inline bool cache_on_tensor_cores(const dsdpa_cache_problem& p) { return p.dtype != DSDPA_F32 && p.D <= 128; }
// ... and of these a warp's own matrix instructions those with up to 16 rows to a key/value head.
inline bool cache_few_rows(const dsdpa_cache_problem& p) { return cache_on_tensor_cores(p) && p.T * (p.Hq / p.Hkv) <= 16; }

// fp32 with up to 8 rows has few-row kernels too, for caches that are worth a second kernel (plan_tree's `whole`).
constexpr int kFewRowsF32 = 8, kWholeF32 = 256;
inline bool cache_few_f32(const dsdpa_cache_problem& p) {
    return p.dtype == DSDPA_F32 && p.D <= 128 && p.T * (p.Hq / p.Hkv) <= kFewRowsF32 && (long long)p.table_width * p.page_size > kWholeF32;
}
constexpr int few_f32_blocks(int chunks, bool weights) { return weights ? 4 : chunks == 1 ? 3 : 2; }   // by registers

// Blocks of four warps that the few-row kernels are compiled to have on an SM: with 128 elements a row tree attention needs
// more than 128 registers a thread.
constexpr int few_blocks(int hd, int rows, bool weights) {
    if (rows > 8) return weights ? 3 : 2;
    return weights || hd == 64 ? 4 : 3;
}

// A call's work, as far as the host can know it (the lengths are on the device).
struct TreePlan {
    bool whole;              // units are not cut
    int row_unit, row_tiles, part_rows, blocks, weight_blocks;
    long long parts;         // places for them in the workspace
    size_t part, part_lse, bytes;      // workspace: the table of starts at 0
};
inline TreePlan plan_tree(const dsdpa_cache_problem& p) {
    TreePlan t{};
    const bool tc = cache_on_tensor_cores(p), few = cache_few_rows(p), few32 = cache_few_f32(p);
    const long long room = (long long)p.table_width * p.page_size;
    const int hd = p.D <= 64 ? 64 : 128, rows = p.T * (p.Hq / p.Hkv), keys = few || few32 ? 32 : tc ? 128 : 64, workers = few || few32 ? 4 : 1;   // a block's
    t.row_unit = few32 ? kFewRowsF32 : few ? 16 : tc ? 128 : rows <= 16 ? 16 : rows <= 32 || p.D > 128 ? 32 : 64;
    t.row_tiles = (rows + t.row_unit - 1) / t.row_unit;
    t.part_rows = rows < t.row_unit ? rows : t.row_unit;
    const long long units = (long long)p.B * p.Hkv * t.row_tiles, tiles = (room + keys - 1) / keys;
    // A short cache is not worth a second kernel: a block goes through it while the launch of one would take (few rows, one
    // cache of 500 keys: 14 us whole, of 740 19 us whole and 17 us cut; fp32 arithmetic half of that).  With 32 rows a key
    // tile costs less for each: one cache of 740 keys 16.2 us whole and 16.8 us cut, of 1000 19 and 17; and where the units
    // fill half of the SMs by themselves 8 caches of 2000 keys 30 and 35 us, 64 of them 113 and 125 us.
    t.whole = room <= (few ? 512 : !tc ? kWholeF32 : units >= 64 ? 2048 : 768);
    // as many blocks as stay on the SMs at once, but no share below two key tiles
    const long long stay = few32 ? few_f32_blocks(rows <= 4 ? 1 : 2, false) * kSMs : few ? few_blocks(hd, rows, false) * kSMs : tc ? kSMs : p.D <= 64 ? 3 * kSMs : p.D <= 128 ? 2 * kSMs : kSMs;
    const long long stay_weights = few32 ? few_f32_blocks(1, true) * kSMs : few ? few_blocks(hd, rows, true) * kSMs : stay, least = 2 * workers;
    const long long most = t.whole ? units : (units * tiles + least - 1) / least, most_weights = ((long long)p.B * p.Hkv * tiles + least - 1) / least;
    t.blocks = (int)(most < stay || t.whole ? (most < 65536 ? most : 65536) : stay);
    t.weight_blocks = (int)(most_weights < stay_weights ? most_weights : stay_weights);
    const size_t parts = (size_t)t.blocks * workers * 2;
    if (!t.whole) {
        auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
        t.parts = (long long)parts;
        t.part_lse = up(((size_t)p.B + 2) * 8);
        t.part = t.part_lse + up(parts * t.part_rows * 4);
        t.bytes = t.part + parts * t.part_rows * p.D * 4;
    }
    return t;
}

template <typename T> cudaError_t launch_tree_few(const CacheParams& p, const TreePlan& t, void* workspace, cudaStream_t s);
template <typename T> cudaError_t launch_weights_few(const CacheParams& p, const TreePlan& t, cudaStream_t s);
cudaError_t launch_tree_few_f32(const CacheParams& p, const TreePlan& t, void* workspace, cudaStream_t s);
cudaError_t launch_weights_few_f32(const CacheParams& p, const TreePlan& t, cudaStream_t s);
template <typename T> cudaError_t launch_tree_tc(const CacheParams& p, const TreePlan& t, void* workspace, cudaStream_t s);
template <typename T> cudaError_t launch_tree_simt(const CacheParams& p, const TreePlan& t, void* workspace, cudaStream_t s);
template <typename T> cudaError_t launch_weights_tc(const CacheParams& p, const TreePlan& t, cudaStream_t s);
template <typename T> cudaError_t launch_weights_simt(const CacheParams& p, const TreePlan& t, cudaStream_t s);

}  // namespace dsdpa
