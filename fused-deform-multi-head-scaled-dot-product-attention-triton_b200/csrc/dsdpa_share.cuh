// How a call's work over a paged cache is shared out.
//
// The queries that share a key/value head -- tokens times the group's heads, so many a tile: a unit -- meet the same keys.
// The key tiles of all units lie one behind the other, and every worker -- a block, or a warp -- takes an equal share
// of that line, whatever the lengths are (they are known on the device only): whole units, and at the ends
// of its share parts of units, whose results tree_combine_kernel joins.  So all workers end together, and no
// more than two parts a worker have to be written and read again.
#pragma once

#include "dsdpa_cache.cuh"

namespace dsdpa {

// Rows of a unit's tile, keys of a key tile, key tiles of the smallest share, workers of a block.
template <int ROWS, int KEYS, int LEAST = 2, int WORKERS = 1>
struct ShareTile {
    static constexpr int kRows = ROWS, kKeys = KEYS, kLeast = LEAST, kWorkers = WORKERS;
};

struct TreeSplit {
    int whole;            // units are not cut: no parts, no tree_combine_kernel
    int row_tiles;
    int part_rows;        // rows of a part
    long long* start;     // null, or [B + 1]: key tiles of a head's query tile in the sequences before, and [B + 1]: a worker's share
    float* part;          // [workers * 2][part_rows][D], normalised
    float* part_lse;      // [workers * 2][part_rows]
    long long rows;       // workers * 2 * part_rows
};
// Key tiles of a sequence: the same for all of its heads.
template <typename Tile>
__device__ __forceinline__ int tree_tiles(const CacheParams& p, int b) {
    const int real = drafted_tokens(p, b);
    return real > 0 ? (cached_keys(p, b) + real + Tile::kKeys - 1) / Tile::kKeys : 0;
}

// A unit, or the part of one that lies in a worker's share.
struct TreeItem {
    int b, hk, row0, rows, n, real, key0, tiles;
    int part;             // where its result goes: -1 to out and lse, else the number of the part
};
// Goes through the items of a worker; every role of a block has its own.
template <typename Tile>
struct TreeWalk {
    int b, unit, tile;    // unit: of the sequence's heads * row_tiles
    long long left;       // key tiles of the share; whole units: number of the next unit
    bool first;
    int worker;
    __device__ __forceinline__ bool next(const CacheParams& p, const TreeSplit& s, TreeItem& it) {
        const int units = p.Hkv * s.row_tiles;
        if (s.whole) {
            if (left >= (long long)p.B * units) return false;
            b = (int)(left / units);
            unit = (int)(left % units);
            tile = 0;
            it.tiles = tree_tiles<Tile>(p, b);
            it.part = -1;
            left += gridDim.x;
        } else {
            int nt = 0;
            while (left > 0) {
                nt = tree_tiles<Tile>(p, b);
                if (unit < units && nt > 0) break;
                ++b;
                unit = 0;
            }
            if (left <= 0) return false;
            it.tiles = (int)min((long long)(nt - tile), left);
            it.part = it.tiles == nt ? -1 : worker * 2 + (first ? 0 : 1);
            left -= it.tiles;
        }
        first = false;
        it.b = b;
        it.hk = unit / s.row_tiles;
        it.row0 = unit % s.row_tiles * Tile::kRows;
        it.rows = min(Tile::kRows, p.T * p.group - it.row0);
        it.n = cached_keys(p, b);
        it.real = drafted_tokens(p, b);
        it.key0 = tile * Tile::kKeys;
        ++unit;
        tile = 0;
        return true;
    }
};

// Where the shares of this block's workers begin, by all of its threads; the caller waits for them before it looks.
template <int THREADS, int WORKERS = 1>
struct TreeShare {
    long long sum[THREADS / 32], left[WORKERS];
    int b[WORKERS], unit[WORKERS], tile[WORKERS];
    template <typename Tile>
    __device__ __forceinline__ TreeWalk<Tile> walk(int w = 0) const {
        return TreeWalk<Tile>{ b[w], unit[w], tile[w], left[w], true, (int)blockIdx.x * WORKERS + w };
    }
};
template <typename Tile, int THREADS>
__device__ __forceinline__ void find_share(const CacheParams& p, const TreeSplit& sp, TreeShare<THREADS, Tile::kWorkers>& out) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (sp.whole) {
        if (tid < Tile::kWorkers) { out.left[tid] = blockIdx.x; out.b[tid] = out.unit[tid] = out.tile[tid] = 0; }
    } else {
        // where this block's share begins: a thread has the key tiles of a few sequences
        const int per = (p.B + THREADS - 1) / THREADS, b0 = min(p.B, tid * per), b1 = min(p.B, b0 + per);
        long long mine = 0;
        for (int b = b0; b < b1; ++b) mine += tree_tiles<Tile>(p, b);
        long long upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long t = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += t;
        }
        if (lane == 31) out.sum[warp] = upto;
        if (tid < Tile::kWorkers) { out.left[tid] = 0; out.b[tid] = out.unit[tid] = out.tile[tid] = 0; }
        __syncthreads();
        long long before = upto - mine, total = 0;
        for (int w = 0; w < THREADS / 32; ++w) {
            if (w < warp) before += out.sum[w];
            total += out.sum[w];
        }
        const int units = p.Hkv * sp.row_tiles;
        const long long line = total * units, workers = (long long)gridDim.x * Tile::kWorkers;
        const long long share = max((long long)Tile::kLeast, (line + workers - 1) / workers);
        if (blockIdx.x == 0 && sp.start) {
            long long at = before;
            for (int b = b0; b < b1; ++b) { sp.start[b] = at; at += tree_tiles<Tile>(p, b); }
            if (tid == 0) { sp.start[p.B] = total; sp.start[p.B + 1] = share; }
        }
        for (int k = 0; k < Tile::kWorkers; ++k) {
            const long long from = share * ((long long)blockIdx.x * Tile::kWorkers + k);
            if (from >= line || from < before * units || from >= (before + mine) * units) continue;
            long long at = before * units;
            int b = b0;
            for (;; ++b) {
                const long long span = (long long)tree_tiles<Tile>(p, b) * units;
                if (from < at + span) break;
                at += span;
            }
            const int nt = tree_tiles<Tile>(p, b);
            out.b[k] = b;
            out.unit[k] = (int)((from - at) / nt);
            out.tile[k] = (int)((from - at) % nt);
            out.left[k] = min(share, line - from);
        }
    }
}

// Joins the parts of a row: out = sum_c 2^(lse_c - lse) part_c; rows that see no key get their zeros.  A row has WARPS warps of a
// block of kCombineWarps: one where there are many rows, all where a few long caches leave many parts to each.
constexpr int kCombineWarps = 8;
template <typename T, typename Tile, int WARPS>
__global__ void __launch_bounds__(kCombineWarps * 32, 3) tree_combine_kernel(const __grid_constant__ CacheParams p, const __grid_constant__ TreeSplit sp) {
    __shared__ __align__(16) float s_acc[WARPS > 1 ? kCombineWarps : 1][WARPS > 1 ? 256 : 1], s_sum[kCombineWarps];
    const int warp = threadIdx.x / 32, mine = warp % WARPS;           // the same row for all threads, or no barrier below
    const long long row = (long long)blockIdx.x * (kCombineWarps / WARPS) + warp / WARPS;
    if (row >= (long long)p.B * p.Hq * p.T) return;
    const int lane = threadIdx.x & 31, t = (int)(row % p.T), h = (int)(row / p.T % p.Hq), b = (int)(row / p.T / p.Hq);
    // the workers whose shares the row's unit lies in
    const int gr = t * p.group + h % p.group, nt = tree_tiles<Tile>(p, b);
    asm volatile("griddepcontrol.wait;" ::: "memory");                // the first kernel's results from here on
    const long long share = sp.start[p.B + 1];
    const long long from = sp.start[b] * p.Hkv * sp.row_tiles + (long long)(h / p.group * sp.row_tiles + gr / Tile::kRows) * nt;
    const int c0 = (int)(from / share), c1 = nt > 0 ? (int)((from + nt - 1) / share) : c0 - 1;
    if (c0 == c1) return;                                // written by the worker itself
    const int used = c1 - c0 + 1;                        // 0: a query that sees no key
    auto place = [&](int c) {                            // a worker's first part, or its second
        const long long at = ((long long)(c0 + c) * 2 + ((c0 + c) * share >= from ? 0 : 1)) * sp.part_rows + gr % Tile::kRows;
        return in_range(at, sp.rows, p.err) ? at : 0ll;
    };
    float m = kNegInf, kept = kNegInf;                    // kept: of this warp's first 32 parts
    bool nan = false;
    for (int c = lane; c < used; c += 32) {
        const float x = sp.part_lse[place(c)];
        if (c - lane == mine * 32) kept = x;
        nan = nan || x != x;
        m = fmaxf(m, x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    nan = __any_sync(0xffffffffu, nan);
    const float m0 = m == kNegInf ? 0.0f : m;
    float sum = 0.0f, acc[2][4] = {};
    // A lane has a part's factor, so that the parts themselves are asked for several at a time; lanes without elements read
    // the first ones (a load behind a condition would be waited for at once).
    const float *part0 = sp.part + (lane * 4 < p.D ? lane * 4 : 0), *part1 = sp.part + (128 + lane * 4 < p.D ? 128 + lane * 4 : 0);
    auto add = [&](float (&to)[4], float f, const float* from) {
        const float4 v = *reinterpret_cast<const float4*>(from);
        to[0] = fmaf(f, v.x, to[0]);
        to[1] = fmaf(f, v.y, to[1]);
        to[2] = fmaf(f, v.z, to[2]);
        to[3] = fmaf(f, v.w, to[3]);
    };
    for (int first = mine * 32; first < used; first += WARPS * 32) {
        const float own = first + lane < used ? exp2f((first == mine * 32 ? kept : sp.part_lse[place(first + lane)]) - m0) : 0.0f;
        sum += own;
        const int n = min(32, used - first);
#pragma unroll 8
        for (int c = 0; c < n; ++c) add(acc[0], __shfl_sync(0xffffffffu, own, c), part0 + place(first + c) * p.D);
        if (p.D > 128) {
#pragma unroll 8
            for (int c = 0; c < n; ++c) add(acc[1], __shfl_sync(0xffffffffu, own, c), part1 + place(first + c) * p.D);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if constexpr (WARPS > 1) {
        static_assert(WARPS == kCombineWarps, "a block has one row");
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (k * 128 + lane * 4 < p.D) *reinterpret_cast<float4*>(&s_acc[warp][k * 128 + lane * 4]) = make_float4(acc[k][0], acc[k][1], acc[k][2], acc[k][3]);
        if (lane == 0) s_sum[warp] = sum;
        __syncthreads();
        if (warp > 0) return;
        for (int w = 1; w < WARPS; ++w) {
            sum += s_sum[w];
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (k * 128 + lane * 4 < p.D) acc[k][e] += s_acc[w][k * 128 + lane * 4 + e];
        }
    }
    const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
    bool fine = !nan;
    T* out = (T*)p.out + row * p.D + lane * 4;
#pragma unroll
    for (int k = 0; k < 2; ++k)
        if (k * 128 + lane * 4 < p.D) {
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = acc[k][e] * inv;
                fine = fine && fabsf(v[e]) <= 3.0e38f;
            }
            store4(out + k * 128, v);
        }
    if (lane == 0) p.lse[row] = sum != 0.0f ? m0 + log2f(sum) : kNegInf;
    __syncwarp();
    if (__any_sync(0xffffffffu, !fine)) exact_row_tree<T>(p, b, h, t);
}

}  // namespace dsdpa
