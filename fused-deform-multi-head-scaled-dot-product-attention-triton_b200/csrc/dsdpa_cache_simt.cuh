// Tree attention and accumulated weights in fp32 arithmetic: fp32 storage, and 16-bit storage with more than 128
// elements a row.  Units of 16, 32 or 64 rows, keys 64 at a time, on the register tiles of
// dsdpa_masked_simt.cuh; work is shared out as in dsdpa_share.cuh.  Bound by the fma pipe and, for
// short caches, by latency: 17 tokens over three caches of 2000 keys (8 heads, D = 64, fp32) take 15 us.  (Up to
// eight rows of fp32 over longer caches have kernels of their own, dsdpa_few_f32.cuh.)
#pragma once

#include "dsdpa_masked_simt.cuh"
#include "dsdpa_share.cuh"

namespace dsdpa {

template <int HD, int RM> struct CacheSimt : SimtShape<HD, RM> {
    using L = SimtShape<HD, RM>;
    using Tile = ShareTile<L::BM, kSimtKeys>;
    static constexpr int kSmemTree = (L::BM * L::S + 2 * kSimtKeys * L::S + L::BM * L::W) * 4;
    static constexpr int kSmemWeights = (L::BM * L::S + kSimtKeys * L::S + 16 * kSimtKeys) * 4;
};

// N rows into shared memory as fp32; row r comes from from(r), zeros where that is null.
template <typename T, int HD, int N, typename F>
__device__ __forceinline__ void simt_gather(float* dst, int D, const void* any, F from) {
    constexpr int S = SimtShape<HD>::S, kPer = HD / 4;
    for (int e = threadIdx.x; e < N * kPer; e += kSimtThreads) {
        const int r = e / kPer, d = e % kPer * 4;
        const T* row = from(r);
        const bool there = row != nullptr && d < D;
        if constexpr (sizeof(T) == 4) {
            cp_async16(smem_addr(dst + r * S + d), there ? (const void*)(row + d) : any, there ? 16u : 0u);
        } else {
            float2 a = make_float2(0.0f, 0.0f), b = a;
            if (there) {
                const uint2 u = __ldg(reinterpret_cast<const uint2*>(row + d));
                a = to_float2<T>(u.x);
                b = to_float2<T>(u.y);
            }
            *reinterpret_cast<float4*>(dst + r * S + d) = make_float4(a.x, a.y, b.x, b.y);
        }
    }
    cp_async_commit();
}

// What the drafted tokens of a sequence see (tokens_above), for the whole block: the parents come from memory once, and the walks
// up the tree, every step of which waits for the one before, go through shared memory.  All threads; the caller
// waits before anybody reads, and before the next call.
struct SimtTokens { int parent[kTreeMax]; unsigned long long above[kTreeMax]; };
__device__ __forceinline__ void simt_tokens(const CacheParams& p, const TreeItem& it, SimtTokens& s) {
    const int t = threadIdx.x;
    if (t < it.real) s.parent[t] = p.parents ? __ldg(p.parents + (long long)it.b * p.T + t) : t - 1;
    __syncthreads();
    if (t < it.real) s.above[t] = walk_up(t, p.err, [&](int at) { return s.parent[at]; });
}

// What a tile's keys are, by threads 0 .. 63: their pages (-1: absent) and positions.
__device__ __forceinline__ void simt_keys(const CacheParams& p, const TreeItem& it, const SimtTokens& tokens, int k0, int* s_page, float* s_at) {
    const int t = threadIdx.x;
    if (t >= kSimtKeys) return;
    const int j = k0 + t;
    int page = -1;
    float at = 0.0f;
    if (j < it.n + it.real) {
        page = page_of(p.table, p.width, p.pages, p.err, it.b, page_index(p.div, j));
        if (p.slopes) at = j >= it.n ? (float)depth_of(tokens.above[j - it.n]) : key_position(p, it.b, it.hk, j, first_position(p, it.b, it.n));
    }
    s_page[t] = page;
    s_at[t] = at;
}

template <typename T, int HD, int RM>
__global__ void __launch_bounds__(kSimtThreads)
tree_simt_kernel(const __grid_constant__ CacheParams p, const __grid_constant__ TreeSplit sp) {
    using C = CacheSimt<HD, RM>;
    using L = typename C::L;
    using Tile = typename C::Tile;
    extern __shared__ float4 simt_smem[];
    float *sq = reinterpret_cast<float*>(simt_smem), *sk = sq + L::BM * L::S, *sv = sk + kSimtKeys * L::S, *sw = sv + kSimtKeys * L::S;
    __shared__ int s_page[2][kSimtKeys];
    __shared__ float s_at[2][kSimtKeys];
    __shared__ TreeShare<kSimtThreads> share;
    __shared__ SimtTokens tokens;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    find_share<Tile>(p, sp, share);
    __syncthreads();
    TreeWalk<Tile> walk = share.template walk<Tile>();
    TreeItem it;
    while (walk.next(p, sp, it)) {
        __syncthreads();                                        // the last item's tiles are read
        simt_tokens(p, it, tokens);
        simt_gather<T, HD, L::BM>(sq, p.D, p.q, [&](int r) -> const T* {
            const int gr = it.row0 + r;
            return r < it.rows ? row_of<T>(p.q, p.sq, it.b, it.hk * p.group + gr % p.group, gr / p.group) : nullptr;
        });
        __syncthreads();
        float m[RM], l[RM], slope2[RM], pos[RM];
        unsigned long long above[RM];
        bool real[RM];
        float2 acc[RM][L::NJ][2] = {};
#pragma unroll
        for (int r = 0; r < RM; ++r) {
            const int in_tile = ty * RM + r, gr = it.row0 + in_tile, t = gr / p.group, h = it.hk * p.group + gr % p.group;
            real[r] = in_tile < it.rows && t < it.real;
            above[r] = real[r] ? tokens.above[t] : 0ull;
            slope2[r] = p.slopes && real[r] ? __ldg(p.slopes + h) * kLog2e : 0.0f;
            pos[r] = p.slopes && real[r] ? (float)depth_of(above[r]) : 0.0f;
            m[r] = kNegInf;
            l[r] = 0.0f;
        }
        auto rows_of = [&](const void* base, const long long (&st)[3], int k0, const int* pages) {
            return [=, &st](int r) -> const T* {
                const int page = pages[r], j = k0 + r;
                return page < 0 ? nullptr : row_of<T>(base, st, 0, it.hk, j - page_index(p.div, j) * p.page_size) + page * st[0];
            };
        };
        if (it.tiles > 0) {
            simt_keys(p, it, tokens, it.key0, s_page[0], s_at[0]);
            __syncthreads();
            simt_gather<T, HD, kSimtKeys>(sk, p.D, p.k, rows_of(p.k, p.sk, it.key0, s_page[0]));
        }
        for (int i = 0; i < it.tiles; ++i) {
            const int k0 = it.key0 + i * kSimtKeys, cur = i & 1;
            if (i + 1 < it.tiles) simt_keys(p, it, tokens, k0 + kSimtKeys, s_page[cur ^ 1], s_at[cur ^ 1]);
            cp_async_wait<0>();
            __syncthreads();                                    // q, k are there; the last tile's v and weights are read
            simt_gather<T, HD, kSimtKeys>(sv, p.D, p.v, rows_of(p.v, p.sv, k0, s_page[cur]));
            float s[RM][4];
            simt_dot<HD, RM>(sq, sk, s);
            const float unit = simt_cap(s, p.sm_scale, p.cap);
#pragma unroll
            for (int r = 0; r < RM; ++r) {
                float top = kNegInf;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int key = k0 + tx + 16 * c, draft = key - it.n;
                    float x = s[r][c] * unit;
                    if (p.slopes) x = fmaf(-slope2[r], fabsf(pos[r] - s_at[cur][tx + 16 * c]), x);
                    const bool sees = real[r] && s_page[cur][tx + 16 * c] >= 0 && (draft < 0 || (above[r] >> (draft & 63) & 1u));
                    s[r][c] = sees ? x : kNegInf;
                    top = fmaxf(top, s[r][c]);
                }
                top = fmaxf(m[r], half_warp_max(top));
                const float t0 = top == kNegInf ? 0.0f : top, f = fast_exp2(m[r] - t0);
                float sum = 0.0f;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const float w = fast_exp2(s[r][c] - t0);
                    sw[(ty * RM + r) * L::W + tx + 16 * c] = w;
                    sum += w;
                }
                l[r] = fmaf(l[r], f, sum);
                m[r] = top;
#pragma unroll
                for (int x = 0; x < L::NJ; ++x)
#pragma unroll
                    for (int z = 0; z < L::CW / 2; ++z) { acc[r][x][z].x *= f; acc[r][x][z].y *= f; }
            }
            cp_async_wait<0>();
            __syncthreads();                                    // weights and v are there, k is read
            if (i + 1 < it.tiles) simt_gather<T, HD, kSimtKeys>(sk, p.D, p.k, rows_of(p.k, p.sk, k0 + kSimtKeys, s_page[cur ^ 1]));
            simt_rows<HD, RM>(sw, sv, acc);
        }
        unsigned bad = 0;
#pragma unroll
        for (int r = 0; r < RM; ++r) {
            const int in_tile = ty * RM + r, gr = it.row0 + in_tile, t = gr / p.group, h = it.hk * p.group + gr % p.group;
            const long long row = ((long long)it.b * p.Hq + h) * p.T + t, part = (long long)it.part * sp.part_rows + in_tile;
            const bool valid = in_tile < it.rows && (it.part < 0 || in_range(part, sp.rows, p.err));
            const float sum = half_warp_sum(l[r]), inv = sum != 0.0f ? 1.0f / sum : 0.0f, lse = sum != 0.0f ? m[r] + log2f(sum) : kNegInf;
            float nan;
            if (it.part < 0) nan = simt_store<T, HD>(valid ? (T*)p.out + row * p.D : nullptr, acc[r], inv, p.D);
            else nan = simt_store<float, HD>(valid ? sp.part + part * p.D : nullptr, acc[r], inv, p.D);
            nan = half_warp_sum(nan + sum * 0.0f);
            if (valid) {
                if (tx == 0) (it.part < 0 ? p.lse[row] : sp.part_lse[part]) = lse;
                if (nan != nan && it.part < 0) bad |= 1u << r;
            }
        }
        simt_redo<RM>(bad, [&](int r) {
            const int gr = it.row0 + r;
            exact_row_tree<T>(p, it.b, it.hk * p.group + gr % p.group, gr / p.group);
        });
    }
}

template <typename T, int HD, int RM>
__global__ void __launch_bounds__(kSimtThreads)
weights_simt_kernel(const __grid_constant__ CacheParams p, const __grid_constant__ TreeSplit sp) {
    using C = CacheSimt<HD, RM>;
    using L = typename C::L;
    using Tile = typename C::Tile;
    extern __shared__ float4 simt_smem[];
    float *sq = reinterpret_cast<float*>(simt_smem), *sk = sq + L::BM * L::S, *part = sk + kSimtKeys * L::S;
    __shared__ int s_page[kSimtKeys];
    __shared__ float s_at[kSimtKeys];
    __shared__ TreeShare<kSimtThreads> share;
    __shared__ SimtTokens tokens;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int rows = p.T * p.group, passes = (rows + L::BM - 1) / L::BM;
    find_share<Tile>(p, sp, share);
    __syncthreads();
    TreeWalk<Tile> walk = share.template walk<Tile>();
    TreeItem it;
    while (walk.next(p, sp, it)) {
        float* out = p.weights + ((long long)it.b * p.Hkv + it.hk) * p.slots;
        float slope2[RM], pos[RM], lse[RM];
        unsigned long long above[RM];
        // the rows of a pass; a row that does not count has an infinite lse
        auto take_rows = [&](int pass) {
            simt_gather<T, HD, L::BM>(sq, p.D, p.q, [&](int r) -> const T* {
                const int gr = pass * L::BM + r;
                return gr < rows ? row_of<T>(p.q, p.sq, it.b, it.hk * p.group + gr % p.group, gr / p.group) : nullptr;
            });
#pragma unroll
            for (int r = 0; r < RM; ++r) {
                const int gr = pass * L::BM + ty * RM + r, t = gr / p.group, h = it.hk * p.group + gr % p.group;
                lse[r] = -kNegInf;
                above[r] = 0;
                slope2[r] = pos[r] = 0.0f;
                if (gr < rows && t < it.real && !(p.take && !p.take[(long long)it.b * p.T + t])) {
                    const float x = p.lse[((long long)it.b * p.Hq + h) * p.T + t];
                    lse[r] = x == kNegInf ? -kNegInf : x;
                    above[r] = tokens.above[t];
                    if (p.slopes) {
                        slope2[r] = __ldg(p.slopes + h) * kLog2e;
                        pos[r] = (float)depth_of(above[r]);
                    }
                }
            }
        };
        __syncthreads();
        simt_tokens(p, it, tokens);
        __syncthreads();
        if (passes == 1) take_rows(0);
        for (int i = 0; i < it.tiles; ++i) {
            const int k0 = it.key0 + i * kSimtKeys;
            simt_keys(p, it, tokens, k0, s_page, s_at);
            __syncthreads();
            simt_gather<T, HD, kSimtKeys>(sk, p.D, p.k, [&](int r) -> const T* {
                const int j = k0 + r;
                return s_page[r] < 0 ? nullptr : row_of<T>(p.k, p.sk, 0, it.hk, j - page_index(p.div, j) * p.page_size) + s_page[r] * p.sk[0];
            });
            float sum[4] = { 0.0f, 0.0f, 0.0f, 0.0f };
            for (int pass = 0; pass < passes; ++pass) {
                if (passes > 1) {
                    __syncthreads();                            // the last pass's rows are read
                    take_rows(pass);
                }
                cp_async_wait<0>();
                __syncthreads();
                float s[RM][4];
                simt_dot<HD, RM>(sq, sk, s);
                const float unit = simt_cap(s, p.sm_scale, p.cap);
#pragma unroll
                for (int r = 0; r < RM; ++r)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int draft = k0 + tx + 16 * c - it.n;
                        float x = s[r][c] * unit;
                        if (p.slopes) x = fmaf(-slope2[r], fabsf(pos[r] - s_at[tx + 16 * c]), x);
                        const bool sees = lse[r] != -kNegInf && (draft < 0 || (above[r] >> (draft & 63) & 1u));
                        sum[c] += sees ? fast_exp2(x - lse[r]) : 0.0f;
                    }
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) part[ty * kSimtKeys + tx + 16 * c] = sum[c];
            __syncthreads();
            if (tid < kSimtKeys && s_page[tid] >= 0 && in_range(k0 + tid, p.slots, p.err)) {
                float total = 0.0f;
#pragma unroll
                for (int y = 0; y < 16; ++y) total += part[y * kSimtKeys + tid];
                out[k0 + tid] += total;
            }
            __syncthreads();
        }
    }
}

}  // namespace dsdpa
