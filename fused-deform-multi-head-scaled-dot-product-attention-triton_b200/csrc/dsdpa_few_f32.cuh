// Tree attention and accumulated weights for a few rows in fp32: head dimensions up to 128, at most 8 (token, head) rows
// to a key/value head -- decoding.
//
// The work is to read the cache.  As in dsdpa_few.cuh a warp goes through a share of the keys that is its alone, with
// everything in registers: HD / 4 lanes have a key's row, 16 bytes each, so that every load is whole lines; eight
// keys a step for each such group of lanes.  Each lane multiplies its elements with those of four rows: 32 partial
// sums, which the group adds up by exchanging halves (16 + 8 + .. exchanges for 32 sums, where adding up each by itself
// would take 32 log2(lanes)) and of which a lane then has 32 / lanes: the scores.  Their weights go through
// shared memory back to all lanes.  The register tiles of dsdpa_cache_simt.cuh spend 16 rows' fmas on whatever rows
// there are: for 64 caches of up to 8192 keys, 32 heads on 8, one token each (D = 128) they take 1150 us and
// 723 us (weights), these kernels 318 us (6.2 TB/s of the 6.5 that a copy reaches) and 174 us (5.7).  Bound by DRAM;
// with 8 rows (522 us) by the arithmetic between the loads, two blocks an SM.
#pragma once

#include "dsdpa_cache_launch.h"
#include "dsdpa_share.cuh"

namespace dsdpa {

constexpr int kF32Warps = 4, kF32Rows = kFewRowsF32, kF32Keys = 32;
using F32Tile = ShareTile<kF32Rows, kF32Keys, 2, kF32Warps>;

struct F32Row {
    unsigned long long above;
    float slope2, pos, lse;      // lse: the weights' kernel
    int real;
};

template <int HD, int NC>
struct F32Few {
    static constexpr int kLanes = HD / 4, kGroups = 32 / kLanes, kHeld = 32 / kLanes;   // of a key; of a warp; sums of a lane
    static constexpr int kStep = 8 * kGroups;                                           // keys
    static constexpr int kTurn = 4 / kHeld;          // lanes that lie between one key's sums and the next key's

    int lane, at, group;         // at: lane of the group
    float4 q[NC * 4];
    int page, slot;              // of key `lane` of the step
    unsigned there;

    __device__ __forceinline__ F32Few() : lane(threadIdx.x & 31), at(lane % kLanes), group(lane / kLanes) {}
    __device__ __forceinline__ static int key_of(int e, int group) { return e * kGroups + group; }

    __device__ __forceinline__ void queries(const CacheParams& p, const TreeItem& it, F32Row* rows) {
        __syncwarp();                                    // the last unit's are read
        if (lane < kF32Rows) {
            const int t = lane / p.group, h = it.hk * p.group + lane % p.group;
            const bool valid = lane < it.rows;
            F32Row r{};
            r.real = valid && t < it.real;
            r.above = r.real ? tokens_above(p, it.b, t) : 0ull;
            r.slope2 = p.slopes && valid ? __ldg(p.slopes + h) * kLog2e : 0.0f;
            r.pos = p.slopes && r.real ? (float)depth_of(r.above) : 0.0f;
            rows[lane] = r;
        }
#pragma unroll
        for (int r = 0; r < NC * 4; ++r) {
            q[r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (r < it.rows && at * 4 < p.D)
                q[r] = __ldg(reinterpret_cast<const float4*>(row_of<float>(p.q, p.sq, it.b, it.hk * p.group + r % p.group, r / p.group) + at * 4));
        }
        __syncwarp();
    }
    // table entry of the step's key `lane`
    __device__ __forceinline__ int ask(const CacheParams& p, const TreeItem& it, int k0) const {
        const int j = k0 + lane;
        return lane < kStep && j < it.n + it.real ? table_entry(p.table, p.width, it.b, page_index(p.div, j)) : 0;
    }
    __device__ __forceinline__ void find(const CacheParams& p, const TreeItem& it, int k0, int entry) {
        const int j = k0 + lane;
        page = lane < kStep && j < it.n + it.real ? checked_page(entry, p.pages, p.err) : -1;
        slot = j - page_index(p.div, j) * p.page_size;
        there = __ballot_sync(0xffffffffu, page >= 0);
    }
    __device__ __forceinline__ static float4 row_part(const float* from) {
        const uint4 u = ldg128_stream(from);
        return make_float4(__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z), __uint_as_float(u.w));
    }
    __device__ __forceinline__ void load(const CacheParams& p, const TreeItem& it, const void* base, const long long (&st)[3], float4 (&x)[8]) const {
        const float* from = row_of<float>(base, st, 0, it.hk, 0) + at * 4;
        // the usual step: all keys there, every lane with elements (no load behind a condition: it would be waited for at once)
        if (there == (kStep == 32 ? ~0u : (1u << kStep % 32) - 1) && p.D == HD) {
            if (p.page_size % kStep == 0) {              // on one page
                from += __shfl_sync(0xffffffffu, page, 0) * st[0] + (__shfl_sync(0xffffffffu, slot, 0) + group) * st[2];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = row_part(from + e * kGroups * st[2]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int key = key_of(e, group);
                    x[e] = row_part(from + __shfl_sync(0xffffffffu, page, key) * st[0] + __shfl_sync(0xffffffffu, slot, key) * st[2]);
                }
            }
            return;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int key = key_of(e, group), pg = __shfl_sync(0xffffffffu, page, key), sl = __shfl_sync(0xffffffffu, slot, key);
            x[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (pg >= 0 && at * 4 < p.D) x[e] = row_part(from + pg * st[0] + sl * st[2]);
        }
    }
    // Scores in base 2 of this lane's (key, row) pairs: numbers at * kHeld + v, key the number / 4, row 4 c + the number % 4.
    __device__ __forceinline__ void scores(const CacheParams& p, const TreeItem& it, int k0, const float4 (&k)[8], const F32Row* rows,
                                           unsigned now, float (&s)[NC][kHeld]) const {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float x[32];
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float4 a = q[c * 4 + r];
                    const float2 y = fma2(make_float2(k[e].z, k[e].w), make_float2(a.z, a.w), mul2(make_float2(k[e].x, k[e].y), make_float2(a.x, a.y)));
                    x[e * 4 + r] = y.x + y.y;
                }
#pragma unroll
            for (int stage = 0; stage < 5; ++stage) {
                const int o = kLanes / 2 >> stage, n = 16 >> stage;
                const bool upper = lane & o;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    if (o == 0 || i >= n) continue;
                    const float mine = upper ? x[i + n] : x[i], other = upper ? x[i] : x[i + n];
                    x[i] = mine + __shfl_xor_sync(0xffffffffu, other, o);
                }
            }
#pragma unroll
            for (int v = 0; v < kHeld; ++v) {
                const int number = at * kHeld + v, in_step = key_of(number >> 2, group), j = k0 + in_step, draft = j - it.n;
                const F32Row& row = rows[c * 4 + (number & 3)];
                const bool sees = row.real && (now >> in_step & 1u) && (draft < 0 || (row.above >> (draft & 63) & 1u));
                float y = soft_cap(p.sm_scale * x[v], p.cap) * kLog2e;
                if (p.slopes && sees) {
                    const float where = draft >= 0 ? (float)depth_of(tokens_above(p, it.b, draft))
                                                   : key_position(p, it.b, it.hk, j, first_position(p, it.b, it.n));
                    y = fmaf(-row.slope2, fabsf(row.pos - where), y);
                }
                s[c][v] = sees ? y : kNegInf;
            }
        }
    }
    // x of row r of chunk c, which the first lanes of the group have
    template <int N>
    __device__ __forceinline__ float of_row(const float (&x)[N], int r) const {
        return __shfl_sync(0xffffffffu, x[r % kHeld], group * kLanes + r / kHeld);
    }
    // over the lanes of the group that have the same rows
    template <typename F>
    __device__ __forceinline__ float over_keys(float x, F f) const {
#pragma unroll
        for (int o = kTurn; o < 8 * kTurn; o *= 2) x = f(x, __shfl_xor_sync(0xffffffffu, x, o));
        return x;
    }
};

template <int HD, int NC>
__global__ void __launch_bounds__(kF32Warps * 32, few_f32_blocks(NC, false))
tree_few_f32_kernel(const __grid_constant__ CacheParams p, const __grid_constant__ TreeSplit sp) {
    using F = F32Few<HD, NC>;
    __shared__ float4 s_w[kF32Warps][NC][F::kGroups * 8];       // weights of a step: [key of the group][4 rows]
    __shared__ F32Row s_rows[kF32Warps][kF32Rows];
    __shared__ TreeShare<kF32Warps * 32, kF32Warps> share;
    const int warp = threadIdx.x >> 5;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    find_share<F32Tile>(p, sp, share);
    __syncthreads();
    TreeWalk<F32Tile> walk = share.template walk<F32Tile>(warp);
    F32Row* rows = s_rows[warp];
    F few;
    TreeItem it;
    while (walk.next(p, sp, it)) {
        few.queries(p, it, rows);
        float m[NC][F::kHeld], l[NC][F::kHeld];
        float2 o[NC * 4][2] = {};
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int v = 0; v < F::kHeld; ++v) { m[c][v] = kNegInf; l[c][v] = 0.0f; }
        const int keys = min(it.tiles * kF32Keys, it.n + it.real - it.key0);
        float4 k[8], v[8];
        few.find(p, it, it.key0, few.ask(p, it, it.key0));
        few.load(p, it, p.k, p.sk, k);
        few.load(p, it, p.v, p.sv, v);
        int ahead = few.ask(p, it, it.key0 + F::kStep);
        for (int i = 0; i < keys; i += F::kStep) {
            const int k0 = it.key0 + i;
            const bool more = i + F::kStep < keys;
            float s[NC][F::kHeld];
            few.scores(p, it, k0, k, rows, few.there, s);
            if (more) {
                few.find(p, it, k0 + F::kStep, ahead);
                few.load(p, it, p.k, p.sk, k);
                ahead = few.ask(p, it, k0 + 2 * F::kStep);
            }
            // a row's reference point moves when its maximum is more than 8 above it, whatever the other rows' do
            float top[NC][F::kHeld];
            bool move[NC][F::kHeld], any = false;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int x = 0; x < F::kHeld; ++x) {
                    top[c][x] = few.over_keys(s[c][x], [](float a, float b) { return fmaxf(a, b); });
                    move[c][x] = top[c][x] > m[c][x] + 8.0f || (m[c][x] == kNegInf && top[c][x] > kNegInf);
                    any = any || move[c][x];
                }
            if (__any_sync(0xffffffffu, any)) {
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    float f[F::kHeld];
#pragma unroll
                    for (int x = 0; x < F::kHeld; ++x) {
                        f[x] = move[c][x] ? fast_exp2(m[c][x] - top[c][x]) : 1.0f;
                        if (move[c][x]) m[c][x] = top[c][x];
                        l[c][x] *= f[x];
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float g = few.of_row(f, r);
#pragma unroll
                        for (int y = 0; y < 2; ++y) o[c * 4 + r][y] = mul2(o[c * 4 + r][y], make_float2(g, g));
                    }
                }
            }
            __syncwarp();                                // the last step's weights are read
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int x = 0; x < F::kHeld; ++x) {
                    const float w = fast_exp2(s[c][x] - (m[c][x] == kNegInf ? 0.0f : m[c][x]));
                    l[c][x] += w;
                    reinterpret_cast<float*>(s_w[warp][c])[few.group * 32 + few.at * F::kHeld + x] = w;
                }
            __syncwarp();
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float4 w = s_w[warp][c][few.group * 8 + e];
                    const float of[4] = { w.x, w.y, w.z, w.w };
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float2 f = make_float2(of[r], of[r]);
                        o[c * 4 + r][0] = fma2(f, make_float2(v[e].x, v[e].y), o[c * 4 + r][0]);
                        o[c * 4 + r][1] = fma2(f, make_float2(v[e].z, v[e].w), o[c * 4 + r][1]);
                    }
                }
            if (more) few.load(p, it, p.v, p.sv, v);
        }
        // the groups' results joined, each row's on all lanes
        unsigned bad = 0;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float f[F::kHeld];
#pragma unroll
            for (int x = 0; x < F::kHeld; ++x) {
                l[c][x] = few.over_keys(l[c][x], [](float a, float b) { return a + b; });
                float top = m[c][x];
#pragma unroll
                for (int d = F::kLanes; d < 32; d *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                f[x] = top == kNegInf ? 1.0f : fast_exp2(m[c][x] - top);
                m[c][x] = top;
                l[c][x] *= f[x];
#pragma unroll
                for (int d = F::kLanes; d < 32; d *= 2) l[c][x] += __shfl_xor_sync(0xffffffffu, l[c][x], d);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int gr = c * 4 + r, t = gr / p.group, h = it.hk * p.group + gr % p.group;
                const float g = few.of_row(f, r), sum = few.of_row(l[c], r), ref = few.of_row(m[c], r);
                const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
                float x[4] = { o[gr][0].x * g, o[gr][0].y * g, o[gr][1].x * g, o[gr][1].y * g };
                float nan = 0.0f * sum;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
#pragma unroll
                    for (int d = F::kLanes; d < 32; d *= 2) x[e] += __shfl_xor_sync(0xffffffffu, x[e], d);
                    x[e] = sum != 0.0f ? x[e] * inv : 0.0f;
                    nan = fmaf(x[e], 0.0f, nan);
                }
                if (gr < it.rows) {                      // the same for the whole warp
                    const long long out_row = ((long long)it.b * p.Hq + h) * p.T + t, part = (long long)it.part * sp.part_rows + gr;
                    if (it.part >= 0 && !in_range(part, sp.rows, p.err)) continue;
                    if (few.group == 0 && few.at * 4 < p.D) store4<float>((it.part < 0 ? (float*)p.out + out_row * p.D : sp.part + part * p.D) + few.at * 4, x);
                    if (few.lane == 0) (it.part < 0 ? p.lse[out_row] : sp.part_lse[part]) = sum != 0.0f ? ref + log2f(sum) : kNegInf;
                    if (__any_sync(0xffffffffu, nan != nan) && it.part < 0) bad |= 1u << gr;
                }
            }
        }
        // rows that something non-finite reached: once more, from the keys they see alone
        __syncwarp();
        while (bad) {
            const int gr = __ffs(bad) - 1;
            bad &= bad - 1;
            exact_row_tree<float>(p, it.b, it.hk * p.group + gr % p.group, gr / p.group);
        }
    }
}

// weights[key] += the sum of a key's weights over the rows.
template <int HD, int NC>
__global__ void __launch_bounds__(kF32Warps * 32, few_f32_blocks(NC, true))
weights_few_f32_kernel(const __grid_constant__ CacheParams p, const __grid_constant__ TreeSplit sp) {
    using F = F32Few<HD, NC>;
    __shared__ F32Row s_rows[kF32Warps][kF32Rows];
    __shared__ TreeShare<kF32Warps * 32, kF32Warps> share;
    const int warp = threadIdx.x >> 5;
    find_share<F32Tile>(p, sp, share);
    __syncthreads();
    TreeWalk<F32Tile> walk = share.template walk<F32Tile>(warp);
    F32Row* rows = s_rows[warp];
    F few;
    TreeItem it;
    while (walk.next(p, sp, it)) {
        few.queries(p, it, rows);
        if (few.lane < kF32Rows) {
            const int t = few.lane / p.group, h = it.hk * p.group + few.lane % p.group;
            bool real = rows[few.lane].real && !(p.take && !p.take[(long long)it.b * p.T + t]);
            const float lse = real ? p.lse[((long long)it.b * p.Hq + h) * p.T + t] : kNegInf;
            if (lse == kNegInf) real = false;            // a query that sees nothing adds nothing
            rows[few.lane].real = real;
            rows[few.lane].lse = lse;
        }
        __syncwarp();
        float* out = p.weights + ((long long)it.b * p.Hkv + it.hk) * p.slots;
        const int keys = min(it.tiles * kF32Keys, it.n + it.real - it.key0);
        float4 k[8];
        few.find(p, it, it.key0, few.ask(p, it, it.key0));
        few.load(p, it, p.k, p.sk, k);
        int ahead = few.ask(p, it, it.key0 + F::kStep);
        for (int i = 0; i < keys; i += F::kStep) {
            const int k0 = it.key0 + i, in_step = F::key_of(few.at * F::kHeld >> 2, few.group);
            // the first of the lanes that have a key's rows writes it
            const bool writes = (few.at * F::kHeld & 3) == 0 && (few.there >> in_step & 1u) && in_range(k0 + in_step, p.slots, p.err);
            const float old = writes ? out[k0 + in_step] : 0.0f;
            float s[NC][F::kHeld];
            few.scores(p, it, k0, k, rows, few.there, s);
            if (i + F::kStep < keys) {
                few.find(p, it, k0 + F::kStep, ahead);
                few.load(p, it, p.k, p.sk, k);
                ahead = few.ask(p, it, k0 + 2 * F::kStep);
            }
            float sum = 0.0f;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int x = 0; x < F::kHeld; ++x) {
                    const F32Row& row = rows[c * 4 + ((few.at * F::kHeld + x) & 3)];
                    sum += row.real ? fast_exp2(s[c][x] - row.lse) : 0.0f;
                }
#pragma unroll
            for (int d = 1; d < F::kTurn; d *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            if (writes) out[k0 + in_step] = old + sum;
        }
    }
}

}  // namespace dsdpa
