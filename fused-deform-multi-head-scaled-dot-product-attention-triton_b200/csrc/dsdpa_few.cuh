// Tree attention and accumulated weights for a few rows: 16-bit storage, head dimensions up to 128, at most 16
// (token, head) rows to a key/value head -- decoding.
//
// With so few rows the work is to read the cache, and what costs is everything between the loads.  So nothing is
// staged and nobody waits for anybody: a warp loads 16 keys' rows and values straight into the registers that
// the warp-wide matrix instruction (m16n8k16) takes its operands from, keeps its own running maximum and sum,
// and goes through a share of the keys that is its alone (dsdpa_share.cuh).  That works because a contraction
// may run in any order: a thread takes eight neighbouring elements of a row, one load, as the operands of two
// instructions, with the queries arranged alike; and the value rows of two neighbouring keys, of which it
// pairs up elements, as operands of eight.  The fifth-generation instructions, whose operands lie in shared
// memory, need 128 rows and a pipeline of roles to do the same: for 64 caches of up to 8192 keys, 32 heads on 8, one
// token each (D = 128, bf16) they take 254 us, this kernel 168 us (5.9 TB/s of the 6.5 that a copy reaches; capped 173, biased 194), and
// weights_few_kernel 86 us (5.9 TB/s).  Bound by DRAM; a warp has 8 KB of loads in flight.
#pragma once

#include "dsdpa_cache_launch.h"
#include "dsdpa_masked_fwd.cuh"
#include "dsdpa_share.cuh"

namespace dsdpa {

constexpr int kFewWarps = 4, kFewRows = 16, kFewKeys = 32;
using FewTile = ShareTile<kFewRows, kFewKeys, 2, kFewWarps>;
// Blocks of four warps an SM, by the registers that they need: few_blocks() has the same for the host.
template <int HD, int NR> constexpr int kFewTreeBlocks = few_blocks(HD, NR * 8, false);
template <int HD, int NR> constexpr int kFewWeightBlocks = few_blocks(HD, NR * 8, true);

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    if constexpr (DtypeOf<T>::value == DSDPA_BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

// A thread has scores of rows lane / 4 and (NR = 2: units of more than eight rows) lane / 4 + 8.
struct FewRow {
    bool real, masked;          // masked: a row of the unit that is not real
    unsigned long long above;
    float slope2, pos, lse;     // lse: the weights' kernel
};

// The unit's queries, as the operands that the matrix instructions take, in shared memory (q: HD / 16 pieces of 32
// lanes): a thread's elements of piece 2 i are 32 i + 8 (lane % 4) .. + 3 of its two rows, of piece 2 i + 1 the next four.
template <typename T, int HD, int NR>
__device__ __forceinline__ void few_queries(const CacheParams& p, const TreeItem& it, int lane, uint4* q, FewRow (&row)[NR]) {
    const int g = lane >> 2, t4 = lane & 3;
    const T* src[2] = { nullptr, nullptr };
#pragma unroll
    for (int s = 0; s < NR; ++s) {
        const int gr = g + 8 * s, t = gr / p.group, h = it.hk * p.group + gr % p.group;
        const bool valid = gr < it.rows;
        row[s].real = valid && t < it.real;
        row[s].masked = valid && !row[s].real;
        row[s].above = row[s].real ? tokens_above(p, it.b, t) : 0ull;
        row[s].slope2 = p.slopes && valid ? __ldg(p.slopes + h) * kLog2e : 0.0f;
        row[s].pos = p.slopes && row[s].real ? (float)depth_of(row[s].above) : 0.0f;
        if (valid) src[s] = row_of<T>(p.q, p.sq, it.b, h, t);
    }
    __syncwarp();                                        // the last unit's are read
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
        const int d = i * 32 + t4 * 8;
        uint4 x[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) x[s] = src[s] && d < p.D ? ldg128_nc(src[s] + d) : make_uint4(0, 0, 0, 0);
        q[(2 * i) * 32 + lane] = make_uint4(x[0].x, x[1].x, x[0].y, x[1].y);
        q[(2 * i + 1) * 32 + lane] = make_uint4(x[0].z, x[1].z, x[0].w, x[1].w);
    }
    __syncwarp();
}

// Where 16 keys' rows lie: a thread's two of K and four of V.  Page numbers are asked for one step ahead.
template <typename T, int HD>
struct FewKeys {
    const T *k[2], *v[4];
    unsigned there;             // bit n: key n is there
    bool whole;                 // all of them, with every element
    __device__ __forceinline__ static int ask(const CacheParams& p, const TreeItem& it, int k0, int lane) {
        // pages of whole 16s: one number for all
        const int j = p.page_size % 16 == 0 ? k0 : k0 + (lane & 15);
        return j < it.n + it.real ? table_entry(p.table, p.width, it.b, page_index(p.div, j)) : 0;
    }
    template <bool VALUES>
    __device__ __forceinline__ void find(const CacheParams& p, const TreeItem& it, int k0, int lane, int entry) {
        const int g = lane >> 2, t4 = lane & 3, keys = it.n + it.real;
        if (p.page_size % 16 == 0) {
            const int page = checked_page(entry, p.pages, p.err), slot = k0 - page_index(p.div, k0) * p.page_size;
            there = page < 0 ? 0u : keys - k0 >= 16 ? 0xffffu : (1u << max(0, keys - k0)) - 1;
            const T* row = row_of<T>(p.k, p.sk, 0, it.hk, slot + g) + (long long)max(page, 0) * p.sk[0];
            k[0] = row + t4 * 8;
            k[1] = k[0] + 8 * p.sk[2];
            if (VALUES) {
                const T* row = row_of<T>(p.v, p.sv, 0, it.hk, slot + 2 * t4) + (long long)max(page, 0) * p.sv[0];
                v[0] = row + g * 8;
                v[1] = v[0] + p.sv[2];
                v[2] = v[0] + 8 * p.sv[2];
                v[3] = v[1] + 8 * p.sv[2];
            }
        } else {
            const int j = k0 + (lane & 15), page = j < keys ? checked_page(entry, p.pages, p.err) : -1;
            const int slot = j - page_index(p.div, j) * p.page_size;
            there = __ballot_sync(0xffffffffu, page >= 0) & 0xffffu;
            auto at = [&](const void* base, const long long (&st)[3], int key) {
                const int pg = __shfl_sync(0xffffffffu, page, key), sl = __shfl_sync(0xffffffffu, slot, key);
                return row_of<T>(base, st, 0, it.hk, sl) + (long long)max(pg, 0) * st[0];
            };
#pragma unroll
            for (int e = 0; e < 2; ++e) k[e] = at(p.k, p.sk, g + 8 * e) + t4 * 8;
            if (VALUES) {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = at(p.v, p.sv, 2 * t4 + (e & 1) + 8 * (e >> 1)) + g * 8;
            }
        }
        whole = there == 0xffffu && p.D == HD;
    }
    // x[j][i]: elements 32 i + 8 (lane % 4) .. + 7 of key 8 j + lane / 4
    __device__ __forceinline__ void load_k(const CacheParams& p, int lane, uint4 (&x)[2][HD / 32]) const {
        if (whole) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < HD / 32; ++i) x[j][i] = ldg128_stream(k[j] + i * 32);
        } else {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < HD / 32; ++i) {
                    x[j][i] = make_uint4(0, 0, 0, 0);
                    if ((there >> (8 * j + (lane >> 2)) & 1u) && i * 32 + (lane & 3) * 8 < p.D) x[j][i] = ldg128_stream(k[j] + i * 32);
                }
        }
    }
    // x[e][c]: elements 64 c + 8 (lane / 4) .. + 7 of keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9 (t = lane % 4)
    __device__ __forceinline__ void load_v(const CacheParams& p, int lane, uint4 (&x)[4][HD / 64]) const {
        if (whole) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int c = 0; c < HD / 64; ++c) x[e][c] = ldg128_stream(v[e] + c * 64);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int c = 0; c < HD / 64; ++c) {
                    x[e][c] = make_uint4(0, 0, 0, 0);
                    if ((there >> (2 * (lane & 3) + (e & 1) + 8 * (e >> 1)) & 1u) && c * 64 + (lane >> 2) * 8 < p.D)
                        x[e][c] = ldg128_stream(v[e] + c * 64);
                }
        }
    }
};
__device__ __forceinline__ uint32_t word_of(const uint4& x, int i) { return i == 0 ? x.x : i == 1 ? x.y : i == 2 ? x.z : x.w; }

// Scores of 16 keys in base 2, masked: s[tile][c], key 8 tile + 2 (lane % 4) + (c & 1), row lane / 4 + 8 (c >> 1).
template <typename T, int HD, int NR>
__device__ __forceinline__ void few_scores(const CacheParams& p, const TreeItem& it, int k0, int lane, const uint4* q,
                                           const uint4 (&k)[2][HD / 32], const FewRow (&row)[NR], unsigned there, float scale2,
                                           float (&s)[2][4]) {
    const int t4 = lane & 3;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[j][c] = 0.0f;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
        const uint4 a = q[(2 * i) * 32 + lane], b = q[(2 * i + 1) * 32 + lane];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            mma16816<T>(s[j], a, k[j][i].x, k[j][i].y);
            mma16816<T>(s[j], b, k[j][i].z, k[j][i].w);
        }
    }
    if (p.cap > 0.0f) {
        const float in = 2.0f * p.sm_scale / p.cap, out = p.cap * kLog2e;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int c = 0; c < 2 * NR; c += 2) {
                const float2 t = half_tanh_any(mul2(make_float2(s[j][c], s[j][c + 1]), make_float2(in, in)));
                s[j][c] = t.x * out;
                s[j][c + 1] = t.y * out;
            }
    } else {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int c = 0; c < 2 * NR; ++c) s[j][c] *= scale2;
    }
    if (p.slopes) {
        const int base = first_position(p, it.b, it.n);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int key = k0 + 8 * j + 2 * t4 + e;
                float at = 0.0f;
                if (key < it.n) at = key_position(p, it.b, it.hk, key, base);
                else if (key < it.n + it.real) at = (float)depth_of(tokens_above(p, it.b, key - it.n));
#pragma unroll
                for (int r = 0; r < NR; ++r) s[j][2 * r + e] = fmaf(-row[r].slope2, fabsf(row[r].pos - at), s[j][2 * r + e]);
            }
    }
    if (!__all_sync(0xffffffffu, there == 0xffffu && k0 + 16 <= it.n && !row[0].masked && !row[NR - 1].masked)) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int c = 0; c < 2 * NR; ++c) {
                const int key = 8 * j + 2 * t4 + (c & 1), draft = k0 + key - it.n;
                const FewRow& r = row[c >> 1];
                const bool sees = r.real && (there >> key & 1u) && (draft < 0 || (r.above >> (draft & 63) & 1u));
                s[j][c] = sees ? s[j][c] : kNegInf;
            }
    }
}

// o[c][j]: rows lane / 4 (first two) and lane / 4 + 8, elements 64 c + 16 t + j and + 8.  With up to 8 rows the other 8 of the
// instruction take what rounding the weights to the storage type has left off: twice its bits, for nothing.
template <typename T, int HD, int NR>
struct FewState {
    float m[NR], l[NR];
    float o[HD / 64][8][4];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int r = 0; r < NR; ++r) { m[r] = kNegInf; l[r] = 0.0f; }
#pragma unroll
        for (int c = 0; c < HD / 64; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[c][j][e] = 0.0f;
    }
    // 16 keys' weights, from their scores, and values
    __device__ __forceinline__ void add(float (&s)[2][4], const uint4 (&v)[4][HD / 64]) {
        bool move[NR], any = false;
        float top[NR];
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            top[r] = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]));
            top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
            top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
            move[r] = top[r] > m[r] + 8.0f || (m[r] == kNegInf && top[r] > kNegInf);
            any = any || move[r];
        }
        // a row's reference point moves when its maximum is more than 8 above it, whatever the other rows' do
        if (__any_sync(0xffffffffu, any)) {
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                const float f = move[r] ? fast_exp2(m[r] - top[r]) : 1.0f;
                if (move[r]) m[r] = top[r];
                l[r] *= f;
#pragma unroll
                for (int c = 0; c < HD / 64; ++c)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        o[c][j][2 * r] *= f;
                        o[c][j][2 * r + 1] *= f;
                        if (NR == 1) { o[c][j][2] *= f; o[c][j][3] *= f; }
                    }
            }
        }
        uint32_t a[2][2] = {};
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const float m0 = m[r] == kNegInf ? 0.0f : m[r];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float x = fast_exp2(s[j][2 * r] - m0), y = fast_exp2(s[j][2 * r + 1] - m0);
                l[r] += x + y;                            // this thread's part of the sum
                a[j][r] = pack2<T>(x, y);
                if (NR == 1) {
                    const float2 hi = to_float2<T>(a[j][0]);
                    a[j][1] = pack2<T>(x - hi.x, y - hi.y);
                }
            }
        }
        const uint4 w = make_uint4(a[0][0], a[0][1], a[1][0], a[1][1]);
#pragma unroll
        for (int c = 0; c < HD / 64; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t pick = j & 1 ? 0x7632u : 0x5410u;
                mma16816<T>(o[c][j], w, __byte_perm(word_of(v[0][c], j >> 1), word_of(v[1][c], j >> 1), pick),
                            __byte_perm(word_of(v[2][c], j >> 1), word_of(v[3][c], j >> 1), pick));
            }
    }
    __device__ __forceinline__ void join() {
        if (NR > 1) return;
#pragma unroll
        for (int c = 0; c < HD / 64; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) { o[c][j][0] += o[c][j][2]; o[c][j][1] += o[c][j][3]; }
    }
    // the keys of an item, 16 at a time: groups first, first + step, ...
    __device__ __forceinline__ void run(const CacheParams& p, const TreeItem& it, int lane, int first, int step, const uint4* q,
                                        const FewRow (&row)[NR], float scale2) {
        const int groups = min(it.tiles * (kFewKeys / 16), (it.n + it.real - it.key0 + 15) / 16);
        if (first >= groups) return;
        using Keys = FewKeys<T, HD>;
        const int entry = Keys::ask(p, it, it.key0 + first * 16, lane);
        int ahead = first + step < groups ? Keys::ask(p, it, it.key0 + (first + step) * 16, lane) : 0;
        Keys keys;
        uint4 k[2][HD / 32], v[4][HD / 64];
        keys.template find<true>(p, it, it.key0 + first * 16, lane, entry);
        keys.load_k(p, lane, k);
        keys.load_v(p, lane, v);
        for (int i = first; i < groups; i += step) {
            const int k0 = it.key0 + i * 16, next = i + step;
            float s[2][4];
            few_scores<T, HD, NR>(p, it, k0, lane, q, k, row, keys.there, scale2, s);
            if (next < groups) {
                keys.template find<true>(p, it, it.key0 + next * 16, lane, ahead);
                keys.load_k(p, lane, k);
                ahead = next + step < groups ? Keys::ask(p, it, it.key0 + (next + step) * 16, lane) : 0;
            }
            add(s, v);
            if (next < groups) keys.load_v(p, lane, v);
        }
    }
};
__device__ __forceinline__ float quad_sum(float x) {
    x += __shfl_xor_sync(0xffffffffu, x, 1);
    return x + __shfl_xor_sync(0xffffffffu, x, 2);
}

template <typename T, int HD, int NR>
__global__ void __launch_bounds__(kFewWarps * 32, kFewTreeBlocks<HD, NR>)
tree_few_kernel(const __grid_constant__ CacheParams p, const __grid_constant__ TreeSplit sp) {
    extern __shared__ float s_part[];         // whole units: [warp][row][HD + 2], with m and l behind the sums
    __shared__ uint4 s_q[kFewWarps][HD / 16 * 32];
    __shared__ TreeShare<kFewWarps * 32, kFewWarps> share;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    find_share<FewTile>(p, sp, share);
    __syncthreads();
    TreeWalk<FewTile> walk = share.walk<FewTile>(warp);
    const float scale2 = p.sm_scale * kLog2e;
    TreeItem it;
    FewState<T, HD, NR> st;
    uint4* q = s_q[warp];
    FewRow row[NR];
    while (walk.next(p, sp, it)) {
        few_queries<T, HD, NR>(p, it, lane, q, row);
        st.clear();
        st.run(p, it, lane, sp.whole ? warp : 0, sp.whole ? kFewWarps : 1, q, row, scale2);
        st.join();
        unsigned bad[NR] = {};
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const int gr = g + 8 * r, t = gr / p.group, h = it.hk * p.group + gr % p.group;
            const bool valid = gr < it.rows;
            const float l = quad_sum(st.l[r]);
            if (sp.whole) {
                if (valid) {
                    float* to = s_part + (warp * it.rows + gr) * (HD + 2);
#pragma unroll
                    for (int c = 0; c < HD / 64; ++c)
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            to[c * 64 + 16 * t4 + j] = st.o[c][j][2 * r];
                            to[c * 64 + 16 * t4 + 8 + j] = st.o[c][j][2 * r + 1];
                        }
                    if (t4 == 0) { to[HD] = st.m[r]; to[HD + 1] = l; }
                }
                continue;
            }
            const float m0 = st.m[r] == kNegInf ? 0.0f : st.m[r], inv = l != 0.0f ? 1.0f / l : 0.0f, lse = l != 0.0f ? m0 + log2f(l) : kNegInf;
            const long long out_row = ((long long)it.b * p.Hq + h) * p.T + t, part = (long long)it.part * sp.part_rows + gr;
            float nan = 0.0f * l;
#pragma unroll
            for (int c = 0; c < HD / 64; ++c)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int d = c * 64 + 16 * t4 + 8 * half;
                    float x[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        x[j] = l != 0.0f ? st.o[c][j][2 * r + half] * inv : 0.0f;
                        nan = fmaf(x[j], 0.0f, nan);
                    }
                    if (valid && d < p.D) {
                        if (it.part < 0) store8<T>((T*)p.out + out_row * p.D + d, x);
                        else if (in_range(part, sp.rows, p.err)) store8<float>(sp.part + part * p.D + d, x);
                    }
                }
            nan = quad_sum(nan);
            if (valid && t4 == 0) (it.part < 0 ? p.lse[out_row] : sp.part_lse[part]) = lse;
            bad[r] = __ballot_sync(0xffffffffu, it.part < 0 && valid && t4 == 0 && nan != nan);
        }
        if (!sp.whole) {
            __syncwarp();
            // rows that something non-finite reached: once more, from the keys they see alone
#pragma unroll
            for (int r = 0; r < NR; ++r)
                while (bad[r]) {
                    const int gr = (__ffs(bad[r]) - 1) / 4 + 8 * r;
                    bad[r] &= bad[r] - 1;
                    exact_row_tree<T>(p, it.b, it.hk * p.group + gr % p.group, gr / p.group);
                }
            continue;
        }
        // the block's warps had every fourth 16 keys each: a warp joins every fourth row
        __syncthreads();
        for (int gr = warp; gr < it.rows; gr += kFewWarps) {
            const int t = gr / p.group, h = it.hk * p.group + gr % p.group;
            float top = kNegInf, sum = 0.0f, x[HD / 32] = {};
#pragma unroll
            for (int w = 0; w < kFewWarps; ++w) top = fmaxf(top, s_part[(w * it.rows + gr) * (HD + 2) + HD]);
            const float m0 = top == kNegInf ? 0.0f : top;
#pragma unroll
            for (int w = 0; w < kFewWarps; ++w) {
                const float* from = s_part + (w * it.rows + gr) * (HD + 2);
                const float f = fast_exp2(from[HD] - m0);
                sum = fmaf(f, from[HD + 1], sum);
#pragma unroll
                for (int e = 0; e < HD / 32; ++e) x[e] = fmaf(f, from[e * 32 + lane], x[e]);
            }
            const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
            const long long out_row = ((long long)it.b * p.Hq + h) * p.T + t;
            float nan = 0.0f * sum;
#pragma unroll
            for (int e = 0; e < HD / 32; ++e) {
                const float y = sum != 0.0f ? x[e] * inv : 0.0f;
                nan = fmaf(y, 0.0f, nan);
                if (e * 32 + lane < p.D) ((T*)p.out)[out_row * p.D + e * 32 + lane] = from_float<T>(y);
            }
            if (lane == 0) p.lse[out_row] = sum != 0.0f ? m0 + log2f(sum) : kNegInf;
            __syncwarp();
            if (__any_sync(0xffffffffu, nan != nan)) exact_row_tree<T>(p, it.b, h, t);
        }
        __syncthreads();                                 // before the next unit's parts take the places
    }
}

// weights[key] += the sum of a key's weights over the rows.
template <typename T, int HD, int NR>
__global__ void __launch_bounds__(kFewWarps * 32, kFewWeightBlocks<HD, NR>)
weights_few_kernel(const __grid_constant__ CacheParams p, const __grid_constant__ TreeSplit sp) {
    __shared__ uint4 s_q[kFewWarps][HD / 16 * 32];
    __shared__ TreeShare<kFewWarps * 32, kFewWarps> share;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
    find_share<FewTile>(p, sp, share);
    __syncthreads();
    TreeWalk<FewTile> walk = share.walk<FewTile>(warp);
    const float scale2 = p.sm_scale * kLog2e;
    TreeItem it;
    uint4 *q = s_q[warp], k[2][HD / 32];
    FewRow row[NR];
    while (walk.next(p, sp, it)) {
        few_queries<T, HD, NR>(p, it, lane, q, row);
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const int gr = g + 8 * r, t = gr / p.group, h = it.hk * p.group + gr % p.group;
            row[r].real = row[r].real && !(p.take && !p.take[(long long)it.b * p.T + t]);
            row[r].lse = row[r].real ? p.lse[((long long)it.b * p.Hq + h) * p.T + t] : kNegInf;
            row[r].real = row[r].lse != kNegInf;         // a query that sees nothing adds nothing
            row[r].masked = false;
        }
        float* out = p.weights + ((long long)it.b * p.Hkv + it.hk) * p.slots;
        const int groups = min(it.tiles * (kFewKeys / 16), (it.n + it.real - it.key0 + 15) / 16);
        using Keys = FewKeys<T, HD>;
        const int entry = Keys::ask(p, it, it.key0, lane);
        int ahead = Keys::ask(p, it, it.key0 + 16, lane);
        Keys keys;
        keys.template find<false>(p, it, it.key0, lane, entry);
        keys.load_k(p, lane, k);
        for (int i = 0; i < groups; ++i) {
            const int k0 = it.key0 + i * 16;
            // lanes 0 .. 3 write keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9
            float old[4];
            const unsigned now = keys.there;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int key = 2 * t4 + (e & 1) + 8 * (e >> 1);
                old[e] = g == 0 && (now >> key & 1u) && in_range(k0 + key, p.slots, p.err) ? out[k0 + key] : 0.0f;
            }
            float s[2][4];
            few_scores<T, HD, NR>(p, it, k0, lane, q, k, row, now, scale2, s);
            if (i + 1 < groups) {
                keys.template find<false>(p, it, k0 + 16, lane, ahead);
                keys.load_k(p, lane, k);
                ahead = Keys::ask(p, it, k0 + 32, lane);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float x = 0.0f;
#pragma unroll
                for (int r = 0; r < NR; ++r) x += row[r].real ? fast_exp2(s[e >> 1][2 * r + (e & 1)] - row[r].lse) : 0.0f;
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                const int key = 2 * t4 + (e & 1) + 8 * (e >> 1);
                if (g == 0 && (now >> key & 1u) && in_range(k0 + key, p.slots, p.err)) out[k0 + key] = old[e] + x;
            }
        }
    }
}

}  // namespace dsdpa
