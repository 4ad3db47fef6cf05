// Paged key/value cache: where a key's row lies, what a drafted token sees, and one drafted token's
// result computed by one warp that visits the keys it sees only (the definition written out; the
// tiled kernel hands it the rows that came out non-finite).
#pragma once

#include "dsdpa_masked.cuh"

namespace dsdpa {

constexpr int kTreeMax = DSDPA_TREE_MAX;

// n / page_size = n mul >> shift for 0 <= n < 2^30.  With l = ceil(log2 d), k = 30 + l and m = floor(2^k / d) + 1: m d =
// 2^k + e with 0 < e <= d <= 2^l, so n m / 2^k is n / d plus less than 2^30 / 2^k = 2^-l <= 1 / d, which cannot reach the
// next whole number.
struct PageDivision {
    unsigned long long mul;
    int shift;
};
inline PageDivision page_division(int page_size) {
    int l = 0;
    while ((1ll << l) < page_size) ++l;
    return { (1ull << (30 + l)) / (unsigned)page_size + 1, 30 + l };
}
__device__ __forceinline__ int page_index(const PageDivision& d, int n) { return (int)(((unsigned)n * d.mul) >> d.shift); }

struct CacheParams {
    const void *q, *k, *v;
    const int *table, *lens, *parents, *drafted, *positions, *start;
    const float* slopes;
    void* out;
    float* lse;                // tree: written; weights: read
    int B, Hq, Hkv, group, T, D;
    int pages, page_size, width, slots;
    float sm_scale, cap;
    long long sq[3], sk[3], sv[3];
    int* err;
    PageDivision div;
    // weights
    const unsigned char* take;
    float* weights;
};

// Keys that sequence b has cached, and its real drafted tokens.  Numbers that a table cannot hold are
// cut to what it holds, and reported.
__device__ __forceinline__ int cached_keys(const CacheParams& p, int b) {
    const int n = __ldg(p.lens + b), room = p.width * p.page_size;
    if (n > room) atomicCAS(p.err, 0, kErrBounds);
    return max(0, min(n, room));
}
__device__ __forceinline__ int drafted_tokens(const CacheParams& p, int b) {
    return p.drafted ? max(0, min(__ldg(p.drafted + b), p.T)) : p.T;
}
// Entry `index` of sequence b's row of the table, as it stands there; -1 behind the row's end.
__device__ __forceinline__ int table_entry(const int* table, int width, int b, int index) {
    return index < width ? __ldg(table + (long long)b * width + index) : -1;
}
// The page, or -1 (and a report) where it is none.  (Apart from table_entry, so that a kernel can ask for an entry long
// before it has to look at it.)
__device__ __forceinline__ int checked_page(int page, int pages, int* err) {
    if ((unsigned)page < (unsigned)pages) return page;
    atomicCAS(err, 0, kErrBounds);
    return -1;
}
__device__ __forceinline__ int page_of(const int* table, int width, int pages, int* err, int b, int index) {
    return checked_page(table_entry(table, width, b, index), pages, err);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, unsigned bytes) {   // the rest of 16 is zero
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory"); }

// The tokens that token t sees (bit u: token u), itself among them, from its chain of parents; its
// depth is their number less one.  Every step goes to an earlier token, so the walk ends.
template <typename F>
__device__ __forceinline__ unsigned long long walk_up(int t, int* err, F parent) {
    unsigned long long seen = 1ull << t;
    int at = t;
    while (true) {
        const int up = parent(at);
        if (up < -1 || up >= at) atomicCAS(err, 0, kErrBounds);
        if (up < 0 || up >= at) return seen;
        seen |= 1ull << up;
        at = up;
    }
}
__device__ __forceinline__ unsigned long long tokens_above(const CacheParams& p, int b, int t) {
    if (!p.parents) return t == 63 ? ~0ull : (1ull << (t + 1)) - 1;
    return walk_up(t, p.err, [&](int at) { return __ldg(p.parents + (long long)b * p.T + at); });
}
__device__ __forceinline__ int depth_of(unsigned long long above) { return __popcll(above) - 1; }
__device__ __forceinline__ int first_position(const CacheParams& p, int b, int n) { return p.start ? __ldg(p.start + b) : n; }
// Positions are taken from that of a drafted token without parent on: a drafted token's is then its depth, and a cached key's
// far behind it, whatever the numbers themselves are, off by no more than the distance's own rounding to fp32.
__device__ __forceinline__ float from_first(int at, int first) {       // the halves' differences are exact, and so is their sum up to one rounding
    return fmaf((float)((at >> 16) - (first >> 16)), 65536.0f, (float)((at & 0xffff) - (first & 0xffff)));
}
// Position of cached key j of head hk.
__device__ __forceinline__ float key_position(const CacheParams& p, int b, int hk, int j, int first) {
    return from_first(p.positions && in_range(j, p.slots, p.err) ? __ldg(p.positions + ((long long)b * p.Hkv + hk) * p.slots + j) : j, first);
}

// out and lse of one drafted token, by one warp (as in dsdpa_masked.cuh).
template <typename T>
__device__ __noinline__ void exact_row_tree(const CacheParams& p, int b, int h, int t) {
    constexpr int kSteps = 2;
    const int lane = threadIdx.x & 31, hk = h / p.group, D = p.D;
    const RowLanes rl(D, lane);
    const int n = cached_keys(p, b), real = drafted_tokens(p, b);
    const float slope = p.slopes ? __ldg(p.slopes + h) : 0.0f, sm_scale = p.sm_scale, cap = p.cap;
    float acc[8] = {};
    RowSoftmax sum;
    if (t < real) {
        const unsigned long long above = tokens_above(p, b, t);
        const int base = first_position(p, b, n), depth = depth_of(above);
        const T *k = row_of<T>(p.k, p.sk, 0, hk, 0), *v = row_of<T>(p.v, p.sv, 0, hk, 0);
        float q[8];
        load_piece<T>(row_of<T>(p.q, p.sq, b, h, t), rl.at, D, q);
        // (a sum of weights that is NaN stays one, and out and lse with it)
        for (int j0 = 0; j0 < n + real && !__any_sync(0xffffffffu, sum.l != sum.l); j0 += kSteps * rl.places) {
            RowPiece<T> kr[kSteps], vr[kSteps];
            float s[kSteps], w[kSteps], f[8];
            bool on[kSteps];
#pragma unroll
            for (int e = 0; e < kSteps; ++e) {
                const int j = j0 + e * rl.places + rl.place, index = page_index(p.div, j);
                int page = -1;
                if (j < n + real && (j < n || (above >> (j - n) & 1))) page = page_of(p.table, p.width, p.pages, p.err, b, index);
                on[e] = page >= 0;
                const int slot = on[e] ? j - index * p.page_size : 0;
                kr[e].load(k + max(page, 0) * p.sk[0] + slot * p.sk[2], rl.at, D);
                vr[e].load(v + max(page, 0) * p.sv[0] + slot * p.sv[2], rl.at, D);
            }
#pragma unroll
            for (int e = 0; e < kSteps; ++e) {
                kr[e].get(rl.at, D, f);
                s[e] = rl.row_sum(dot8(q, f));
            }
#pragma unroll
            for (int e = 0; e < kSteps; ++e) {
                const int j = j0 + e * rl.places + rl.place;
                s[e] = soft_cap(sm_scale * s[e], cap);
                if (p.slopes && on[e]) {
                    const float at = j >= n ? (float)depth_of(tokens_above(p, b, j - n)) : key_position(p, b, hk, j, base);
                    s[e] -= slope * fabsf((float)depth - at);
                }
                s[e] = on[e] ? s[e] * kLog2e : kNegInf;
            }
            const float c = sum.next(s, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] *= c;
#pragma unroll
            for (int e = 0; e < kSteps; ++e) {
                vr[e].get(rl.at, D, f);
                if (s[e] != kNegInf) add_piece(acc, w[e], f);
            }
        }
    }
    sum.join(rl, acc);
    const float inv = sum.l != 0.0f ? 1.0f / sum.l : 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] *= inv;
    const long long row = ((long long)b * p.Hq + h) * p.T + t;
    if (rl.place == 0 && rl.at * 8 < D) store8<T>((T*)p.out + row * D + rl.at * 8, acc);
    if (lane == 0) p.lse[row] = sum.l != 0.0f ? sum.m + log2f(sum.l) : kNegInf;
}

}  // namespace dsdpa
