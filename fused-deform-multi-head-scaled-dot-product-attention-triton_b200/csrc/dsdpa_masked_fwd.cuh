// Forward of masked attention on the tensor cores, 16-bit storage, head dimensions up to 128.
//
// A block has 256 queries of one head, as two tiles of 128, and goes over the keys that any of them sees in
// blocks of 128: scores q k^T into tensor memory (fp32), the softmax weights back into the same columns
// (16 bits), p v accumulated in tensor memory.  One pass with the running maximum and sum; a row's
// accumulator is rescaled only when its maximum has grown by more than 2^8, since the division by the
// final sum makes any reference point as good (weights up to 2^8 stay far inside both types).
// Roles: two warpgroups, each with one tile's softmax (a thread has a whole row: no shuffles), one warp
// that loads tiles with TMA, one that issues the matrix instructions.  While one tile's softmax runs,
// the other tile's products do, so that both units stay busy.  (Two query tiles in turn, rescaling only past a
// threshold and the hand-over of registers are a published method of attention on this chip.)
//
// Measured, 32 heads on 8 of 8192 x 8192, bf16: D = 128 842-845 us (1.30 PFLOP/s, 0.79 of a large library matrix product's
// rate), causal 526-536 us (1.04), capped 1.35-1.37 ms (0.81), causal with a bias 611-614 us (0.90); D = 64 0.83-0.85 ms.
// Bound by the softmax: of the special-function unit's time 0.63 is used at D = 64, since a scheduler has two
// warps only and their chains (load, maximum, exp2, store) leave gaps.  A quarter of exp2 moved to the fma
// pipes did not help (832 -> 875 us at D = 128, 813 -> 791 at 64), nor did going through capped scores 32 or 64 columns
// at a time (1532 -> 1750, 1691 us at D = 128).
#pragma once

#include "dsdpa_masked.cuh"
#include "dsdpa_tc.cuh"

namespace dsdpa {

constexpr int kTileQ = 128, kTileK = 128;
constexpr int kFwdThreads = 384;               // warps 0-3, 4-7: softmax; 8: loads; 9: matrix instructions; 10, 11 idle
// The launch gives 168 registers a thread, 384 x 168 = 64512; a softmax thread holds a row of 128 scores
// and needs more, the last warpgroup hardly any: 256 x 208 + 128 x 80 = 63488.

template <int HD>
struct FwdLayout {
    static constexpr int kTileBytes = 128 * HD * 2;
    static constexpr int kStages = HD == 128 ? 5 : 8;   // K and V tiles in flight, together
    static constexpr int kSmem = 2 * kTileBytes + kStages * kTileBytes + 1024 + 512;
};

// The least positive number for 0, which it is in all but name for scores of any size.
__device__ __forceinline__ float positive_scale(float sm_scale) { return fmaxf(fabsf(sm_scale) * kLog2e, __int_as_float(1)); }

struct ScoreConsts {
    float scale2;       // sm_scale log2(e), made positive (the sign is the matrix instruction's); not 0: -inf times it is -inf
    float cap_in;       // 2 |sm_scale| / cap
    float cap_out;      // cap log2(e)
};
// Products q.k of one thread to 2 x / cap; whether all of the warp's are in half_tanh_small's range.
template <int N>
__device__ __forceinline__ bool scale_scores(float (&s)[N], const ScoreConsts& c) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const float2 a = mul2(make_float2(s[i], s[i + 1]), make_float2(c.cap_in, c.cap_in));
        s[i] = a.x;
        s[i + 1] = a.y;
    }
    return all_small(s);
}
// Products q.k of one thread to tanh(x / cap); y = cap of it.
template <int N>
__device__ __forceinline__ void cap_scores(float (&s)[N], const ScoreConsts& c) {
    if (scale_scores(s, c)) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 t = half_tanh_small(make_float2(s[i], s[i + 1]));
            s[i] = t.x;
            s[i + 1] = t.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 t = half_tanh_any(make_float2(s[i], s[i + 1]));
            s[i] = t.x;
            s[i + 1] = t.y;
        }
    }
}

// s unit - slope2 |d0 - x| for keys x = 0, 1, ...; `past`: none of them lies behind the query (the usual case, in which the
// distance needs no magnitude and the bias is linear in x).
template <int N>
__device__ __forceinline__ void add_bias(float (&s)[N], float unit, float slope2, float d0, bool past) {
    const float2 u = make_float2(unit, unit);
    if (__all_sync(0xffffffffu, past)) {
        const float2 k = make_float2(slope2, slope2), b = make_float2(-slope2 * d0, -slope2 * d0);
#pragma unroll
        for (int x = 0; x < N; x += 2) {
            const float2 v = fma2(make_float2(s[x], s[x + 1]), u, fma2(k, make_float2((float)x, (float)(x + 1)), b));
            s[x] = v.x;
            s[x + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int x = 0; x < N; ++x) s[x] = fmaf(-slope2, fabsf(d0 - (float)x), s[x] * unit);
    }
}

// A warp's rows whose values' sums something non-finite reached: once more, from the keys they see alone.  A function of its own, which
// finds its place by itself: nothing has to be kept for it while the block works.
template <typename T>
__device__ __noinline__ void redo_rows_forward(const MaskedParams& p, unsigned rows, int qtiles) {
    const int warp = threadIdx.x >> 5, bh = blockIdx.x % (p.B * p.Hq);
    const int row0 = (qtiles - 1 - (int)(blockIdx.x / (p.B * p.Hq))) * 2 * kTileQ + warp * 32;
    for (; rows; rows &= rows - 1) exact_row_forward<T>(p, bh / p.Hq, bh % p.Hq, row0 + __ffs(rows) - 1);
}

__device__ __forceinline__ int warp_min(int x) { return __reduce_min_sync(0xffffffffu, x); }
__device__ __forceinline__ int warp_max(int x) { return __reduce_max_sync(0xffffffffu, x); }

template <typename T, int HD, bool CAP, bool BIAS>
__global__ void __launch_bounds__(kFwdThreads, 1)
masked_fwd_kernel(const __grid_constant__ MaskedParams p, const __grid_constant__ CUtensorMap mq,
                  const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, int qtiles, int negate) {
    using L = FwdLayout<HD>;
    extern __shared__ char smem_raw[];
    const uint32_t smem = (smem_addr(smem_raw) + 1023u) & ~1023u;
    const uint32_t sm_q = smem, sm_ring = smem + 2 * L::kTileBytes, bars = sm_ring + L::kStages * L::kTileBytes;
    const uint32_t bar_q = bars, bar_s = bars + 8, bar_p = bars + 24, bar_o = bars + 40, bar_full = bars + 56,
                   bar_empty = bar_full + 8 * L::kStages, slot = bar_empty + 8 * L::kStages;
    __shared__ int s_lo[2], s_hi[2];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // longest rows first: with a causal mask these are the last ones
    const int bh = blockIdx.x % (p.B * p.Hq), b = bh / p.Hq, h = bh % p.Hq, hk = h / p.group;
    const int q0 = (qtiles - 1 - (int)(blockIdx.x / (p.B * p.Hq))) * 2 * kTileQ;

    if (tid < 2) { s_lo[tid] = 0x7fffffff; s_hi[tid] = 0; }
    if (tid == 0) {
        mbar_init(bar_q, 1);
        for (int t = 0; t < 2; ++t) {
            mbar_init(bar_s + 8 * t, 1);
            mbar_init(bar_p + 8 * t, 4);
            mbar_init(bar_o + 8 * t, 1);
        }
        for (int i = 0; i < L::kStages; ++i) { mbar_init(bar_full + 8 * i, 1); mbar_init(bar_empty + 8 * i, 1); }
        fence_mbar_init();
    }
    if (warp == 9) tmem_alloc(slot, 512);
    __syncthreads();
    if (warp == 8 && elect_one()) {
        mbar_expect_tx(bar_q, 2 * L::kTileBytes);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int x = 0; x < HD / kPanel; ++x)
                tma_load_4d(sm_q + t * L::kTileBytes + x * 128 * 128, &mq, x * kPanel, q0 + t * kTileQ, h, b, bar_q);
    }
    int2 r = make_int2(0, 0);
    int lo_most = -1, hi_least = 0x7fffffff;     // over the warp's rows: keys inside need no mask
    const int tile = warp >> 2, row = q0 + tile * kTileQ + (warp & 3) * 32 + lane;
    if (warp < 8) {
        if (row < p.Lq) {
            r = key_range(p, b, row);
            if (r.x >= r.y) r = make_int2(0, 0);
            lo_most = r.x;
            hi_least = r.y;
        }
        const int lo = warp_min(r.x < r.y ? r.x : 0x7fffffff), hi = warp_max(r.y);
        lo_most = warp_max(lo_most);
        hi_least = warp_min(hi_least);
        if (lane == 0) { atomicMin(&s_lo[tile], lo); atomicMax(&s_hi[tile], hi); }
    }
    uint32_t tmem;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(slot));
    int first[2], end[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const bool any = s_hi[t] > 0;
        first[t] = any ? s_lo[t] / kTileK : 0;
        end[t] = any ? (s_hi[t] + kTileK - 1) / kTileK : 0;
    }
    const int jb = end[0] == 0 ? first[1] : end[1] == 0 ? first[0] : min(first[0], first[1]), je = max(end[0], end[1]);
    auto used = [&](int t, int j) { return j >= first[t] && j < end[t]; };
    // With a bias the nearest keys, which lie last, come first: they have the large scores, and a row's reference point
    // is found once instead of moving with every tile.
    auto turn = [](int j, int from, int to) { return BIAS ? from + to - 1 - j : j; };

    if (warp >= 8) {
        regs_release<80>();
        if (warp == 8) {
            if (elect_one()) {
                int st = 0, ph = 1;      // the ring starts empty
                bool ok = true;
                for (int i = jb; i < je && ok; ++i) {
                    const int j = turn(i, jb, je);
                    if (!used(0, j) && !used(1, j)) continue;
#pragma unroll
                    for (int kv = 0; kv < 2; ++kv) {
                        if (!mbar_wait_bounded(bar_empty + 8 * st, ph, p.err)) { ok = false; break; }
                        const uint32_t dst = sm_ring + st * L::kTileBytes, full = bar_full + 8 * st;
                        mbar_expect_tx(full, L::kTileBytes);
#pragma unroll
                        for (int x = 0; x < HD / kPanel; ++x)
                            tma_load_4d(dst + x * 128 * 128, kv ? &mv : &mk, x * kPanel, j * kTileK, hk, b, full);
                        if (++st == L::kStages) { st = 0; ph ^= 1; }
                    }
                }
            }
        } else if (warp == 9) {
            if (elect_one()) {
                const uint32_t id_s = mma_desc<T>(kTileK, false, negate != 0), id_o = mma_desc<T>(HD, true);
                bool ok = mbar_wait_bounded(bar_q, 0, p.err), pending[2] = { false, false }, begun[2] = { false, false };
                int st = 0, ph = 0, vst = 0, pp[2] = { 0, 0 };
                // i == je: the products that are still to be done
                for (int i = jb; i <= je && ok; ++i) {
                    const int j = turn(i, jb, je);
                    const bool any = i < je && (used(0, j) || used(1, j));
                    if (i < je && !any) continue;
                    const bool had = pending[0] || pending[1];
                    int kst = 0;
                    if (had) {
                        vst = st;
                        if (!mbar_wait_bounded(bar_full + 8 * vst, ph, p.err)) { ok = false; break; }
                        if (++st == L::kStages) { st = 0; ph ^= 1; }
                    }
                    if (any) {
                        kst = st;
                        if (!mbar_wait_bounded(bar_full + 8 * kst, ph, p.err)) { ok = false; break; }
                        if (++st == L::kStages) { st = 0; ph ^= 1; }
                    }
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const uint32_t s_at = tmem + t * kTileK, o_at = tmem + 2 * kTileK + t * HD;
                        if (pending[t]) {
                            if (!mbar_wait_bounded(bar_p + 8 * t, pp[t], p.err)) { ok = false; break; }
                            pp[t] ^= 1;
                            tc_fence_after();
                            mma_weights<kTileK>(o_at, s_at, sm_ring + vst * L::kTileBytes, id_o, begun[t]);
                            begun[t] = true;
                            mma_commit(bar_o + 8 * t);
                            pending[t] = false;
                        }
                        if (any && used(t, j)) {
                            mma_rows<HD>(s_at, sm_q + t * L::kTileBytes, sm_ring + kst * L::kTileBytes, kTileK, id_s);
                            mma_commit(bar_s + 8 * t);
                            pending[t] = true;
                        }
                    }
                    if (!ok) break;
                    if (had) mma_commit(bar_empty + 8 * vst);
                    if (any) mma_commit(bar_empty + 8 * kst);
                }
            }
        }
    } else {
        regs_claim<208>();
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;        // 32 lanes a warp, in the address's upper half
        const uint32_t s_at = tmem + tile * kTileK + lanes, o_at = tmem + 2 * kTileK + tile * HD + lanes;
        ScoreConsts c;
        c.scale2 = positive_scale(p.sm_scale);
        c.cap_in = CAP ? 2.0f * fabsf(p.sm_scale) / p.cap : 0.0f;
        c.cap_out = CAP ? p.cap * kLog2e : 0.0f;
        const float unit = CAP ? c.cap_out : c.scale2;            // of what cap_scores, or the product, left: scores in base 2
        const float slope2 = BIAS ? __ldg(p.slopes + h) * kLog2e : 0.0f;
        const int pos = row + (p.Lk - p.Lq);
        constexpr bool kLate = CAP && !BIAS;
        float cap_term[kTanhTerms];
#pragma unroll
        for (int i = 0; i < kTanhTerms; ++i) cap_term[i] = kLate ? tanh_term(i) * c.cap_out : 0.0f;
        float m = kNegInf, l = 0.0f;
        int n = 0;
        bool ok = true;
        for (int i = first[tile]; i < end[tile]; ++i, ++n) {
            if (!mbar_wait_bounded(bar_s + 8 * tile, n & 1, p.err)) { ok = false; break; }
            tc_fence_after();
            float s[kTileK];
#pragma unroll
            for (int x = 0; x < kTileK; x += 32) tmem_ld32(s_at + x, s + x);
            tmem_wait_ld();
            const int n0 = turn(i, first[tile], end[tile]) * kTileK;
            const int a = r.x - n0, e = r.y - n0;
            const bool partial = lo_most > n0 || hi_least < n0 + kTileK;
            float top;
            bool small = false;
            auto largest = [&]() {
                float mx[4] = { s[0], s[1], s[2], s[3] };
#pragma unroll
                for (int x = 4; x < kTileK; ++x) mx[x & 3] = fmaxf(mx[x & 3], s[x]);
                return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
            };
            if (kLate) {
                // the cap keeps the order: the largest score is the largest product's, and the cap itself is done together with
                // exp2, so that the fma pipes and the special-function unit work at the same time
                small = scale_scores(s, c);
                if (partial) {
                    top = kNegInf;
#pragma unroll
                    for (int x = 0; x < kTileK; ++x) top = fmaxf(top, x >= a && x < e ? s[x] : kNegInf);
                    if (max(a, 0) < min(e, kTileK)) top = half_tanh(top) * unit;
                } else {
                    top = half_tanh(largest()) * unit;
                }
            } else {
                if (CAP) cap_scores(s, c);
                if (BIAS) add_bias(s, unit, slope2, (float)(pos - n0), pos - n0 >= kTileK - 1);
                if (partial) {
#pragma unroll
                    for (int x = 0; x < kTileK; ++x) s[x] = x >= a && x < e ? s[x] : kNegInf;
                }
                top = largest();
                if (!BIAS) top *= unit;                           // not negative: the order stays
            }
            // the reference point moves when a row's maximum is more than 8 above it (or it has none yet)
            const bool move = top > m + 8.0f || (m == kNegInf && top > kNegInf);
            if (__any_sync(0xffffffffu, move)) {
                const float f = move ? (m == kNegInf ? 0.0f : fast_exp2(m - top)) : 1.0f;
                if (move) m = top;
                l *= f;
                if (n > 0) {
                    if (!mbar_wait_bounded(bar_o + 8 * tile, (n - 1) & 1, p.err)) { ok = false; break; }
                    tc_fence_after();
#pragma unroll
                    for (int x = 0; x < HD; x += 32) {
                        float o[32];
                        tmem_ld32(o_at + x, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int y = 0; y < 32; ++y) o[y] *= f;
                        tmem_st32(o_at + x, reinterpret_cast<const uint32_t*>(o));
                    }
                }
            }
            const float m0 = m == kNegInf ? 0.0f : m;
            float2 sum[2] = { make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f) };
            const float2 scale = make_float2(unit, unit), to = make_float2(-m0, -m0);
            // weights from what `score` says of two columns, less the reference point
            auto weigh = [&](auto score) {
#pragma unroll
                for (int x = 0; x < kTileK; x += 32) {
                    uint32_t w[16];
#pragma unroll
                    for (int y = 0; y < 32; y += 2) {
                        const float2 v = score(x + y), e = make_float2(fast_exp2(v.x), fast_exp2(v.y));
                        sum[(y >> 1) & 1] = add2(sum[(y >> 1) & 1], e);
                        w[y / 2] = pack2<T>(e.x, e.y);
                    }
                    tmem_st16(s_at + x / 2, w);
                }
            };
            if constexpr (kLate) {
                auto seen = [&](int x, float2 v) { return make_float2(x >= a && x < e ? v.x : kNegInf, x + 1 >= a && x + 1 < e ? v.y : kNegInf); };
                auto capped = [&](int x) {
                    const float2 v = make_float2(s[x], s[x + 1]), u = mul2(v, v);
                    float2 t = make_float2(cap_term[kTanhTerms - 1], cap_term[kTanhTerms - 1]);
#pragma unroll
                    for (int i = kTanhTerms - 2; i >= 0; --i) t = fma2(t, u, make_float2(cap_term[i], cap_term[i]));
                    return fma2(t, v, to);
                };
                // each by its own size, as half_tanh_any has it
                auto any = [&](int x) {
                    const float2 t = capped(x), g = fma2(make_float2(half_tanh(s[x]), half_tanh(s[x + 1])), scale, to);
                    return make_float2(is_small(s[x]) ? t.x : g.x, is_small(s[x + 1]) ? t.y : g.y);
                };
                if (!small) weigh([&](int x) { return seen(x, any(x)); });
                else if (partial) weigh([&](int x) { return seen(x, capped(x)); });
                else weigh(capped);
            } else {
                weigh([&](int x) {
                    const float2 v = make_float2(s[x], s[x + 1]);
                    return BIAS ? add2(v, to) : fma2(v, scale, to);
                });
            }
            l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_p + 8 * tile);
        }
        if (ok && n > 0) ok = mbar_wait_bounded(bar_o + 8 * tile, (n - 1) & 1, p.err);
        if (ok) {
            tc_fence_after();
            const float inv = l != 0.0f ? 1.0f / l : 0.0f;
            bool fine = true;
#pragma unroll
            for (int x = 0; x < HD; x += 32) {
                float o[32];
                if (n > 0) {
                    tmem_ld32(o_at + x, o);
                    tmem_wait_ld();
                }
                if (row < p.Lq) {
                    T* out = row_of<T>(p.out, p.so, b, h, row) + x;
#pragma unroll
                    for (int y = 0; y < 32; y += 8) {
                        float v[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            v[e] = n > 0 && l != 0.0f ? o[y + e] * inv : 0.0f;
                            fine = fine && fabsf(v[e]) <= 3.0e38f;
                        }
                        if (x + y < p.D) stg128(out + y, pack16(v, (T*)nullptr));
                    }
                }
            }
            if (row < p.Lq) p.lse[(long long)bh * p.Lq + row] = l != 0.0f ? m + log2f(l) : kNegInf;
            // (a sum of weights that is NaN is the row's own)
            const unsigned bad = __ballot_sync(0xffffffffu, row < p.Lq && !fine && l == l);
            __syncwarp();
            if (bad) redo_rows_forward<T>(p, bad, qtiles);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 9) tmem_free(tmem, 512);
}

}  // namespace dsdpa
