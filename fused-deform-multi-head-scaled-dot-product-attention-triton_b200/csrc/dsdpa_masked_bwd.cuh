// Backward of masked attention on the tensor cores, 16-bit storage, head dimensions up to 128: two kernels,
// both of which compute the scores again.
//
//   masked_dq_kernel    a block has 128 queries of one head and goes over their keys:
//                         S = q k^T, dP = dout v^T, dS = P (dP - delta), dq += dS k
//   masked_dkdv_kernel  a block has 128 keys of one key/value head and goes over the queries that see them, of all
//                       heads of the group:  S^T = k q^T, dP^T = v dout^T, dv += P^T dout, dk += dS^T q
//
// Every gradient has one writer and one order of sums, so two runs give the same bits; the price, against
// one kernel that adds dq up with atomics, is seven products a tile pair instead of five.  P and dS go to
// tensor memory in the storage type, as operands; everything before them and every sum is fp32.  For fp16 P^T is
// scaled by 2^15 and dS by a power of two: dq's by the row's largest |dout|, dk's by a bound of what the key's row of dS^T can
// hold, since even weights of many keys, or a loss that is scaled far down, would take them out of the type's range.
// Both kernels: 8 warps of elementwise work (a thread has one row and 64 of its 128 columns), one warp of
// TMA loads, one that issues the matrix instructions.
//
// Measured, 32 heads on 8 of 8192 x 8192, bf16, D = 128: 3.14-3.29 ms, 0.86 PFLOP/s by the formula's five products and 1.20
// by the seven done; causal 1.64 ms (0.84); capped 4.33-4.42 ms; 4 x 16 heads of 2048, D = 64: 345 us (0.50).  D = 128 is near the
// products' rate; at D = 64 these are half as long and the elementwise work between them bounds.
// Tiles of 64 columns, one for each half of the threads and half a turn apart, were slower: products of that
// width wait for shared memory (3473 -> 4074 us, D = 128).
#pragma once

#include "dsdpa_masked_fwd.cuh"

namespace dsdpa {

constexpr int kBwdThreads = 320;

struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };

__device__ __forceinline__ float4 lds_float4(uint32_t at) {
    float4 f;
    asm("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w) : "r"(at) : "memory");
    return f;
}

// What masked_dq_kernel leaves for masked_dkdv_kernel, in whole tiles of 128 queries.  Odd queries are spoilt ones (what sees
// them becomes NaN) and such as see no key but hold something non-finite: masked_dkdv_kernel keeps their rows out of
// the sums that they have no part in.
struct BwdStats {
    float* stats;     // [B, Hq, tiles][2][128]: -lse (-inf: no weight; NaN: an odd query), and -delta
    int2* ranges;     // [B, tiles * 128]: visible keys
    int4* tiles;      // [B, tiles]: least lo, largest hi over rows that see something; largest lo, least hi over all rows
    unsigned* amax;   // [B, Hq, tiles]: bit 8: the tile has an odd query; fp16: exponent fields of the largest |dout| (bits 0-7) and
                      // the largest |delta| (bits 16-23) of the others
    int n;            // tiles of a sequence
};

// 2^-e for numbers in [2^e, 2^(e+1)), from their exponent field; 1 for zero, infinity and NaN.
__device__ __forceinline__ float scale_down(unsigned e) {
    return e == 0 || e >= 254 ? 1.0f : __uint_as_float((unsigned)(254 - e) << 23);
}

// Power of two that P^T of fp16 is scaled by: weights are at most 1, the type's largest number is above 2^15.
constexpr float kWeightBits = 15.0f, kWeightUp = 32768.0f;
// Scale of dS of a key whose row of V has the sum of magnitudes `norm`, from the exponent fields of the largest |dout| and
// |delta|: |dp - delta| < 2^(fields - 126) each way, so that dS, whose weights are at most 1, stays below 2^14.
__device__ __forceinline__ float scale_up(float norm, unsigned dout, unsigned delta) {
    const float most = fmaf(norm, __uint_as_float(min(dout + 1u, 254u) << 23), __uint_as_float(min(delta + 1u, 254u) << 23));
    const unsigned e = __float_as_uint(most) >> 23;             // most < 2^(e - 126)
    return e >= 254u ? 1.0f : __uint_as_float(min(267u - e, 200u) << 23);
}

// Two products that scale_scores has been at to tanh(x / cap); as they are where there is no cap.  Done pair by pair with what
// follows, so that the fma pipes and the special-function unit work at the same time.
template <bool CAP, bool SMALL>
__device__ __forceinline__ float2 capped_pair(float2 a) {
    if (!CAP) return a;
    return SMALL ? half_tanh_small(a) : half_tanh_any(a);
}
// The weights of two pairs from what capped_pair left; `slope` gets the factors that the cap's derivative
// puts on ds: 1 - tanh^2.
template <bool CAP, bool BIAS>
__device__ __forceinline__ float2 pair_weights(float2 t, float unit, float slope2, float2 dist, float2 neg_lse, float2& slope) {
    float2 s = fma2(t, make_float2(unit, unit), neg_lse);
    if (CAP) slope = fma2(make_float2(-t.x, -t.y), t, make_float2(1.0f, 1.0f));
    if (BIAS) s = fma2(make_float2(-slope2, -slope2), make_float2(fabsf(dist.x), fabsf(dist.y)), s);
    return make_float2(fast_exp2(s.x), fast_exp2(s.y));
}

// Rows of a block's tile that something non-finite reached (bits of `bad`, by warps of either half of the threads): once more, from
// what they see alone, shared out over the block's warps.  A function of its own, which finds its place by itself:
// nothing has to be kept for it while the block works.
template <typename T, bool KEYS>
__device__ __noinline__ void redo_rows(const MaskedParams& p, const unsigned* bad, int tiles) {
    const int warp = threadIdx.x >> 5, heads = KEYS ? p.Hkv : p.Hq;
    const int bh = blockIdx.x % (p.B * heads), b = bh / heads, h = bh % heads, block = (int)(blockIdx.x / (p.B * heads));
    const int row0 = KEYS ? block * kTileK : (tiles - 1 - block) * kTileQ;
    int turn = 0;
    for (int quad = 0; quad < 4; ++quad)
        for (unsigned rows = bad[quad] | bad[quad + 4]; rows; rows &= rows - 1) {
            if (turn++ % (kBwdThreads / 32) != warp) continue;
            const int row = row0 + quad * 32 + __ffs(rows) - 1;
            if constexpr (KEYS) exact_row_dkdv<T>(p, b, h, row);
            else exact_row_dq<T>(p, b, h, row);
        }
}
__device__ __forceinline__ bool any_bad(const unsigned (&bad)[8]) {
    unsigned any = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) any |= bad[i];
    return any != 0u;
}

// d[128 x HD] (+)= w[128 x 128] b[128 x HD]; w's halves lie in columns 0 .. 31 and 64 .. 95 of its region, each
// where the half of the scores was that the same threads have read.
template <int HD>
__device__ __forceinline__ void mma_halves(uint32_t d, uint32_t w, uint32_t b, uint32_t idesc, bool add) {
#pragma unroll
    for (int s = 0; s < 8; ++s)
        mma_ts(d, w + (s & 3) * 8 + (s >> 2) * 64, smem_desc(b + s * 2048, 128 * 128), idesc, add || s > 0);
}

// Sums of p dp and of p over this thread's 64 columns of the block's only key tile, whose scores and dP lie in tensor memory.
template <bool CAP, bool BIAS>
__device__ __noinline__ float2 weigh_dp(uint32_t s_at, uint32_t d_at, const ScoreConsts c, float lse, float slope2, float d0, int a, int e) {
    const float unit = CAP ? c.cap_out : c.scale2;
    float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll 1
    for (int x = 0; x < 64; x += 32) {
        float s[32], dp[32];
        tmem_ld32(s_at + x, s);
        tmem_ld32(d_at + x, dp);
        tmem_wait_ld();
        if (CAP) cap_scores(s, c);
#pragma unroll
        for (int y = 0; y < 32; y += 2) {
            const float at = (float)(x + y);
            float2 slope;
            const float2 w = pair_weights<false, BIAS>(make_float2(s[y], s[y + 1]), unit, slope2, make_float2(d0 - at, d0 - at - 1.0f), make_float2(-lse, -lse), slope);
            if (x + y >= a && x + y < e && w.x != 0.0f) { sum.x = fmaf(w.x, dp[y], sum.x); sum.y += w.x; }
            if (x + y + 1 >= a && x + y + 1 < e && w.y != 0.0f) { sum.x = fmaf(w.y, dp[y + 1], sum.x); sum.y += w.y; }
        }
    }
    return sum;
}

template <typename T, int HD, bool CAP, bool BIAS>
__global__ void __launch_bounds__(kBwdThreads, 1)
masked_dq_kernel(const __grid_constant__ MaskedParams p, const __grid_constant__ BwdStats st, const __grid_constant__ CUtensorMap mq,
                 const __grid_constant__ CUtensorMap mdo, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                 int negate) {
    using L = FwdLayout<HD>;     // q and dout where the forward has its two tiles, then the ring of k and v tiles
    constexpr bool kScaled = DtypeOf<T>::value == DSDPA_F16;
    extern __shared__ char smem_raw[];
    const uint32_t smem = (smem_addr(smem_raw) + 1023u) & ~1023u;
    const uint32_t sm_q = smem, sm_do = smem + L::kTileBytes, sm_ring = smem + 2 * L::kTileBytes, bars = sm_ring + L::kStages * L::kTileBytes;
    const uint32_t bar_q = bars, bar_s = bars + 8, bar_dp = bars + 24, bar_ds = bars + 32, bar_done = bars + 40, bar_full = bars + 48,
                   bar_empty = bar_full + 8 * L::kStages, slot = bar_empty + 8 * L::kStages;
    __shared__ int s_lo, s_hi, s_lomax, s_himin;
    __shared__ unsigned s_top, s_delta, s_odd;
    __shared__ float s_part[2][kTileQ];
    __shared__ unsigned char s_big[2][kTileQ];
    __shared__ unsigned s_bad[8];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int bh = blockIdx.x % (p.B * p.Hq), b = bh / p.Hq, h = bh % p.Hq, hk = h / p.group;
    const int qt = st.n - 1 - (int)(blockIdx.x / (p.B * p.Hq)), q0 = qt * kTileQ;

    if (tid == 0) {
        s_lo = 0x7fffffff; s_hi = 0; s_lomax = -1; s_himin = 0x7fffffff; s_top = s_delta = s_odd = 0;
        mbar_init(bar_q, 1);
        mbar_init(bar_s, 1);
        mbar_init(bar_s + 8, 1);
        mbar_init(bar_dp, 1);
        mbar_init(bar_ds, 8);
        mbar_init(bar_done, 1);
        for (int i = 0; i < L::kStages; ++i) { mbar_init(bar_full + 8 * i, 1); mbar_init(bar_empty + 8 * i, 1); }
        fence_mbar_init();
    }
    if (warp == 9) tmem_alloc(slot, 512);
    __syncthreads();
    if (warp == 8 && elect_one()) {
        mbar_expect_tx(bar_q, 2 * L::kTileBytes);
#pragma unroll
        for (int x = 0; x < HD / kPanel; ++x) {
            tma_load_4d(sm_q + x * 128 * 128, &mq, x * kPanel, q0, h, b, bar_q);
            tma_load_4d(sm_do + x * 128 * 128, &mdo, x * kPanel, q0, h, b, bar_q);
        }
    }
    const int half = warp >> 2, in_tile = (warp & 3) * 32 + lane, row = q0 + in_tile;
    int2 r = make_int2(0, 0);
    int lo_most = -1, hi_least = 0x7fffffff;
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
        if (lane == 0 && half == 0) {
            atomicMin(&s_lo, lo);
            atomicMax(&s_hi, hi);
            atomicMax(&s_lomax, lo_most);
            atomicMin(&s_himin, hi_least);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    uint32_t tmem;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(slot));
    const int first = s_hi > 0 ? s_lo / kTileK : 0, n = s_hi > 0 ? (s_hi + kTileK - 1) / kTileK - first : 0;
    if (tid == 0 && h == 0) st.tiles[(long long)b * st.n + qt] = make_int4(s_lo, s_hi, s_lomax, s_himin);

    if (warp == 8) {
        if (elect_one() && n > 0) {
            int at = 0, ph = 1;
            bool ok = true;
            for (int i = 0; i < n && ok; ++i)
#pragma unroll
                for (int kv = 0; kv < 2; ++kv) {
                    if (!mbar_wait_bounded(bar_empty + 8 * at, ph, p.err)) { ok = false; break; }
                    const uint32_t dst = sm_ring + at * L::kTileBytes, full = bar_full + 8 * at;
                    mbar_expect_tx(full, L::kTileBytes);
#pragma unroll
                    for (int x = 0; x < HD / kPanel; ++x)
                        tma_load_4d(dst + x * 128 * 128, kv ? &mv : &mk, x * kPanel, (first + i) * kTileK, hk, b, full);
                    if (++at == L::kStages) { at = 0; ph ^= 1; }
                }
        }
    } else if (warp == 9) {
        // (a block without keys waits for its queries too: it must not end before they are there)
        if (elect_one()) {
            // columns: S of even and of odd key blocks (dS in their place), dP, dq
            const uint32_t id_s = mma_desc<T>(kTileK, false, negate != 0), id_dp = mma_desc<T>(kTileK, false), id_dq = mma_desc<T>(HD, true);
            const uint32_t t_dp = tmem + 256, t_dq = tmem + 384;
            bool ok = mbar_wait_bounded(bar_q, 0, p.err) && n > 0;
            auto tile = [&](int e) { return sm_ring + (uint32_t)(e % L::kStages) * L::kTileBytes; };     // entry e: k of block e/2, or v
            auto arrived = [&](int e) { return mbar_wait_bounded(bar_full + 8 * (e % L::kStages), (e / L::kStages) & 1, p.err); };
            auto score = [&](int i) {
                if (!arrived(2 * i)) return false;
                mma_rows<HD>(tmem + (i & 1) * kTileK, sm_q, tile(2 * i), kTileK, id_s);
                mma_commit(bar_s + 8 * (i & 1));
                return true;
            };
            auto dprod = [&](int i) {
                if (!arrived(2 * i + 1)) return false;
                mma_rows<HD>(t_dp, sm_do, tile(2 * i + 1), kTileK, id_dp);
                mma_commit(bar_dp);
                mma_commit(bar_empty + 8 * ((2 * i + 1) % L::kStages));
                return true;
            };
            ok = ok && score(0) && dprod(0) && (n < 2 || score(1));
            for (int i = 0; i < n && ok; ++i) {
                if (!(ok = mbar_wait_bounded(bar_ds, i & 1, p.err))) break;
                tc_fence_after();
                if (i + 1 < n && !(ok = dprod(i + 1))) break;
                mma_halves<HD>(t_dq, tmem + (i & 1) * kTileK, tile(2 * i), id_dq, i > 0);
                mma_commit(bar_empty + 8 * ((2 * i) % L::kStages));
                if (i + 2 < n) ok = score(i + 2);
            }
            if (ok) mma_commit(bar_done);
        }
    } else {
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;
        ScoreConsts c;
        c.scale2 = fabsf(p.sm_scale) * kLog2e;
        c.cap_in = CAP ? 2.0f * fabsf(p.sm_scale) / p.cap : 0.0f;
        c.cap_out = CAP ? p.cap * kLog2e : 0.0f;
        const float unit = CAP ? c.cap_out : c.scale2;
        const float slope2 = BIAS ? __ldg(p.slopes + h) * kLog2e : 0.0f;
        const bool sees = r.x < r.y;
        // delta = out.dout, while the first products are made: each half of the threads has half of the row
        float sum = 0.0f;
        unsigned most = 0;
        if (sees) {
            const T* o = row_of<T>(p.out_in, p.so, b, h, row);
            const T* g = row_of<T>(p.dout, p.sdo, b, h, row);
#pragma unroll
            for (int x = 0; x < HD / 2; x += 8) {
                const int d = half * (HD / 2) + x;
                if (d < p.D) {
                    float a[8], e[8];
                    load8<T>(o + d, a);
                    load8<T>(g + d, e);
                    sum += dot8(a, e);
                    if (kScaled) {
#pragma unroll
                        for (int y = 0; y < 8; ++y) most = max(most, __float_as_uint(e[y]) & 0x7fffffffu);
                    }
                }
            }
        } else if (row < p.Lq) {
            // NaN where its rows hold something non-finite
            const T* a = row_of<T>(p.q, p.sq, b, h, row);
            const T* g = row_of<T>(p.dout, p.sdo, b, h, row);
#pragma unroll
            for (int z = 0; z < HD / 2; z += 8) {
                const int d = half * (HD / 2) + z;
                if (d < p.D) {
                    float x[8], y[8];
                    load8<T>(a + d, x);
                    load8<T>(g + d, y);
#pragma unroll
                    for (int e = 0; e < 8; ++e) sum = fmaf(x[e], 0.0f, fmaf(y[e], 0.0f, sum));
                }
            }
        }
        s_part[half][in_tile] = sum;
        s_big[half][in_tile] = (unsigned char)(most >> 23);
        asm volatile("bar.sync 1, 256;" ::: "memory");
        float delta = s_part[0][in_tile] + s_part[1][in_tile];
        const int pos = row + (p.Lk - p.Lq);
        const unsigned big = max((unsigned)s_big[0][in_tile], (unsigned)s_big[1][in_tile]);
        const float sigma = kScaled ? scale_down(big) : 1.0f;
        const long long at = (long long)bh * p.Lq + row;
        float lse = sees ? p.lse[at] : kNegInf;
        if (lse == kNegInf) lse = -kNegInf;                 // weight exp2(s - inf) = 0
        bool ok = true;
        if (n == 1) {
            // A row of a few keys may have nearly all of its weight on one of them; its gradients are then differences in which out's
            // rounding to storage shows (two keys, bf16: dq off by up to 5 %).  Where the keys are one tile delta comes from
            // p and dp themselves.
            const int n0 = first * kTileK + half * 64;
            const uint32_t mine = sm_ring + 2 * L::kTileBytes + in_tile * 8;       // of the ring, which holds two tiles
            ok = mbar_wait_bounded(bar_s, 0, p.err) && mbar_wait_bounded(bar_dp, 0, p.err);
            tc_fence_after();
            const float2 sum = weigh_dp<CAP, BIAS>(tmem + half * 64 + lanes, tmem + 256 + half * 64 + lanes, c, lse, slope2, (float)(pos - n0), r.x - n0, r.y - n0);
            asm volatile("st.shared.v2.f32 [%0], {%1, %2};" :: "r"(mine + half * kTileQ * 8), "f"(sum.x), "f"(sum.y) : "memory");
            asm volatile("bar.sync 1, 256;" ::: "memory");
            float2 other;
            asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(other.x), "=f"(other.y) : "r"(mine + (half ^ 1) * kTileQ * 8) : "memory");
            const float all = half ? other.y + sum.y : sum.y + other.y;
            if (sees && all != 0.0f) delta = (half ? other.x + sum.x : sum.x + other.x) / all;
        }
        if (half == 0) {
            const bool odd = sees ? spoilt(lse, delta) : delta != delta;
            if (odd) s_odd = 1;
            float* stats = st.stats + ((long long)bh * st.n + qt) * 2 * kTileQ + in_tile;
            stats[0] = odd ? __int_as_float(0x7fffffff) : kScaled ? kWeightBits - lse : -lse;
            stats[kTileQ] = odd || !sees ? 0.0f : -delta;
            if (!sees) delta = 0.0f;
            if (h == 0) st.ranges[(long long)b * st.n * kTileQ + row] = r;
            if (row < p.Lq) p.delta[at] = delta;
            if (kScaled) {
                const unsigned top = __reduce_max_sync(0xffffffffu, odd ? 0u : big);
                const unsigned most = __reduce_max_sync(0xffffffffu, odd ? 0u : (__float_as_uint(delta) & 0x7fffffffu) >> 23);
                if (lane == 0) { atomicMax(&s_top, top); atomicMax(&s_delta, most); }
            }
        }
        const float ndelta = sees ? -delta * sigma : 0.0f;
        for (int i = 0; i < n && ok; ++i) {
            const uint32_t s_at = tmem + (i & 1) * kTileK + half * 64 + lanes, d_at = tmem + 256 + half * 64 + lanes;
            float w[64];
            if (!mbar_wait_bounded(bar_s + 8 * (i & 1), (i >> 1) & 1, p.err)) { ok = false; break; }
            tc_fence_after();
            tmem_ld32(s_at, w);
            tmem_ld32(s_at + 32, w + 32);
            tmem_wait_ld();
            const int n0 = (first + i) * kTileK + half * 64;
            const float d0 = (float)(pos - n0);
            const bool partial = lo_most > n0 || hi_least < n0 + 64;
            const int a = r.x - n0, e = r.y - n0;
            auto weights = [&](auto small) {
#pragma unroll
                for (int x = 0; x < 64; x += 2) {
                    const float2 y = capped_pair<CAP, decltype(small)::value>(make_float2(w[x], w[x + 1]));
                    float2 slope, v = pair_weights<CAP, BIAS>(y, unit, slope2, add2(make_float2(d0, d0), make_float2(-(float)x, -(float)(x + 1))),
                                                              make_float2(-lse, -lse), slope);
                    if (CAP) v = mul2(v, slope);
                    w[x] = v.x;
                    w[x + 1] = v.y;
                }
            };
            if (!CAP || scale_scores(w, c)) weights(Yes{});
            else weights(No{});
            if (partial) {
#pragma unroll
                for (int x = 0; x < 64; ++x) w[x] = x >= a && x < e ? w[x] : 0.0f;
            }
            if (!mbar_wait_bounded(bar_dp, i & 1, p.err)) { ok = false; break; }
            tc_fence_after();
#pragma unroll
            for (int x = 0; x < 64; x += 32) {
                float d[32];
                uint32_t o[16];
                tmem_ld32(d_at + x, d);
                tmem_wait_ld();
#pragma unroll
                for (int y = 0; y < 32; y += 2) {
                    const float2 dp = make_float2(d[y], d[y + 1]), nd = make_float2(ndelta, ndelta);
                    const float2 u = kScaled ? fma2(dp, make_float2(sigma, sigma), nd) : add2(dp, nd);
                    const float2 ds = mul2(make_float2(w[x + y], w[x + y + 1]), u);
                    o[y / 2] = pack2<T>(ds.x, ds.y);
                }
                tmem_st16(s_at + x / 2, o);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_ds);
        }
        if (ok && n > 0) ok = mbar_wait_bounded(bar_done, 0, p.err);
        if (ok) {
            tc_fence_after();
            const float back = p.sm_scale / sigma;         // sigma is a power of two
            bool fine = true;
#pragma unroll
            for (int x = 0; x < HD / 2; x += 32) {
                float o[32];
                const int d0 = half * (HD / 2) + x;
                if (n > 0) {
                    tmem_ld32(tmem + 384 + d0 + lanes, o);
                    tmem_wait_ld();
                }
                if (row < p.Lq) {
                    T* out = row_of<T>(p.dq, p.sdq, b, h, row) + d0;
#pragma unroll
                    for (int y = 0; y < 32; y += 8) {
                        float v[8];
#pragma unroll
                        for (int z = 0; z < 8; ++z) {
                            v[z] = n > 0 ? o[y + z] * back : 0.0f;
                            fine = fine && fabsf(v[z]) <= 3.0e38f;
                        }
                        if (d0 + y < p.D) stg128(out + y, pack16(v, (T*)nullptr));
                    }
                }
            }
            const unsigned bad = __ballot_sync(0xffffffffu, n > 0 && row < p.Lq && !fine && !spoilt(lse, delta));
            if (lane == 0) s_bad[warp] = bad;
        } else if (lane == 0) s_bad[warp] = 0;
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 9) tmem_free(tmem, 512);
    if (tid == 0) st.amax[(long long)bh * st.n + qt] = s_top | s_odd << 8 | s_delta << 16;
    if (any_bad(s_bad)) redo_rows<T, false>(p, s_bad, st.n);
}

// The rows of a tile's odd queries to zero before any product reads them, by one thread: scores and dP^T of a query that a key does not
// see are then finite whatever it holds, and the zeros of P^T and dS^T keep it out of the sums.
template <int HD>
__device__ __noinline__ void clear_odd_rows(uint32_t tile, uint32_t stats) {
    for (int r = 0; r < kTileQ; ++r) {
        float stat;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(stat) : "r"(stats + r * 4) : "memory");
        if (stat != stat)
            for (int x = 0; x < HD / 8; ++x)
                asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" :: "r"(tile + x / 8 * 128 * 128 + r * 128 + x % 8 * 16), "r"(0) : "memory");
    }
    fence_proxy_async();
}

template <int HD>
struct DkdvLayout {
    static constexpr int kTileBytes = 128 * HD * 2;
    static constexpr int kRowBytes = 128 * 8;                       // stats, or ranges, of a tile
    static constexpr int kStage = 2 * kTileBytes + 2 * kRowBytes;   // q, dout, stats, ranges
    static constexpr int kSmem = 2 * kTileBytes + 2 * kStage + 1024 + 256;
};

template <typename T, int HD, bool CAP, bool BIAS>
__global__ void __launch_bounds__(kBwdThreads, 1)
masked_dkdv_kernel(const __grid_constant__ MaskedParams p, const __grid_constant__ BwdStats st, const __grid_constant__ CUtensorMap mq,
                   const __grid_constant__ CUtensorMap mdo, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                   int negate) {
    using L = DkdvLayout<HD>;
    constexpr bool kScaled = DtypeOf<T>::value == DSDPA_F16;
    extern __shared__ char smem_raw[];
    const uint32_t smem = (smem_addr(smem_raw) + 1023u) & ~1023u;
    const uint32_t sm_k = smem, sm_v = smem + L::kTileBytes, sm_q = smem + 2 * L::kTileBytes;    // q and dout of both stages first
    const uint32_t sm_rows = sm_q + 4 * L::kTileBytes, bars = sm_rows + 4 * L::kRowBytes;
    const uint32_t bar_kv = bars, bar_qf = bars + 8, bar_qe = bars + 24, bar_of = bars + 40, bar_oe = bars + 56, bar_s = bars + 72,
                   bar_dp = bars + 80, bar_p = bars + 88, bar_ds = bars + 96, bar_done = bars + 104, slot = bars + 112;
    __shared__ int s_first, s_end;
    __shared__ unsigned s_bad[8], s_top, s_delta, s_odd;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int bh = blockIdx.x % (p.B * p.Hkv), b = bh / p.Hkv, hk = bh % p.Hkv;
    const int k0 = (int)(blockIdx.x / (p.B * p.Hkv)) * kTileK;       // first keys first: with a causal mask most queries see them
    auto tile_q = [&](int e) { return sm_q + (uint32_t)(e & 1) * 2 * L::kTileBytes; };
    auto tile_do = [&](int e) { return tile_q(e) + L::kTileBytes; };
    auto tile_rows = [&](int e) { return sm_rows + (uint32_t)(e & 1) * 2 * L::kRowBytes; };

    if (tid == 0) {
        s_first = 0x7fffffff; s_end = 0; s_top = s_delta = s_odd = 0;
        mbar_init(bar_kv, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar_qf + 8 * i, 1);
            mbar_init(bar_qe + 8 * i, 1);
            mbar_init(bar_of + 8 * i, 1);
            mbar_init(bar_oe + 8 * i, 1);
        }
        mbar_init(bar_s, 1);
        mbar_init(bar_dp, 1);
        mbar_init(bar_p, 8);
        mbar_init(bar_ds, 8);
        mbar_init(bar_done, 1);
        fence_mbar_init();
    }
    if (warp == 9) tmem_alloc(slot, 512);
    __syncthreads();
    if (warp == 8 && elect_one()) {
        mbar_expect_tx(bar_kv, 2 * L::kTileBytes);
#pragma unroll
        for (int x = 0; x < HD / kPanel; ++x) {
            tma_load_4d(sm_k + x * 128 * 128, &mk, x * kPanel, k0, hk, b, bar_kv);
            tma_load_4d(sm_v + x * 128 * 128, &mv, x * kPanel, k0, hk, b, bar_kv);
        }
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");      // masked_dq_kernel's results from here on
    // the query tiles between the first and the last that see any of these keys; the largest |dout| and |delta| of those that do;
    // whether any has odd queries
    int lo = 0x7fffffff, hi = 0;
    const unsigned* amax = st.amax + (long long)(b * p.Hq + hk * p.group) * st.n;
    unsigned top = 0, most = 0, odd = 0;
    for (int i = tid; i < p.group * st.n; i += kBwdThreads) {          // a head's tile a step: one wait for memory, mostly
        const int tile = i % st.n;
        const int4 t = st.tiles[(long long)b * st.n + tile];
        const unsigned a = amax[i];
        odd |= a >> 8 & 1u;
        if (t.x < k0 + kTileK && t.y > k0) {
            lo = min(lo, tile);
            hi = max(hi, tile + 1);
            if (kScaled) { top = max(top, a & 255u); most = max(most, a >> 16); }
        }
    }
    lo = warp_min(lo);
    hi = warp_max(hi);
    if (lane == 0) { atomicMin(&s_first, lo); atomicMax(&s_end, hi); }
    if (kScaled) {
        top = __reduce_max_sync(0xffffffffu, top);
        most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0) { atomicMax(&s_top, top); atomicMax(&s_delta, most); }
    }
    if (odd) s_odd = 1;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    uint32_t tmem;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(slot));
    const int first = s_first, span = s_end > 0 ? s_end - first : 0, n = span * p.group;

    if (warp == 8) {
        if (elect_one() && n > 0) {
            bool ok = true;
            for (int e = 0; e < n && ok; ++e) {
                const int h = hk * p.group + e / span, q0 = (first + e % span) * kTileQ;
                const uint32_t ph = ((e >> 1) & 1) ^ 1, full = bar_qf + 8 * (e & 1), dfull = bar_of + 8 * (e & 1);
                if (!(ok = mbar_wait_bounded(bar_qe + 8 * (e & 1), ph, p.err))) break;
                mbar_expect_tx(full, L::kTileBytes + 2 * L::kRowBytes);
#pragma unroll
                for (int x = 0; x < HD / kPanel; ++x) tma_load_4d(tile_q(e) + x * 128 * 128, &mq, x * kPanel, q0, h, b, full);
                bulk_g2s(tile_rows(e), st.stats + (((long long)b * p.Hq + h) * st.n * kTileQ + q0) * 2, L::kRowBytes, full);
                bulk_g2s(tile_rows(e) + L::kRowBytes, st.ranges + (long long)b * st.n * kTileQ + q0, L::kRowBytes, full);
                if (!(ok = mbar_wait_bounded(bar_oe + 8 * (e & 1), ph, p.err))) break;
                mbar_expect_tx(dfull, L::kTileBytes);
#pragma unroll
                for (int x = 0; x < HD / kPanel; ++x) tma_load_4d(tile_do(e) + x * 128 * 128, &mdo, x * kPanel, q0, h, b, dfull);
            }
        }
    } else if (warp == 9) {
        if (elect_one()) {
            // columns: S^T (P^T in its place), dP^T (dS^T in its place), dv, dk
            const uint32_t id_s = mma_desc<T>(kTileQ, false, negate != 0), id_dp = mma_desc<T>(kTileQ, false), id_g = mma_desc<T>(HD, true);
            const uint32_t t_dp = tmem + 128, t_dv = tmem + 256, t_dk = tmem + 384;
            bool ok = mbar_wait_bounded(bar_kv, 0, p.err) && n > 0;
            auto clean = [&](int e, uint32_t tile) {
                if (st.amax[((long long)b * p.Hq + hk * p.group + e / span) * st.n + first + e % span] >> 8 & 1u) clear_odd_rows<HD>(tile, tile_rows(e));
            };
            const bool any_odd = s_odd != 0;
            auto score = [&](int e) {
                if (!mbar_wait_bounded(bar_qf + 8 * (e & 1), (e >> 1) & 1, p.err)) return false;
                if (any_odd) clean(e, tile_q(e));
                mma_rows<HD>(tmem, sm_k, tile_q(e), kTileQ, id_s);
                mma_commit(bar_s);
                return true;
            };
            auto dprod = [&](int e) {
                if (!mbar_wait_bounded(bar_of + 8 * (e & 1), (e >> 1) & 1, p.err)) return false;
                if (any_odd) clean(e, tile_do(e));
                mma_rows<HD>(t_dp, sm_v, tile_do(e), kTileQ, id_dp);
                mma_commit(bar_dp);
                return true;
            };
            ok = ok && score(0) && dprod(0);
            for (int e = 0; e < n && ok; ++e) {
                if (!(ok = mbar_wait_bounded(bar_p, e & 1, p.err))) break;
                tc_fence_after();
                mma_halves<HD>(t_dv, tmem, tile_do(e), id_g, e > 0);
                mma_commit(bar_oe + 8 * (e & 1));
                if (e + 1 < n && !(ok = score(e + 1))) break;
                if (!(ok = mbar_wait_bounded(bar_ds, e & 1, p.err))) break;
                tc_fence_after();
                mma_halves<HD>(t_dk, t_dp, tile_q(e), id_g, e > 0);
                mma_commit(bar_qe + 8 * (e & 1));
                if (e + 1 < n) ok = dprod(e + 1);
            }
            if (ok) mma_commit(bar_done);
        }
    } else {
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;
        const int half = warp >> 2, in_tile = (warp & 3) * 32 + lane, key = k0 + in_tile;
        ScoreConsts c;
        c.scale2 = fabsf(p.sm_scale) * kLog2e;
        c.cap_in = CAP ? 2.0f * fabsf(p.sm_scale) / p.cap : 0.0f;
        c.cap_out = CAP ? p.cap * kLog2e : 0.0f;
        const float unit = CAP ? c.cap_out : c.scale2;
        const uint32_t s_at = tmem + half * 64 + lanes, d_at = s_at + 128;
        bool ok = true;
        float sigma = 1.0f;
        if (kScaled && n > 0) {
            // the key's row of V: its sum of magnitudes, pieces in an order that keeps lanes apart in the banks
            float norm = 0.0f;
            ok = mbar_wait_bounded(bar_kv, 0, p.err);
#pragma unroll
            for (int x = 0; x < HD / 8; ++x) {
                float v[8];
                unpack16(lds128(sm_v + x / 8 * 128 * 128 + in_tile * 128 + ((x + lane) & 7) * 16), v, (T*)nullptr);
#pragma unroll
                for (int y = 0; y < 8; ++y) norm += fabsf(v[y]);
            }
            sigma = scale_up(norm, s_top, s_delta);
        }
        const float dsigma = sigma / kWeightUp;                    // P^T has its own scale in it
        for (int e = 0; e < n && ok; ++e) {
            const int qt = first + e % span, q0 = qt * kTileQ + half * 64;
            const float slope2 = BIAS ? __ldg(p.slopes + hk * p.group + e / span) * kLog2e : 0.0f;
            const int4 t = st.tiles[(long long)b * st.n + qt];          // written while this kernel was resident: not by the read-only path
            const bool partial = t.z > k0 || t.w < k0 + kTileK;
            const uint32_t neg_lse = tile_rows(e) + half * 64 * 4, neg_delta = neg_lse + kTileQ * 4;
            const uint32_t ranges = tile_rows(e) + L::kRowBytes + half * 64 * 8;
            const float d0 = (float)(q0 + (p.Lk - p.Lq) - key);
            float w[64];
            if (!mbar_wait_bounded(bar_qf + 8 * (e & 1), (e >> 1) & 1, p.err) || !mbar_wait_bounded(bar_s, e & 1, p.err)) { ok = false; break; }
            tc_fence_after();
            tmem_ld32(s_at, w);
            tmem_ld32(s_at + 32, w + 32);
            tmem_wait_ld();
            const bool small = !CAP || scale_scores(w, c);
            auto weights = [&](auto masked, auto is_small) {
#pragma unroll
                for (int x = 0; x < 64; x += 32) {
                    uint32_t o[16];
#pragma unroll
                    for (int y = 0; y < 32; y += 4) {
                        const float4 nl = lds_float4(neg_lse + (x + y) * 4);
#pragma unroll
                        for (int z = 0; z < 4; z += 2) {
                            const int at = x + y + z;
                            const float2 t = capped_pair<CAP, decltype(is_small)::value>(make_float2(w[at], w[at + 1]));
                            float2 slope, v = pair_weights<CAP, BIAS>(t, unit, slope2, add2(make_float2(d0, d0), make_float2((float)at, (float)(at + 1))),
                                                                      z ? make_float2(nl.z, nl.w) : make_float2(nl.x, nl.y), slope);
                            if (decltype(masked)::value) {
                                const uint4 k = lds128(ranges + at * 8);
                                v.x = key >= (int)k.x && key < (int)k.y ? v.x : 0.0f;
                                v.y = key >= (int)k.z && key < (int)k.w ? v.y : 0.0f;
                            }
                            o[(y + z) / 2] = pack2<T>(v.x, v.y);
                            if (CAP) v = mul2(v, slope);
                            w[at] = v.x;
                            w[at + 1] = v.y;
                        }
                    }
                    tmem_st16(s_at + x / 2, o);
                }
            };
            if (!small) weights(Yes{}, No{});
            else if (partial) weights(Yes{}, Yes{});
            else weights(No{}, Yes{});
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_p);
            if (!mbar_wait_bounded(bar_dp, e & 1, p.err)) { ok = false; break; }
            tc_fence_after();
#pragma unroll
            for (int x = 0; x < 64; x += 32) {
                float d[32];
                uint32_t o[16];
                tmem_ld32(d_at + x, d);
                tmem_wait_ld();
#pragma unroll
                for (int y = 0; y < 32; y += 4) {
                    const float4 nd = lds_float4(neg_delta + (x + y) * 4);
#pragma unroll
                    for (int z = 0; z < 4; z += 2) {
                        float2 u = add2(make_float2(d[y + z], d[y + z + 1]), z ? make_float2(nd.z, nd.w) : make_float2(nd.x, nd.y));
                        if (kScaled) u = mul2(u, make_float2(dsigma, dsigma));
                        const float2 ds = mul2(make_float2(w[x + y + z], w[x + y + z + 1]), u);
                        o[(y + z) / 2] = pack2<T>(ds.x, ds.y);
                    }
                }
                tmem_st16(d_at + x / 2, o);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_ds);
        }
        if (ok && n > 0) ok = mbar_wait_bounded(bar_done, 0, p.err);
        if (ok) {
            tc_fence_after();
            const float back = half ? p.sm_scale / sigma : kScaled ? 1.0f / kWeightUp : 1.0f;
            bool fine = true;
            // the first half of the threads has dv, the second dk
            T* out = key < p.Lk ? (half ? row_of<T>(p.dk, p.sdk, b, hk, key) : row_of<T>(p.dv, p.sdv, b, hk, key)) : nullptr;
#pragma unroll
            for (int x = 0; x < HD; x += 32) {
                float o[32];
                if (n > 0) {
                    tmem_ld32(tmem + 256 + half * 128 + x + lanes, o);
                    tmem_wait_ld();
                }
                if (key < p.Lk) {
#pragma unroll
                    for (int y = 0; y < 32; y += 8) {
                        float v[8];
#pragma unroll
                        for (int z = 0; z < 8; ++z) {
                            v[z] = n > 0 ? o[y + z] * back : 0.0f;
                            fine = fine && fabsf(v[z]) <= 3.0e38f;
                        }
                        if (x + y < p.D) stg128(out + x + y, pack16(v, (T*)nullptr));
                    }
                }
            }
            const unsigned bad = __ballot_sync(0xffffffffu, n > 0 && key < p.Lk && !fine);
            if (lane == 0) s_bad[warp] = bad;
        } else if (lane == 0) s_bad[warp] = 0;
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 9) tmem_free(tmem, 512);
    if (any_bad(s_bad)) redo_rows<T, true>(p, s_bad, 0);
}

}  // namespace dsdpa
