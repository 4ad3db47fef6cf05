// Masked attention over a sequence: parameters, the score function, and one row's results computed
// by one warp that visits visible keys (or queries) only.
//
// The row functions are the definition written out: any storage type, any head dimension that is a
// multiple of 8, any mask.  The tiled kernels multiply whole tiles, where a masked probability of zero
// meets whatever the masked row holds; a row that comes out non-finite there is computed again here,
// so that NaN or infinity in a place that a query does not see never reaches its results.  A row that
// is non-finite by itself (its lse, or the gradient that comes in) is not: nothing hidden made it so.
#pragma once

#include "dsdpa_common.cuh"

namespace dsdpa {

struct MaskedParams {
    const void *q, *k, *v, *out_in, *dout;
    void *out, *dq, *dk, *dv;
    float* lse;          // forward: written; backward: read
    float* delta;        // backward: sum_d out dout, [B, Hq, Lq]
    const int2* visible; // or null
    const float* slopes; // or null
    int B, Hq, Hkv, group, Lq, Lk, D;
    int causal;
    float sm_scale, cap; // cap <= 0: none
    long long sq[3], sk[3], sv[3], so[3], sdo[3], sdq[3], sdk[3], sdv[3];
    long long s_visible; // in int2
    int* err;
};

constexpr float kNegInf = -__builtin_huge_valf();

// Keys [x, y) that query i of batch element b sees; x >= y: none.
__device__ __forceinline__ int2 key_range(const MaskedParams& p, int b, int i) {
    int lo = 0, hi = p.Lk;
    if (p.visible) {
        const int2 r = __ldg(p.visible + b * p.s_visible + i);
        lo = max(lo, r.x);
        hi = min(hi, r.y);
    }
    if (p.causal) hi = min(hi, i + (p.Lk - p.Lq) + 1);
    return make_int2(lo, hi);
}

// cap tanh(x / cap): CUDA's tanhf, whose error is a few units in the last place of the result.
__device__ __forceinline__ float soft_cap(float x, float cap) { return cap > 0.0f ? cap * tanhf(x / cap) : x; }

// Eight consecutive elements of a row, as fp32.
template <typename T> __device__ __forceinline__ void load8(const T* p, float (&f)[8]) {
    unpack16(ldg128_nc(p), f, (T*)nullptr);
}
template <> __device__ __forceinline__ void load8<float>(const float* p, float (&f)[8]) {
    float a[4], b[4];
    unpack16(ldg128_nc(p), a, (float*)nullptr);
    unpack16(ldg128_nc(p + 4), b, (float*)nullptr);
#pragma unroll
    for (int e = 0; e < 4; ++e) { f[e] = a[e]; f[4 + e] = b[e]; }
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
    stg128(p, pack16(f, (T*)nullptr));
}
template <> __device__ __forceinline__ void store8<float>(float* p, const float (&f)[8]) {
    const float a[4] = { f[0], f[1], f[2], f[3] }, b[4] = { f[4], f[5], f[6], f[7] };
    stg128(p, pack16(a, (float*)nullptr));
    stg128(p + 4, pack16(b, (float*)nullptr));
}
template <typename T> __device__ __forceinline__ void store4(T* p, const float (&f)[4]) {
    const float g[8] = { f[0], f[1], f[2], f[3], 0.0f, 0.0f, 0.0f, 0.0f };
    const uint4 r = pack16(g, (T*)nullptr);
    *reinterpret_cast<uint2*>(p) = make_uint2(r.x, r.y);
}
template <> __device__ __forceinline__ void store4<float>(float* p, const float (&f)[4]) { stg128(p, pack16(f, (float*)nullptr)); }
template <typename T> __device__ __forceinline__ void store2(T* p, float a, float b) {
    const float g[8] = { a, b, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f };
    *reinterpret_cast<uint32_t*>(p) = pack16(g, (T*)nullptr).x;
}
template <> __device__ __forceinline__ void store2<float>(float* p, float a, float b) { *reinterpret_cast<float2*>(p) = make_float2(a, b); }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
// Two packed 16-bit elements as fp32.
template <typename T> __device__ __forceinline__ float2 to_float2(uint32_t u) {
    float f[8];
    unpack16(make_uint4(u, 0, 0, 0), f, (T*)nullptr);
    return make_float2(f[0], f[1]);
}
__device__ __forceinline__ float dot8(const float (&a)[8], const float (&b)[8]) {
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(a[e], b[e], s);
    return s;
}

// Two fp32 lanes at a time.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
        "fma.rn.f32x2 z, x, y, z;\n\tmov.b64 {%0, %1}, z;\n\t}" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// tanh(a / 2), the cap's argument being a = 2 x / cap.  For |a| < 2 (scores below the cap) an odd polynomial, fitted to
// the least largest relative error (5e-8; evaluated in fp32 1.5e-7): ten fma-pipe operations for two values where
// the general form, 1 - 2 / (1 + e^a), takes four of the special-function unit, which is what these kernels run
// out of: the capped backward over four sequences of 1571 image and text tokens (16 heads, D = 64) took 245 us with
// that form alone, 208 us with this one.
constexpr int kTanhTerms = 7;
__device__ __forceinline__ float tanh_term(int i) {
    constexpr float k[kTanhTerms] = { 4.999999702e-01f, -4.166604951e-02f, 4.164126236e-03f, -4.176330403e-04f, 3.962886694e-05f, -3.028993660e-06f, 1.270779535e-07f };
    return k[i];
}
__device__ __forceinline__ float2 half_tanh_small(float2 a) {
    const float2 u = mul2(a, a);
    float2 r = make_float2(tanh_term(kTanhTerms - 1), tanh_term(kTanhTerms - 1));
#pragma unroll
    for (int i = kTanhTerms - 2; i >= 0; --i) r = fma2(r, u, make_float2(tanh_term(i), tanh_term(i)));
    return mul2(r, a);
}
__device__ __forceinline__ float half_tanh(float a) { return fmaf(-2.0f, rcp_approx(1.0f + fast_exp2(a * kLog2e)), 1.0f); }
__device__ __forceinline__ bool is_small(float a) { return fabsf(a) < 2.0f; }
// Any two values, each by the form that its own size asks for: what a score becomes does not depend on the others that a
// warp happens to hold, hidden ones among them, and the general form, which is good to a step of 1, is not taken where
// that is much of the result.  (Both forms for every value of a warp that has one above the cap: a forward all of whose
// key tiles have some takes 220 us where the general form alone took 171, 4 x 16 heads of 2048, D = 64.)
__device__ __forceinline__ float2 half_tanh_any(float2 a) {
    const float2 t = half_tanh_small(a);
    return make_float2(is_small(a.x) ? t.x : half_tanh(a.x), is_small(a.y) ? t.y : half_tanh(a.y));
}
// Whether all of a warp's values are small: their top exponent bit says so (NaN is not).
template <int N>
__device__ __forceinline__ bool all_small(const float (&a)[N]) {
    unsigned any = 0;
#pragma unroll
    for (int i = 0; i < N; i += 2) any |= __float_as_uint(a[i]) | __float_as_uint(a[i + 1]);
    return !__any_sync(0xffffffffu, any & 0x40000000u);
}

template <typename T>
__device__ __forceinline__ const T* row_of(const void* base, const long long (&st)[3], int b, int h, long long i) {
    return (const T*)base + b * st[0] + h * st[1] + i * st[2];
}
template <typename T>
__device__ __forceinline__ T* row_of(void* base, const long long (&st)[3], int b, int h, long long i) {
    return (T*)base + b * st[0] + h * st[1] + i * st[2];
}

// ---- one row again, from what it sees alone ----------------------------------------------------------------------
// By one warp.  As many lanes as a row has pieces of eight elements (rounded up to a power of two) have a key's, or a query's,
// row together: the warp has several rows at once, loads them whole lines at a time and without a condition, and takes
// what it has loaded both for the products and for the sums of rows.  The lanes of every row place have sums of their
// own, joined at the end.  Gradients with one infinite row, 16 heads on 4 of 4096 x 4096, D = 128, fp16: backward 1.6 ms, 0.36 ms
// without (a key at a time by the whole warp, every row that came out non-finite: about 1000); all of them infinite 2.5 ms;
// a NaN in one value in the middle: forward 11 ms, 0.09 without.
struct RowLanes {
    int n, at, place, places;        // lanes of a row, this one's number among them, the row's place, places of the warp
    __device__ __forceinline__ RowLanes(int D, int lane) : n(1) {
        while (n * 8 < D) n *= 2;
        at = lane & (n - 1);
        place = lane / n;
        places = 32 / n;
    }
    // over the lanes of a row; all lanes call (exchanges without a condition: those of several rows can then overlap)
    __device__ __forceinline__ float row_sum(float x) const {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float y = __shfl_xor_sync(0xffffffffu, x, o);
            x = o < n ? x + y : x;
        }
        return x;
    }
    // over the places
    __device__ __forceinline__ float place_sum(float x) const {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            if (o >= n) x += __shfl_xor_sync(0xffffffffu, x, o);
        return x;
    }
    __device__ __forceinline__ float place_max(float x) const {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            if (o >= n) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
        return x;
    }
    // Whether every element of a row of sums is NaN at some place, and with that in the end.
    __device__ __forceinline__ bool all_nan(const float (&acc)[8], int D) const {
        bool nan = true;
#pragma unroll
        for (int e = 0; e < 8; ++e) nan = nan && acc[e] != acc[e];
        unsigned b = __ballot_sync(0xffffffffu, nan);
        for (int o = n; o < 32; o *= 2) b |= b >> o;
        const unsigned need = D >= 256 ? ~0u : (1u << (D / 8)) - 1;
        return (b & need) == need;
    }
};
// A running softmax over keys that come at several places.
struct RowSoftmax {
    float m = kNegInf, l = 0.0f;
    // the next STEPS scores of this place, in base 2, to their weights; returns what the sums so far have to be multiplied by
    template <int STEPS>
    __device__ __forceinline__ float next(const float (&s)[STEPS], float (&w)[STEPS]) {
        float m2 = m;
#pragma unroll
        for (int e = 0; e < STEPS; ++e) m2 = fmaxf(m2, s[e]);
        const float c = m == kNegInf ? 0.0f : exp2f(m - m2);
        m = m2;
        l *= c;
#pragma unroll
        for (int e = 0; e < STEPS; ++e) {
            w[e] = s[e] == kNegInf ? 0.0f : exp2f(s[e] - m2);
            l += w[e];
        }
        return c;
    }
    // all places to one reference point: their sums of weights, and of rows, added up
    __device__ __forceinline__ void join(const RowLanes& r, float (&acc)[8]) {
        const float top = r.place_max(m), f = m == kNegInf ? 0.0f : exp2f(m - top);
        l = r.place_sum(l == 0.0f ? 0.0f : l * f);
        m = top;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = r.place_sum(acc[e] * f);
    }
};
// A lane's piece of a row, as it lies in memory.  Loaded without a condition, from a row that exists in any case, and looked at
// later: a load behind a condition is waited for at once.
template <typename T>
struct RowPiece {
    uint4 u[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* row, int at, int D) {
        const T* from = row + (at * 8 < D ? at * 8 : 0);
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) u[i] = ldg128_nc(reinterpret_cast<const uint4*>(from) + i);
    }
    __device__ __forceinline__ void get(int at, int D, float (&f)[8]) const {
        const bool there = at * 8 < D;
        if constexpr (sizeof(T) == 4) {
            float a[4], b[4];
            unpack16(u[0], a, (T*)nullptr);
            unpack16(u[1], b, (T*)nullptr);
#pragma unroll
            for (int e = 0; e < 4; ++e) { f[e] = there ? a[e] : 0.0f; f[4 + e] = there ? b[e] : 0.0f; }
        } else {
            unpack16(u[0], f, (T*)nullptr);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = there ? f[e] : 0.0f;
        }
    }
};
template <typename T>
__device__ __forceinline__ void load_piece(const T* row, int at, int D, float (&f)[8]) {
    RowPiece<T> x;
    x.load(row, at, D);
    x.get(at, D, f);
}
__device__ __forceinline__ void add_piece(float (&acc)[8], float w, const float (&f)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = fmaf(w, f[e], acc[e]);
}

// out and lse of one query.  A row of NaN is left as soon as it is one, with the lse that the caller found: the tiled kernels' is
// right, since a mask takes hidden scores out before they are summed.
template <typename T>
__device__ __noinline__ void exact_row_forward(const MaskedParams& p, int b, int h, int i) {
    constexpr int kSteps = 2;
    const int lane = threadIdx.x & 31, hk = h / p.group, D = p.D;
    const RowLanes rl(D, lane);
    const int2 r = key_range(p, b, i);
    const int pos = i + (p.Lk - p.Lq);
    const float slope = p.slopes ? __ldg(p.slopes + h) : 0.0f, sm_scale = p.sm_scale, cap = p.cap;
    const long long sk = p.sk[2], sv = p.sv[2];
    const T *k = row_of<T>(p.k, p.sk, b, hk, 0), *v = row_of<T>(p.v, p.sv, b, hk, 0);
    float q[8], acc[8] = {};
    load_piece<T>(row_of<T>(p.q, p.sq, b, h, i), rl.at, D, q);
    RowSoftmax sum;
    bool nan = false;
    for (int j0 = r.x; j0 < r.y && !nan; j0 += kSteps * rl.places) {
        RowPiece<T> kr[kSteps], vr[kSteps];
        float s[kSteps], w[kSteps], f[8];
#pragma unroll
        for (int e = 0; e < kSteps; ++e) {
            const int j = min(j0 + e * rl.places + rl.place, r.y - 1);
            kr[e].load(k + j * sk, rl.at, D);
            vr[e].load(v + j * sv, rl.at, D);
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
            if (p.slopes) s[e] -= slope * fabsf((float)(pos - j));
            s[e] = j < r.y ? s[e] * kLog2e : kNegInf;
        }
        const float c = sum.next(s, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] *= c;
#pragma unroll
        for (int e = 0; e < kSteps; ++e) {
            vr[e].get(rl.at, D, f);
            if (s[e] != kNegInf) add_piece(acc, w[e], f);          // weight zero, whatever the value's row holds
        }
        nan = rl.all_nan(acc, D);
    }
    sum.join(rl, acc);
    const float inv = sum.l != 0.0f ? 1.0f / sum.l : 0.0f;   // a NaN sum stays NaN
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] *= inv;
    if (rl.place == 0 && rl.at * 8 < D) store8<T>(row_of<T>(p.out, p.so, b, h, i) + rl.at * 8, acc);
    if (lane == 0 && !nan) p.lse[((long long)b * p.Hq + h) * p.Lq + i] = sum.l != 0.0f ? sum.m + log2f(sum.l) : kNegInf;
}

// Whether a query's own part of the gradients is not finite: its row of dq is then what it is, and so is all that it sees.
__device__ __forceinline__ bool spoilt(float lse, float delta) {
    return lse != kNegInf && lse != -kNegInf && !(lse == lse && fabsf(delta) < -kNegInf);
}

// What a pair's gradient needs of the call, read once (the parameters of a function that is not inlined lie in memory).
struct PairForm {
    float sm_scale, cap;
    bool biased;
    __device__ __forceinline__ explicit PairForm(const MaskedParams& p) : sm_scale(p.sm_scale), cap(p.cap), biased(p.slopes != nullptr) {}
    // p and d(loss)/d(sm_scale q.k) of one (query, key) pair; x = q.k, dp = dout.v
    __device__ __forceinline__ void grad(float x, float dp, float lse, float delta, float slope, int dist, float& w, float& ds) const {
        const float y = soft_cap(sm_scale * x, cap);
        float s = y;
        if (biased) s -= slope * fabsf((float)dist);
        w = lse == kNegInf ? 0.0f : exp2f(s * kLog2e - lse);
        ds = w == 0.0f ? 0.0f : w * (dp - delta);
        if (cap > 0.0f) {
            const float t = y / cap;
            ds *= 1.0f - t * t;
        }
    }
};

// dq of one query.
template <typename T>
__device__ __noinline__ void exact_row_dq(const MaskedParams& p, int b, int h, int i) {
    constexpr int kSteps = 2;
    const int lane = threadIdx.x & 31, hk = h / p.group, D = p.D;
    const RowLanes rl(D, lane);
    int2 r = key_range(p, b, i);
    const int pos = i + (p.Lk - p.Lq);
    const float slope = p.slopes ? __ldg(p.slopes + h) : 0.0f;
    const long long row = ((long long)b * p.Hq + h) * p.Lq + i, sk = p.sk[2], sv = p.sv[2];
    const T *k = row_of<T>(p.k, p.sk, b, hk, 0), *v = row_of<T>(p.v, p.sv, b, hk, 0);
    const float lse = p.lse[row], delta = p.delta[row];
    const PairForm form(p);
    float q[8], go[8], acc[8] = {};
    load_piece<T>(row_of<T>(p.q, p.sq, b, h, i), rl.at, D, q);
    load_piece<T>(row_of<T>(p.dout, p.sdo, b, h, i), rl.at, D, go);
    if (lse == kNegInf) r.y = r.x;
    for (int j0 = r.x; j0 < r.y && !rl.all_nan(acc, D); j0 += kSteps * rl.places) {
        RowPiece<T> kr[kSteps], vr[kSteps];
#pragma unroll
        for (int e = 0; e < kSteps; ++e) {
            const int j = min(j0 + e * rl.places + rl.place, r.y - 1);
            kr[e].load(k + j * sk, rl.at, D);
            vr[e].load(v + j * sv, rl.at, D);
        }
        float x[kSteps], dp[kSteps], f[8];
#pragma unroll
        for (int e = 0; e < kSteps; ++e) {
            kr[e].get(rl.at, D, f);
            x[e] = rl.row_sum(dot8(q, f));
            vr[e].get(rl.at, D, f);
            dp[e] = rl.row_sum(dot8(go, f));
        }
#pragma unroll
        for (int e = 0; e < kSteps; ++e) {
            const int j = j0 + e * rl.places + rl.place;
            float w, ds;
            form.grad(x[e], dp[e], lse, delta, slope, pos - j, w, ds);
            kr[e].get(rl.at, D, f);
            if (j < r.y && w != 0.0f) add_piece(acc, ds * form.sm_scale, f);
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = rl.place_sum(acc[e]);
    if (rl.place == 0 && rl.at * 8 < D) store8<T>(row_of<T>(p.dq, p.sdq, b, h, i) + rl.at * 8, acc);
}

// dk and dv of one key, summed over the query heads that share it.  Where a query that sees the key is spoilt they stay as the
// caller found them: not finite.
template <typename T>
__device__ __noinline__ void exact_row_dkdv(const MaskedParams& p, int b, int hk, int j) {
    constexpr int kSteps = 2;
    const int lane = threadIdx.x & 31, D = p.D;
    const RowLanes rl(D, lane);
    const PairForm form(p);
    const int Lq = p.Lq, Lk = p.Lk, group = p.group, first = p.causal ? max(0, j - (Lk - Lq)) : 0;
    const bool causal = p.causal != 0;
    const int2* visible = p.visible ? p.visible + b * p.s_visible : nullptr;
    const float *lses = p.lse + ((long long)b * p.Hq + hk * group) * Lq, *deltas = p.delta + ((long long)b * p.Hq + hk * group) * Lq;
    auto sees = [&](int i) {                         // i < Lq
        const int2 r = visible ? __ldg(visible + i) : make_int2(0, Lk);
        return j >= r.x && j < r.y && (!causal || j <= i + (Lk - Lq));
    };
    // 32 queries at a time; from the first to the last that see the key
    int lo = Lq, hi = 0;
    for (int i0 = first; i0 < Lq; i0 += 32) {
        const int i = min(i0 + lane, Lq - 1);
        const bool on = i0 + lane < Lq && sees(i);
        const unsigned any = __ballot_sync(0xffffffffu, on);
        if (!any) continue;
        lo = min(lo, i0 + __ffs(any) - 1);
        hi = i0 + 32 - __clz(any);
        bool bad = false;
#pragma unroll 4
        for (int g = 0; g < group; ++g) bad |= spoilt(lses[(long long)g * Lq + i], deltas[(long long)g * Lq + i]);
        if (__any_sync(0xffffffffu, on && bad)) return;
    }
    float k[8], v[8], ak[8] = {}, av[8] = {};
    load_piece<T>(row_of<T>(p.k, p.sk, b, hk, j), rl.at, D, k);
    load_piece<T>(row_of<T>(p.v, p.sv, b, hk, j), rl.at, D, v);
    const long long sq = p.sq[2], sdo = p.sdo[2];
    bool nan = false;
    for (int g = 0; g < group && !nan; ++g) {
        const int h = hk * group + g;
        const float slope = form.biased ? __ldg(p.slopes + h) : 0.0f;
        const T *q = row_of<T>(p.q, p.sq, b, h, 0), *go = row_of<T>(p.dout, p.sdo, b, h, 0);
        const float *lse_h = lses + (long long)g * Lq, *delta_h = deltas + (long long)g * Lq;
        for (int i0 = lo; i0 < hi && !nan; i0 += kSteps * rl.places) {
            RowPiece<T> qr[kSteps], gr[kSteps];
            float lse[kSteps], delta[kSteps];
            bool on[kSteps];
#pragma unroll
            for (int e = 0; e < kSteps; ++e) {
                const int i = min(i0 + e * rl.places + rl.place, hi - 1);
                on[e] = sees(i);
                qr[e].load(q + i * sq, rl.at, D);
                gr[e].load(go + i * sdo, rl.at, D);
                lse[e] = lse_h[i];
                delta[e] = delta_h[i];
            }
            float x[kSteps], dp[kSteps], f[8];
#pragma unroll
            for (int e = 0; e < kSteps; ++e) {
                qr[e].get(rl.at, D, f);
                x[e] = rl.row_sum(dot8(f, k));
                gr[e].get(rl.at, D, f);
                dp[e] = rl.row_sum(dot8(f, v));
            }
#pragma unroll
            for (int e = 0; e < kSteps; ++e) {
                const int i = i0 + e * rl.places + rl.place;
                float w, ds;
                form.grad(x[e], dp[e], lse[e], delta[e], slope, i + (Lk - Lq) - j, w, ds);
                if (i < hi && on[e] && w != 0.0f) {
                    qr[e].get(rl.at, D, f);
                    add_piece(ak, ds * form.sm_scale, f);
                    gr[e].get(rl.at, D, f);
                    add_piece(av, w, f);
                }
            }
            nan = rl.all_nan(ak, D) && rl.all_nan(av, D);
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) { ak[e] = rl.place_sum(ak[e]); av[e] = rl.place_sum(av[e]); }
    if (rl.place == 0 && rl.at * 8 < D) {
        store8<T>(row_of<T>(p.dk, p.sdk, b, hk, j) + rl.at * 8, ak);
        store8<T>(row_of<T>(p.dv, p.sdv, b, hk, j) + rl.at * 8, av);
    }
}

}  // namespace dsdpa
