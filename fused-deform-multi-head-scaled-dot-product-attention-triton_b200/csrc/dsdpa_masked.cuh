// Masked attention over a sequence: parameters, the score function, and one row's results computed
// by one warp that visits visible keys (or queries) only.
//
// The row functions are the definition written out: any storage type, any head dimension that is a
// multiple of 8, any mask.  The tiled kernels multiply whole tiles, where a masked probability of zero
// meets whatever the masked row holds; a row that comes out non-finite there is computed again here,
// so that NaN or infinity in a place that a query does not see never reaches its results.
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

__device__ __forceinline__ float warp_sum(float x) { return group_sum<32>(x); }

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
// out of: the capped backward over four sequences of 1571 image and text tokens (16 heads, D = 64) takes 245 us with
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
// key tiles have some takes 224 us where the general form alone took 171, 4 x 16 heads of 2048, D = 64.)
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

// Lane l of the warp holds elements 8l .. 8l+7 of a row; lanes behind the row hold zeros and load nothing.
template <typename T>
__device__ __forceinline__ void load_row(const T* row, int D, int lane, float (&f)[8]) {
    if (lane * 8 < D) load8<T>(row + lane * 8, f);
    else {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = 0.0f;
    }
}

// out and lse of one query, by one warp.
template <typename T>
__device__ __noinline__ void exact_row_forward(const MaskedParams& p, int b, int h, int i) {
    const int lane = threadIdx.x & 31, hk = h / p.group;
    const int2 r = key_range(p, b, i);
    const int pos = i + (p.Lk - p.Lq);
    const float slope = p.slopes ? __ldg(p.slopes + h) : 0.0f;
    float q[8], acc[8] = {}, m = kNegInf, l = 0.0f;
    load_row<T>(row_of<T>(p.q, p.sq, b, h, i), p.D, lane, q);
    for (int j = r.x; j < r.y; ++j) {
        float k[8], v[8];
        load_row<T>(row_of<T>(p.k, p.sk, b, hk, j), p.D, lane, k);
        load_row<T>(row_of<T>(p.v, p.sv, b, hk, j), p.D, lane, v);
        float s = soft_cap(p.sm_scale * warp_sum(dot8(q, k)), p.cap);
        if (p.slopes) s -= slope * fabsf((float)(pos - j));
        s *= kLog2e;
        if (s == kNegInf) continue;               // weight zero, whatever v holds
        const float m2 = fmaxf(m, s), c = exp2f(m - m2), w = exp2f(s - m2);
        l = fmaf(l, c, w);
        m = m2;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = fmaf(acc[e], c, w * v[e]);
    }
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;   // a NaN sum stays NaN
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] *= inv;
    if (lane * 8 < p.D) store8<T>(row_of<T>(p.out, p.so, b, h, i) + lane * 8, acc);
    if (lane == 0) p.lse[((long long)b * p.Hq + h) * p.Lq + i] = l != 0.0f ? m + log2f(l) : kNegInf;
}

// p and d(loss)/d(sm_scale q.k) of one (query, key) pair; x = q.k, dp = dout.v
__device__ __forceinline__ void pair_grad(const MaskedParams& p, float x, float dp, float lse, float delta, float slope,
                                          int dist, float& w, float& ds) {
    const float y = soft_cap(p.sm_scale * x, p.cap);
    float s = y;
    if (p.slopes) s -= slope * fabsf((float)dist);
    w = lse == kNegInf ? 0.0f : exp2f(s * kLog2e - lse);
    ds = w == 0.0f ? 0.0f : w * (dp - delta);
    if (p.cap > 0.0f) {
        const float t = y / p.cap;
        ds *= 1.0f - t * t;
    }
}

// dq of one query, by one warp; also the query's delta, which the other functions read.
template <typename T>
__device__ __noinline__ void exact_row_dq(const MaskedParams& p, int b, int h, int i) {
    const int lane = threadIdx.x & 31, hk = h / p.group;
    const int2 r = key_range(p, b, i);
    const int pos = i + (p.Lk - p.Lq);
    const float slope = p.slopes ? __ldg(p.slopes + h) : 0.0f;
    const long long row = ((long long)b * p.Hq + h) * p.Lq + i;
    const float lse = p.lse[row];
    float q[8], o[8], go[8], acc[8] = {};
    load_row<T>(row_of<T>(p.q, p.sq, b, h, i), p.D, lane, q);
    load_row<T>(row_of<T>(p.out_in, p.so, b, h, i), p.D, lane, o);
    load_row<T>(row_of<T>(p.dout, p.sdo, b, h, i), p.D, lane, go);
    const float delta = r.x < r.y ? warp_sum(dot8(o, go)) : 0.0f;
    for (int j = r.x; j < r.y; ++j) {
        float k[8], v[8], w, ds;
        load_row<T>(row_of<T>(p.k, p.sk, b, hk, j), p.D, lane, k);
        load_row<T>(row_of<T>(p.v, p.sv, b, hk, j), p.D, lane, v);
        pair_grad(p, warp_sum(dot8(q, k)), warp_sum(dot8(go, v)), lse, delta, slope, pos - j, w, ds);
        if (w == 0.0f) continue;
        ds *= p.sm_scale;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = fmaf(ds, k[e], acc[e]);
    }
    if (lane * 8 < p.D) store8<T>(row_of<T>(p.dq, p.sdq, b, h, i) + lane * 8, acc);
    if (lane == 0) p.delta[row] = delta;
}

// dk and dv of one key, summed over the query heads that share it, by one warp.
template <typename T>
__device__ __noinline__ void exact_row_dkdv(const MaskedParams& p, int b, int hk, int j) {
    const int lane = threadIdx.x & 31;
    float k[8], v[8], ak[8] = {}, av[8] = {};
    load_row<T>(row_of<T>(p.k, p.sk, b, hk, j), p.D, lane, k);
    load_row<T>(row_of<T>(p.v, p.sv, b, hk, j), p.D, lane, v);
    const int first = p.causal ? max(0, j - (p.Lk - p.Lq)) : 0;
    for (int g = 0; g < p.group; ++g) {
        const int h = hk * p.group + g;
        const float slope = p.slopes ? __ldg(p.slopes + h) : 0.0f;
        for (int i = first; i < p.Lq; ++i) {
            const int2 r = key_range(p, b, i);
            if (j < r.x || j >= r.y) continue;
            const long long row = ((long long)b * p.Hq + h) * p.Lq + i;
            float q[8], go[8], w, ds;
            load_row<T>(row_of<T>(p.q, p.sq, b, h, i), p.D, lane, q);
            load_row<T>(row_of<T>(p.dout, p.sdo, b, h, i), p.D, lane, go);
            pair_grad(p, warp_sum(dot8(q, k)), warp_sum(dot8(go, v)), p.lse[row], p.delta[row], slope,
                      i + (p.Lk - p.Lq) - j, w, ds);
            if (w == 0.0f) continue;
            ds *= p.sm_scale;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                ak[e] = fmaf(ds, q[e], ak[e]);
                av[e] = fmaf(w, go[e], av[e]);
            }
        }
    }
    if (lane * 8 < p.D) {
        store8<T>(row_of<T>(p.dk, p.sdk, b, hk, j) + lane * 8, ak);
        store8<T>(row_of<T>(p.dv, p.sdv, b, hk, j) + lane * 8, av);
    }
}

}  // namespace dsdpa
