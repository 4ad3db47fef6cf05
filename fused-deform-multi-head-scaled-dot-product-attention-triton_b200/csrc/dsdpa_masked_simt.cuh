// Masked attention in fp32 arithmetic: fp32 storage, and 16-bit storage with more than 128 elements a row.
//
// Tiles in shared memory as fp32, products by packed fma on register tiles of 4 x 4 (scores) and 4 x HD/16
// (sums of rows).  A block has 64 queries (32 for 256 elements) and goes over keys 64 at a time, or has 64
// keys and goes over queries.  The 16 threads that share a row exchange its maximum and sum by shuffles.
// Bound by the fma pipe: a thread issues 32 packed fmas for eight 16-byte loads.  Measured, 8 heads of 2816 tokens, an image
// prefix of 700, capped, D = 32: forward 206 us, backward 655 us (0.28 and 0.22 of the pipe's rate for the products
// alone; at D = 32 the cap, exp2 and masks are as much again).
#pragma once

#include "dsdpa_masked.cuh"

namespace dsdpa {

constexpr int kSimtThreads = 256, kSimtKeys = 64;
template <int HD, int ROWS = HD == 256 ? 2 : 4> struct SimtShape {
    static constexpr int RM = ROWS;                    // rows of a thread
    static constexpr int BM = 16 * RM;                 // queries of a tile
    static constexpr int S = HD + 4;                   // floats of a row: rows start 16 bytes further in the banks
    static constexpr int W = kSimtKeys + 4;            // floats of a row of weights
    static constexpr int NJ = HD >= 64 ? HD / 64 : 1;  // pieces of a row of sums that a thread has
    static constexpr int CW = HD >= 64 ? 4 : HD / 16;  // floats of a piece
    static constexpr int kSmemFwd = (BM * S + 2 * kSimtKeys * S + BM * W) * 4;
    static constexpr int kBlocks = HD <= 64 ? 2 : 1;   // of an SM, by shared memory and by registers
    static constexpr int kSmemBwd = (2 * BM * S + 2 * kSimtKeys * S + BM * W) * 4;
};

__device__ __forceinline__ void add_fma2(float2& d, float2 a, float2 b) { d = fma2(a, b, d); }

// Rows [row0, row0 + N) of one head into shared memory as fp32; rows and elements that do not exist are zero.
template <typename T, int HD, int N>
__device__ __forceinline__ void simt_load(float* dst, const T* base, long long stride, int row0, int rows, int D) {
    constexpr int S = SimtShape<HD>::S, kPer = HD / 4;
    for (int e = threadIdx.x; e < N * kPer; e += kSimtThreads) {
        const int r = e / kPer, d = e % kPer * 4;
        const bool there = row0 + r < rows && d < D;
        const T* src = there ? base + (row0 + r) * stride + d : base;
        if constexpr (sizeof(T) == 4) {
            asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" :: "r"(smem_addr(dst + r * S + d)), "l"(src), "r"(there ? 16 : 0) : "memory");
        } else {
            float2 a = make_float2(0.0f, 0.0f), b = a;
            if (there) {
                const uint2 u = __ldg(reinterpret_cast<const uint2*>(src));
                a = to_float2<T>(u.x);
                b = to_float2<T>(u.y);
            }
            *reinterpret_cast<float4*>(dst + r * S + d) = make_float4(a.x, a.y, b.x, b.y);
        }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
}
__device__ __forceinline__ void simt_wait() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

// s[r][c] = row (ty RM + r) of a . row (tx + 16 c) of b
template <int HD, int RM>
__device__ __forceinline__ void simt_dot(const float* a, const float* b, float (&s)[RM][4]) {
    using L = SimtShape<HD, RM>;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float2 acc[L::RM][4] = {};
    const float* pa = a + ty * L::RM * L::S;
    const float* pb = b + tx * L::S;
#pragma unroll 4
    for (int d = 0; d < HD; d += 4) {
        float4 x[L::RM], y[4];
#pragma unroll
        for (int r = 0; r < L::RM; ++r) x[r] = *reinterpret_cast<const float4*>(pa + r * L::S + d);
#pragma unroll
        for (int c = 0; c < 4; ++c) y[c] = *reinterpret_cast<const float4*>(pb + c * 16 * L::S + d);
#pragma unroll
        for (int r = 0; r < L::RM; ++r)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                add_fma2(acc[r][c], make_float2(x[r].x, x[r].y), make_float2(y[c].x, y[c].y));
                add_fma2(acc[r][c], make_float2(x[r].z, x[r].w), make_float2(y[c].z, y[c].w));
            }
    }
#pragma unroll
    for (int r = 0; r < L::RM; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[r][c] = acc[r][c].x + acc[r][c].y;
}

// A thread's piece j of a row: CW floats from column tx CW + 64 j.
template <int HD>
__device__ __forceinline__ void simt_piece(const float* row, int j, float2 (&v)[2]) {
    using L = SimtShape<HD>;
    const int tx = threadIdx.x & 15;
    if constexpr (L::CW == 4) {
        const float4 f = *reinterpret_cast<const float4*>(row + tx * 4 + 64 * j);
        v[0] = make_float2(f.x, f.y);
        v[1] = make_float2(f.z, f.w);
    } else {
        v[0] = *reinterpret_cast<const float2*>(row + tx * 2);
    }
}

// acc[r] += sum_k w[ty RM + r][k] b[k]: w has rows of queries, b keys
template <int HD, int RM>
__device__ __forceinline__ void simt_rows(const float* w, const float* b, float2 (&acc)[RM][SimtShape<HD>::NJ][2]) {
    using L = SimtShape<HD, RM>;
    const int ty = threadIdx.x >> 4;
#pragma unroll 2
    for (int k = 0; k < kSimtKeys; k += 4) {
        float4 x[L::RM];
#pragma unroll
        for (int r = 0; r < L::RM; ++r) x[r] = *reinterpret_cast<const float4*>(w + (ty * L::RM + r) * L::W + k);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int j = 0; j < L::NJ; ++j) {
                float2 v[2];
                simt_piece<HD>(b + (k + e) * L::S, j, v);
#pragma unroll
                for (int r = 0; r < L::RM; ++r) {
                    const float f = e == 0 ? x[r].x : e == 1 ? x[r].y : e == 2 ? x[r].z : x[r].w;
#pragma unroll
                    for (int q = 0; q < L::CW / 2; ++q) add_fma2(acc[r][j][q], make_float2(f, f), v[q]);
                }
            }
    }
}
// acc[c] += sum_q w[q][4 ty + c] b[q]: the keys' sums over the queries of a tile
template <int HD>
__device__ __forceinline__ void simt_columns(const float* w, const float* b, float2 (&acc)[4][SimtShape<HD>::NJ][2]) {
    using L = SimtShape<HD>;
    const int ty = threadIdx.x >> 4;
#pragma unroll 4
    for (int q = 0; q < L::BM; ++q) {
        const float4 x = *reinterpret_cast<const float4*>(w + q * L::W + ty * 4);
#pragma unroll
        for (int j = 0; j < L::NJ; ++j) {
            float2 v[2];
            simt_piece<HD>(b + q * L::S, j, v);
#pragma unroll
            for (int z = 0; z < L::CW / 2; ++z) {
                add_fma2(acc[0][j][z], make_float2(x.x, x.x), v[z]);
                add_fma2(acc[1][j][z], make_float2(x.y, x.y), v[z]);
                add_fma2(acc[2][j][z], make_float2(x.z, x.z), v[z]);
                add_fma2(acc[3][j][z], make_float2(x.w, x.w), v[z]);
            }
        }
    }
}
// One row of sums, times f, to storage; returns a NaN where one of them is not finite.
template <typename T, int HD>
__device__ __forceinline__ float simt_store(T* row, const float2 (&acc)[SimtShape<HD>::NJ][2], float f, int D) {
    using L = SimtShape<HD>;
    const int tx = threadIdx.x & 15;
    float nan = 0.0f;
#pragma unroll
    for (int j = 0; j < L::NJ; ++j) {
        const int d = tx * L::CW + 64 * j;
        float v[4];
#pragma unroll
        for (int z = 0; z < L::CW / 2; ++z) {
            v[2 * z] = acc[j][z].x * f;
            v[2 * z + 1] = acc[j][z].y * f;
        }
#pragma unroll
        for (int e = 0; e < L::CW; ++e) nan = fmaf(v[e], 0.0f, nan);
        if (row && d < D) {
            if constexpr (L::CW == 4) store4<T>(row + d, v);
            else store2<T>(row + d, v[0], v[1]);
        }
    }
    return nan;
}
// Products q.k to scores in base 2 without bias: s times the result.  With a cap s becomes tanh(x / cap), as a polynomial
// where that is enough, by CUDA's tanhf where not (fp32 storage shows more than the short form's error): each score by its
// own size, whatever the others are.
template <int RM>
__device__ __forceinline__ float simt_cap(float (&s)[RM][4], float sm_scale, float cap) {
    if (!(cap > 0.0f)) return sm_scale * kLog2e;
    const float in = 2.0f * sm_scale / cap;
    float a[4 * RM];
#pragma unroll
    for (int i = 0; i < 4 * RM; ++i) a[i] = s[i / 4][i % 4] * in;
    if (all_small(a)) {
#pragma unroll
        for (int i = 0; i < 4 * RM; i += 2) {
            const float2 t = half_tanh_small(make_float2(a[i], a[i + 1]));
            s[i / 4][i % 4] = t.x;
            s[i / 4][i % 4 + 1] = t.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4 * RM; i += 2) {
            const float2 t = half_tanh_small(make_float2(a[i], a[i + 1]));
            s[i / 4][i % 4] = is_small(a[i]) ? t.x : tanhf(0.5f * a[i]);
            s[i / 4][i % 4 + 1] = is_small(a[i + 1]) ? t.y : tanhf(0.5f * a[i + 1]);
        }
    }
    return cap * kLog2e;
}
// What simt_cap left to a weight, and dp to d(loss) / d(sm_scale q.k).
__device__ __forceinline__ void simt_grad(float t, float unit, bool capped, float bias, float dp, float lse, float delta, float& w, float& ds) {
    w = fast_exp2(fmaf(t, unit, -bias) - lse);
    ds = w * (dp - delta);
    if (capped) ds *= fmaf(-t, t, 1.0f);
}
__device__ __forceinline__ float half_warp_max(float x) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
}
__device__ __forceinline__ float half_warp_sum(float x) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

// Rows that something non-finite reached: bit r of `bad` for the thread's row ty RM + r (all 16 threads of a row
// have the same); f(row) by the whole warp.
template <int RM, typename F>
__device__ __forceinline__ void simt_redo(unsigned bad, F f) {
    const int ty = threadIdx.x >> 4, half = ty & 1;
    __syncwarp();
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        unsigned rows = __shfl_sync(0xffffffffu, bad, side * 16);
        while (rows) {
            const int r = __ffs(rows) - 1;
            rows &= rows - 1;
            f((ty - half + side) * RM + r);
        }
    }
}

template <typename T, int HD>
__global__ void __launch_bounds__(kSimtThreads, SimtShape<HD>::kBlocks)
masked_simt_fwd_kernel(const __grid_constant__ MaskedParams p, int qtiles) {
    using L = SimtShape<HD>;
    extern __shared__ float4 simt_smem[];
    float *sq = reinterpret_cast<float*>(simt_smem), *sk = sq + L::BM * L::S, *sv = sk + kSimtKeys * L::S, *sw = sv + kSimtKeys * L::S;
    __shared__ int s_lo, s_hi;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int bh = blockIdx.x % (p.B * p.Hq), b = bh / p.Hq, h = bh % p.Hq, hk = h / p.group;
    const int q0 = (qtiles - 1 - (int)(blockIdx.x / (p.B * p.Hq))) * L::BM;
    if (tid == 0) { s_lo = 0x7fffffff; s_hi = 0; }
    __syncthreads();
    int2 rg[L::RM];
    int lo = 0x7fffffff, hi = 0;
#pragma unroll
    for (int r = 0; r < L::RM; ++r) {
        const int i = q0 + ty * L::RM + r;
        rg[r] = i < p.Lq ? key_range(p, b, i) : make_int2(0, 0);
        if (rg[r].x >= rg[r].y) rg[r] = make_int2(0, 0);
        else { lo = min(lo, rg[r].x); hi = max(hi, rg[r].y); }
    }
    atomicMin(&s_lo, __reduce_min_sync(0xffffffffu, lo));
    atomicMax(&s_hi, __reduce_max_sync(0xffffffffu, hi));
    __syncthreads();
    const int first = s_hi > 0 ? s_lo / kSimtKeys : 0, end = s_hi > 0 ? (s_hi + kSimtKeys - 1) / kSimtKeys : 0;
    const T *kb = row_of<T>(p.k, p.sk, b, hk, 0), *vb = row_of<T>(p.v, p.sv, b, hk, 0);
    const float slope2 = p.slopes ? __ldg(p.slopes + h) * kLog2e : 0.0f;
    float m[L::RM], l[L::RM];
    float2 acc[L::RM][L::NJ][2] = {};
#pragma unroll
    for (int r = 0; r < L::RM; ++r) { m[r] = kNegInf; l[r] = 0.0f; }
    if (first < end) {
        simt_load<T, HD, L::BM>(sq, row_of<T>(p.q, p.sq, b, h, 0), p.sq[2], q0, p.Lq, p.D);
        simt_load<T, HD, kSimtKeys>(sk, kb, p.sk[2], first * kSimtKeys, p.Lk, p.D);
    }
    for (int j = first; j < end; ++j) {
        const int n0 = j * kSimtKeys;
        simt_wait();
        __syncthreads();                                        // q, k are there; the last tile's v and weights are read
        simt_load<T, HD, kSimtKeys>(sv, vb, p.sv[2], n0, p.Lk, p.D);
        float s[L::RM][4];
        simt_dot<HD>(sq, sk, s);
        const float unit = simt_cap(s, p.sm_scale, p.cap);
#pragma unroll
        for (int r = 0; r < L::RM; ++r) {
            const int pos = q0 + ty * L::RM + r + (p.Lk - p.Lq);
            float top = kNegInf;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int key = n0 + tx + 16 * c;
                float x = s[r][c] * unit;
                if (p.slopes) x = fmaf(-slope2, fabsf((float)(pos - key)), x);
                s[r][c] = key >= rg[r].x && key < rg[r].y ? x : kNegInf;
                top = fmaxf(top, s[r][c]);
            }
            top = fmaxf(m[r], half_warp_max(top));
            const float t0 = top == kNegInf ? 0.0f : top, f = fast_exp2(m[r] - t0);
            float sum = 0.0f;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float w = fast_exp2(s[r][c] - t0);
                sw[(ty * L::RM + r) * L::W + tx + 16 * c] = w;
                sum += w;
            }
            l[r] = fmaf(l[r], f, sum);                         // this thread's part of the sum
            m[r] = top;
#pragma unroll
            for (int x = 0; x < L::NJ; ++x)
#pragma unroll
                for (int z = 0; z < L::CW / 2; ++z) { acc[r][x][z].x *= f; acc[r][x][z].y *= f; }
        }
        simt_wait();
        __syncthreads();                                        // weights and v are there, k is read
        if (j + 1 < end) simt_load<T, HD, kSimtKeys>(sk, kb, p.sk[2], n0 + kSimtKeys, p.Lk, p.D);
        simt_rows<HD>(sw, sv, acc);
    }
    unsigned bad = 0;
#pragma unroll
    for (int r = 0; r < L::RM; ++r) {
        const int i = q0 + ty * L::RM + r;
        const float sum = half_warp_sum(l[r]), inv = sum != 0.0f ? 1.0f / sum : 0.0f;
        T* out = i < p.Lq ? row_of<T>(p.out, p.so, b, h, i) : nullptr;
        const float nan = half_warp_sum(simt_store<T, HD>(out, acc[r], inv, p.D) + sum * 0.0f);
        if (i < p.Lq) {
            if (tx == 0) p.lse[(long long)bh * p.Lq + i] = sum != 0.0f ? m[r] + log2f(sum) : kNegInf;
            if (nan != nan && sum == sum) bad |= 1u << r;       // a sum of weights that is NaN is the row's own
        }
    }
    simt_redo<L::RM>(bad, [&](int r) { exact_row_forward<T>(p, b, h, q0 + r); });
}

template <typename T, int HD>
__global__ void __launch_bounds__(kSimtThreads, SimtShape<HD>::kBlocks)
masked_simt_dq_kernel(const __grid_constant__ MaskedParams p, int qtiles) {
    using L = SimtShape<HD>;
    extern __shared__ float4 simt_smem[];
    float *sq = reinterpret_cast<float*>(simt_smem), *sg = sq + L::BM * L::S, *sk = sg + L::BM * L::S, *sv = sk + kSimtKeys * L::S,
          *sw = sv + kSimtKeys * L::S;
    __shared__ int s_lo, s_hi;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int bh = blockIdx.x % (p.B * p.Hq), b = bh / p.Hq, h = bh % p.Hq, hk = h / p.group;
    const int q0 = (qtiles - 1 - (int)(blockIdx.x / (p.B * p.Hq))) * L::BM;
    if (tid == 0) { s_lo = 0x7fffffff; s_hi = 0; }
    __syncthreads();
    int2 rg[L::RM];
    float lse[L::RM], delta[L::RM];
    int lo = 0x7fffffff, hi = 0;
#pragma unroll
    for (int r = 0; r < L::RM; ++r) {
        const int i = q0 + ty * L::RM + r;
        rg[r] = i < p.Lq ? key_range(p, b, i) : make_int2(0, 0);
        if (rg[r].x >= rg[r].y) rg[r] = make_int2(0, 0);
        else { lo = min(lo, rg[r].x); hi = max(hi, rg[r].y); }
        const bool sees = rg[r].x < rg[r].y;
        lse[r] = sees ? p.lse[(long long)bh * p.Lq + i] : kNegInf;
        if (lse[r] == kNegInf) lse[r] = -kNegInf;                // weight exp2(s - inf) = 0
        // delta = out.dout, the row's 16 threads together
        float part = 0.0f;
        if (sees) {
            const T* o = row_of<T>(p.out_in, p.so, b, h, i);
            const T* g = row_of<T>(p.dout, p.sdo, b, h, i);
            for (int d = tx * 8; d < p.D; d += 128) {
                float x[8], y[8];
                load8<T>(o + d, x);
                load8<T>(g + d, y);
                part += dot8(x, y);
            }
        }
        delta[r] = half_warp_sum(part);
        if (tx == 0 && i < p.Lq) p.delta[(long long)bh * p.Lq + i] = delta[r];
    }
    atomicMin(&s_lo, __reduce_min_sync(0xffffffffu, lo));
    atomicMax(&s_hi, __reduce_max_sync(0xffffffffu, hi));
    __syncthreads();
    const int first = s_hi > 0 ? s_lo / kSimtKeys : 0, end = s_hi > 0 ? (s_hi + kSimtKeys - 1) / kSimtKeys : 0;
    const T *kb = row_of<T>(p.k, p.sk, b, hk, 0), *vb = row_of<T>(p.v, p.sv, b, hk, 0);
    const float slope2 = p.slopes ? __ldg(p.slopes + h) * kLog2e : 0.0f;
    float2 acc[L::RM][L::NJ][2] = {};
    if (first < end) {
        simt_load<T, HD, L::BM>(sq, row_of<T>(p.q, p.sq, b, h, 0), p.sq[2], q0, p.Lq, p.D);
        simt_load<T, HD, L::BM>(sg, row_of<T>(p.dout, p.sdo, b, h, 0), p.sdo[2], q0, p.Lq, p.D);
    }
    for (int j = first; j < end; ++j) {
        const int n0 = j * kSimtKeys;
        simt_load<T, HD, kSimtKeys>(sk, kb, p.sk[2], n0, p.Lk, p.D);
        simt_load<T, HD, kSimtKeys>(sv, vb, p.sv[2], n0, p.Lk, p.D);
        simt_wait();
        __syncthreads();
        float s[L::RM][4], dp[L::RM][4];
        simt_dot<HD>(sq, sk, s);
        simt_dot<HD>(sg, sv, dp);
        const float unit = simt_cap(s, p.sm_scale, p.cap);
        if (sizeof(T) == 2 && end - first == 1) {
            // the only tile: delta from p and dp themselves, as in masked_dq_kernel
#pragma unroll
            for (int r = 0; r < L::RM; ++r) {
                const int i = q0 + ty * L::RM + r, pos = i + (p.Lk - p.Lq);
                float sum = 0.0f, all = 0.0f;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int key = n0 + tx + 16 * c;
                    float w, ds;
                    simt_grad(s[r][c], unit, false, p.slopes ? slope2 * fabsf((float)(pos - key)) : 0.0f, dp[r][c], lse[r], 0.0f, w, ds);
                    if (key >= rg[r].x && key < rg[r].y && w != 0.0f) { sum += ds; all += w; }
                }
                sum = half_warp_sum(sum);
                all = half_warp_sum(all);
                if (all != 0.0f) delta[r] = sum / all;
                if (tx == 0 && i < p.Lq) p.delta[(long long)bh * p.Lq + i] = delta[r];
            }
        }
#pragma unroll
        for (int r = 0; r < L::RM; ++r) {
            const int pos = q0 + ty * L::RM + r + (p.Lk - p.Lq);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int key = n0 + tx + 16 * c;
                float w, ds;
                simt_grad(s[r][c], unit, p.cap > 0.0f, p.slopes ? slope2 * fabsf((float)(pos - key)) : 0.0f, dp[r][c], lse[r], delta[r], w, ds);
                if (!(key >= rg[r].x && key < rg[r].y)) ds = 0.0f;
                sw[(ty * L::RM + r) * L::W + tx + 16 * c] = ds;
            }
        }
        __syncthreads();
        simt_rows<HD>(sw, sk, acc);
        __syncthreads();                                        // before the next tile takes the places
    }
    unsigned bad = 0;
#pragma unroll
    for (int r = 0; r < L::RM; ++r) {
        const int i = q0 + ty * L::RM + r;
        T* out = i < p.Lq ? row_of<T>(p.dq, p.sdq, b, h, i) : nullptr;
        const float nan = half_warp_sum(simt_store<T, HD>(out, acc[r], p.sm_scale, p.D));
        if (i < p.Lq && nan != nan && !spoilt(lse[r], delta[r])) bad |= 1u << r;
    }
    simt_redo<L::RM>(bad, [&](int r) { exact_row_dq<T>(p, b, h, q0 + r); });
}

template <typename T, int HD>
__global__ void __launch_bounds__(kSimtThreads, SimtShape<HD>::kBlocks)
masked_simt_dkdv_kernel(const __grid_constant__ MaskedParams p) {
    using L = SimtShape<HD>;
    extern __shared__ float4 simt_smem[];
    float *sq = reinterpret_cast<float*>(simt_smem), *sg = sq + L::BM * L::S, *sk = sg + L::BM * L::S, *sv = sk + kSimtKeys * L::S,
          *sw = sv + kSimtKeys * L::S;
    __shared__ int s_first, s_end;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int bh = blockIdx.x % (p.B * p.Hkv), b = bh / p.Hkv, hk = bh % p.Hkv, k0 = (int)(blockIdx.x / (p.B * p.Hkv)) * kSimtKeys;
    const int k1 = min(p.Lk, k0 + kSimtKeys);
    if (tid == 0) { s_first = 0x7fffffff; s_end = 0; }
    __syncthreads();
    // queries between the first and the last that see any of these keys
    int lo = 0x7fffffff, hi = 0;
    if (!p.visible) {
        lo = p.causal ? max(0, k0 - (p.Lk - p.Lq)) : 0;
        hi = p.Lq;
    } else {
        for (int i = tid; i < p.Lq; i += kSimtThreads) {
            const int2 r = key_range(p, b, i);
            if (r.x < r.y && r.x < k1 && r.y > k0) { lo = min(lo, i); hi = max(hi, i + 1); }
        }
    }
    atomicMin(&s_first, __reduce_min_sync(0xffffffffu, lo));
    atomicMax(&s_end, __reduce_max_sync(0xffffffffu, hi));
    simt_load<T, HD, kSimtKeys>(sk, row_of<T>(p.k, p.sk, b, hk, 0), p.sk[2], k0, p.Lk, p.D);
    simt_load<T, HD, kSimtKeys>(sv, row_of<T>(p.v, p.sv, b, hk, 0), p.sv[2], k0, p.Lk, p.D);
    __syncthreads();
    const int first = s_first / L::BM, end = s_first < s_end ? (s_end + L::BM - 1) / L::BM : first;
    float2 ak[4][L::NJ][2] = {}, av[4][L::NJ][2] = {};
    for (int g = 0; g < p.group; ++g) {
        const int h = hk * p.group + g;
        const float slope2 = p.slopes ? __ldg(p.slopes + h) * kLog2e : 0.0f;
        for (int t = first; t < end; ++t) {
            const int q0 = t * L::BM;
            simt_load<T, HD, L::BM>(sq, row_of<T>(p.q, p.sq, b, h, 0), p.sq[2], q0, p.Lq, p.D);
            simt_load<T, HD, L::BM>(sg, row_of<T>(p.dout, p.sdo, b, h, 0), p.sdo[2], q0, p.Lq, p.D);
            // queries without weight or spoilt: their rows, which may hold anything, out of the sums of rows to come
            bool off = false;
            if (tid < L::BM && q0 + tid < p.Lq) {
                const long long row = ((long long)b * p.Hq + h) * p.Lq + q0 + tid;
                off = p.lse[row] == kNegInf || spoilt(p.lse[row], p.delta[row]);
            }
            simt_wait();
            if (__syncthreads_or(off)) {
                if (off)
                    for (int d = 0; d < HD; ++d) sq[tid * L::S + d] = sg[tid * L::S + d] = 0.0f;
                __syncthreads();
            }
            float s[L::RM][4], dp[L::RM][4];
            simt_dot<HD>(sq, sk, s);
            simt_dot<HD>(sg, sv, dp);
            const float unit = simt_cap(s, p.sm_scale, p.cap);
#pragma unroll
            for (int r = 0; r < L::RM; ++r) {
                const int i = q0 + ty * L::RM + r, pos = i + (p.Lk - p.Lq);
                int2 rg = make_int2(0, 0);
                float lse = 0.0f, delta = 0.0f;
                if (i < p.Lq) {
                    rg = key_range(p, b, i);
                    const long long row = ((long long)b * p.Hq + h) * p.Lq + i;
                    lse = p.lse[row];
                    delta = p.delta[row];
                    if (spoilt(lse, delta)) lse = __int_as_float(0x7fffffff);       // all that sees it becomes NaN
                    if (lse == kNegInf) lse = -kNegInf;
                }
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int key = k0 + tx + 16 * c;
                    float w, ds;
                    simt_grad(s[r][c], unit, p.cap > 0.0f, p.slopes ? slope2 * fabsf((float)(pos - key)) : 0.0f, dp[r][c], lse, delta, w, ds);
                    if (!(key >= rg.x && key < rg.y)) w = ds = 0.0f;
                    sw[(ty * L::RM + r) * L::W + tx + 16 * c] = w;
                    s[r][c] = ds;
                }
            }
            __syncthreads();
            simt_columns<HD>(sw, sg, av);
            __syncthreads();
#pragma unroll
            for (int r = 0; r < L::RM; ++r)
#pragma unroll
                for (int c = 0; c < 4; ++c) sw[(ty * L::RM + r) * L::W + tx + 16 * c] = s[r][c];
            __syncthreads();
            simt_columns<HD>(sw, sq, ak);
            __syncthreads();
        }
    }
    simt_wait();
    unsigned bad = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const int key = k0 + ty * 4 + c;
        T* dk = key < p.Lk ? row_of<T>(p.dk, p.sdk, b, hk, key) : nullptr;
        T* dv = key < p.Lk ? row_of<T>(p.dv, p.sdv, b, hk, key) : nullptr;
        const float nan = half_warp_sum(simt_store<T, HD>(dk, ak[c], p.sm_scale, p.D) + simt_store<T, HD>(dv, av[c], 1.0f, p.D));
        if (key < p.Lk && nan != nan) bad |= 1u << c;
    }
    simt_redo<4>(bad, [&](int r) { exact_row_dkdv<T>(p, b, hk, k0 + r); });
}

}  // namespace dsdpa
