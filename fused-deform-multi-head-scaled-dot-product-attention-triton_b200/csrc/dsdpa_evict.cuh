// Eviction from a paged cache: which keys stay (evict_select_kernel) and their rows moved
// (evict_move_kernel).
#pragma once

#include "dsdpa_cache.cuh"

namespace dsdpa {

struct EvictParams {
    char *k, *v;
    const int *table, *lens, *positions, *out_table;
    const float* weights;
    int *kept, *new_lens, *new_positions;
    float* new_weights;
    int B, Hkv, pages, page_size, width, out_width, slots, keep, sinks, recent;
    int row_bytes;
    long long sk[3], sv[3];   // bytes: page, head, slot
    int* err;
};

constexpr int kSelectThreads = 1024;

// Order of weights as unsigned integers: NaN below everything, both zeros alike.
__device__ __forceinline__ unsigned weight_rank(float w) {
    if (w != w) return 0u;
    const unsigned u = __float_as_uint(w + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One block finds the keys that one (sequence, key/value head) keeps.  A radix select, eight bits a
// pass, finds the rank that the last kept key has; the kept keys are then written in their order, every
// warp having a contiguous part of the keys: it counts first and writes once it knows what lies before.
// All of it reads the weights (L2 holds them after the first pass) and is bound by those reads and by
// the block's barriers.
__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const EvictParams p) {
    constexpr int kWarps = kSelectThreads / 32;
    __shared__ unsigned hist[256];
    __shared__ unsigned s_prefix, s_left;
    __shared__ int s_more[kWarps], s_same[kWarps];
    const int b = blockIdx.x / p.Hkv, h = blockIdx.x % p.Hkv;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int room = p.width * p.page_size;
    int n = __ldg(p.lens + b);
    if (n > room && tid == 0) atomicCAS(p.err, 0, kErrBounds);
    n = max(0, min(n, room));
    const long long row = (long long)b * p.Hkv + h;
    const float* w = p.weights + row * p.slots;
    const int* pos = p.positions ? p.positions + row * p.slots : nullptr;
    float* nw = p.new_weights + row * p.slots;
    int* np = p.new_positions ? p.new_positions + row * p.slots : nullptr;
    int* kept = p.kept + row * p.keep;
    const int left = min(n, p.keep);
    if (h == 0 && tid == 0) p.new_lens[b] = left;
    for (int i = left + tid; i < p.keep; i += kSelectThreads) kept[i] = -1;
    for (int i = left + tid; i < p.slots; i += kSelectThreads) {
        nw[i] = 0.0f;
        if (np) np[i] = 0;
    }
    auto put = [&](int at, int key) {
        kept[at] = key;
        nw[at] = w[key];
        if (np) np[at] = pos ? pos[key] : key;
    };
    if (n <= p.keep) {
        for (int i = tid; i < n; i += kSelectThreads) put(i, i);
        return;
    }
    for (int i = tid; i < p.sinks; i += kSelectThreads) put(i, i);
    for (int i = tid; i < p.recent; i += kSelectThreads) put(p.keep - p.recent + i, n - p.recent + i);
    const int first = p.sinks, last = n - p.recent, want = p.keep - p.sinks - p.recent;
    if (want == 0) return;   // the same for the whole block

    unsigned prefix = 0, mask = 0, need = (unsigned)want;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += kSelectThreads) hist[i] = 0;
        __syncthreads();
        for (int i = first + tid; i < last; i += kSelectThreads) {
            const unsigned u = weight_rank(w[i]);
            if ((u & mask) == prefix) atomicAdd(&hist[(u >> shift) & 255u], 1u);
        }
        __syncthreads();
        if (warp == 0) {
            // the digit d with: keys above d < need <= keys above d plus keys at d; lane l has digits 255-8l down
            unsigned cnt[8], sum = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) { cnt[e] = hist[255 - 8 * lane - e]; sum += cnt[e]; }
            unsigned before = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned t = __shfl_up_sync(0xffffffffu, before, o);
                if (lane >= o) before += t;
            }
            before -= sum;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (before < need && need <= before + cnt[e]) {
                    s_prefix = prefix | (unsigned)(255 - 8 * lane - e) << shift;
                    s_left = need - before;
                }
                before += cnt[e];
            }
        }
        __syncthreads();
        prefix = s_prefix;
        need = s_left;
        mask |= 255u << shift;
        __syncthreads();
    }
    // keys above the rank `prefix` stay, and the first `need` of those at it
    const int span = last - first, part = ((span + kWarps - 1) / kWarps + 31) & ~31;
    const int lo = first + min(span, warp * part), hi = first + min(span, (warp + 1) * part);
    int more = 0, same = 0;
    for (int i = lo + lane; i < hi; i += 32) {
        const unsigned u = weight_rank(w[i]);
        more += u > prefix;
        same += u == prefix;
    }
    more = __reduce_add_sync(0xffffffffu, more);
    same = __reduce_add_sync(0xffffffffu, same);
    if (lane == 0) { s_more[warp] = more; s_same[warp] = same; }
    __syncthreads();
    int more0 = 0, same0 = 0;
    for (int i = 0; i < warp; ++i) { more0 += s_more[i]; same0 += s_same[i]; }
    const unsigned below = (1u << lane) - 1;
    for (int i0 = lo; i0 < hi; i0 += 32) {
        const int i = i0 + lane;
        const unsigned u = i < hi ? weight_rank(w[i]) : 0u;
        const unsigned bm = __ballot_sync(0xffffffffu, i < hi && u > prefix);
        const unsigned bs = __ballot_sync(0xffffffffu, i < hi && u == prefix);
        const int my_more = more0 + __popc(bm & below), my_same = same0 + __popc(bs & below);
        const bool is_more = bm >> lane & 1, is_same = bs >> lane & 1;
        if (is_more || (is_same && my_same < (int)need)) put(p.sinks + my_more + min(my_same, (int)need), i);
        more0 += __popc(bm);
        same0 += __popc(bs);
    }
}

// The kept rows to their new places.  A block has 64 bytes (two sectors) of every row of one
// (sequence, head), of K or of V, and goes through the rows in their order: a row's place is never
// behind it, so with all of a batch of rows loaded before any of it is stored the move is right in
// place too, and the blocks need nothing from one another.  Bound by DRAM: every byte is read and
// written once.
constexpr int kMoveThreads = 512, kMoveRows = 8;
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictParams p) {
    constexpr int kPerPass = kMoveThreads / 4;
    const int slices = (p.row_bytes + 63) / 64;
    int at = blockIdx.x;
    const int slice = at % slices; at /= slices;
    const bool is_v = at & 1; at >>= 1;
    const int h = at % p.Hkv, b = at / p.Hkv;
    const int left = p.new_lens[b];
    const int byte = slice * 64 + (threadIdx.x & 3) * 16;
    const bool active = byte < p.row_bytes;
    char* base = (is_v ? p.v : p.k) + (is_v ? p.sv[1] : p.sk[1]) * h + byte;
    const long long sp = is_v ? p.sv[0] : p.sk[0], ss = is_v ? p.sv[2] : p.sk[2];
    const int* kept = p.kept + ((long long)b * p.Hkv + h) * p.keep;
    for (int i0 = 0; i0 < left; i0 += kPerPass * kMoveRows) {
        uint4 r[kMoveRows];
        char* to[kMoveRows];
#pragma unroll
        for (int u = 0; u < kMoveRows; ++u) {
            const int i = i0 + u * kPerPass + (threadIdx.x >> 2);
            to[u] = nullptr;
            if (i >= left || !active) continue;
            const int key = kept[i];
            const int si = key / p.page_size, di = i / p.page_size;
            const int sp_i = page_of(p.table, p.width, p.pages, p.err, b, si);
            const int dp_i = page_of(p.out_table, p.out_width, p.pages, p.err, b, di);
            if (sp_i < 0 || dp_i < 0) continue;
            const char* from = base + sp_i * sp + (key - si * p.page_size) * ss;
            to[u] = base + dp_i * sp + (i - di * p.page_size) * ss;
            if (from == to[u]) { to[u] = nullptr; continue; }
            r[u] = *reinterpret_cast<const uint4*>(from);
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kMoveRows; ++u)
            if (to[u]) *reinterpret_cast<uint4*>(to[u]) = r[u];
    }
}

}  // namespace dsdpa
