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
    int held;                 // ranks that evict_select_kernel has room for in shared memory
    PageDivision div;
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
// The ranks are held in shared memory, as far as they fit (p.held); the rest is read from L2 again in
// every pass.  (A histogram with a counter for every lane, so that no two lanes meet, measured 3 us slower
// for 16384 keys than four plain ones.)
__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const __grid_constant__ EvictParams p) {
    constexpr int kWarps = kSelectThreads / 32;
    extern __shared__ unsigned s_rank[];
    __shared__ unsigned hist[4][4][256];        // of every digit, four copies that keep warps apart
    __shared__ unsigned s_total[8], s_prefix, s_left;
    __shared__ int s_more[kWarps], s_same[kWarps];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int b = blockIdx.x / p.Hkv, h = blockIdx.x % p.Hkv;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int room = p.width * p.page_size;
    int n = __ldg(p.lens + b);
    if (n > room && tid == 0) atomicCAS(p.err, 0, kErrBounds);
    n = max(0, min(n, room));
    const long long row = (long long)b * p.Hkv + h;
    const float* __restrict__ w = p.weights + row * p.slots;
    const int* __restrict__ pos = p.positions ? p.positions + row * p.slots : nullptr;
    float* __restrict__ nw = p.new_weights + row * p.slots;
    int* __restrict__ np = p.new_positions ? p.new_positions + row * p.slots : nullptr;
    int* __restrict__ kept = p.kept + row * p.keep;
    const int left = min(n, p.keep);
    if (h == 0 && tid == 0) p.new_lens[b] = left;
    auto put = [&](int at, int key) {
        if (!in_range(at, min(p.keep, p.slots), p.err) || !in_range(key, p.slots, p.err)) return;
        kept[at] = key;
        nw[at] = w[key];
        if (np) np[at] = pos ? pos[key] : key;
    };
    const int first = p.sinks, last = n - p.recent, want = p.keep - p.sinks - p.recent;
    if (n <= p.keep) {
        for (int i = tid; i < n; i += kSelectThreads) put(i, i);
    } else {
        for (int i = tid; i < p.sinks; i += kSelectThreads) put(i, i);
        for (int i = tid; i < p.recent; i += kSelectThreads) put(p.keep - p.recent + i, n - p.recent + i);
    }
    if (n > p.keep && want > 0) {       // the same for the whole block
        const int span = last - first;
        auto rank = [&](int i) { return i < p.held ? s_rank[i] : weight_rank(__ldg(w + first + i)); };
        for (int i = tid; i < 4 * 4 * 256; i += kSelectThreads) (&hist[0][0][0])[i] = 0;
        __syncthreads();
        // pass over the top digit, which also fills the held ranks
#pragma unroll 8
        for (int i = tid; i < span; i += kSelectThreads) {
            const unsigned u = weight_rank(__ldg(w + first + i));
            if (i < p.held) s_rank[i] = u;
            atomicAdd(&hist[3][warp & 3][u >> 24], 1u);
        }
        unsigned prefix = 0, mask = 0, need = (unsigned)want;
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (shift < 24) {
#pragma unroll 8
                for (int i = tid; i < span; i += kSelectThreads) {
                    const unsigned u = rank(i);
                    if ((u & mask) == prefix) atomicAdd(&hist[shift >> 3][warp & 3][(u >> shift) & 255u], 1u);
                }
            }
            __syncthreads();
            // the digit d with: keys above d < need <= keys above d plus keys at d; thread t has digit 255 - t
            unsigned cnt = 0, upto = 0;
            if (warp < 8) {
                const unsigned (&c)[4][256] = hist[shift >> 3];
                const int d = 255 - tid;
                cnt = c[0][d] + c[1][d] + c[2][d] + c[3][d];
                upto = cnt;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const unsigned t = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += t;
                }
                if (lane == 31) s_total[warp] = upto;
            }
            __syncthreads();
            if (warp < 8) {
                for (int i = 0; i < warp; ++i) upto += s_total[i];
                if (upto - cnt < need && need <= upto) {
                    s_prefix = prefix | (unsigned)(255 - tid) << shift;
                    s_left = need - (upto - cnt);
                }
            }
            __syncthreads();
            prefix = s_prefix;
            need = s_left;
            mask |= 255u << shift;
        }
        // keys above the rank `prefix` stay, and the first `need` of those at it
        const int part = ((span + kWarps - 1) / kWarps + 31) & ~31;
        const int lo = min(span, warp * part), hi = min(span, (warp + 1) * part);
        int more = 0, same = 0;
#pragma unroll 4
        for (int i = lo + lane; i < hi; i += 32) {
            const unsigned u = rank(i);
            more += u > prefix;
            same += u == prefix;
        }
        more = __reduce_add_sync(0xffffffffu, more);
        same = __reduce_add_sync(0xffffffffu, same);
        if (lane == 0) { s_more[warp] = more; s_same[warp] = same; }
        __syncthreads();
        // what lies before: the sums over the warps in front of this one
        int more0 = __reduce_add_sync(0xffffffffu, lane < warp ? s_more[lane] : 0);
        int same0 = __reduce_add_sync(0xffffffffu, lane < warp ? s_same[lane] : 0);
        const unsigned below = (1u << lane) - 1;
        constexpr int kBatch = 8;                         // places first, then the loads that they need, then the stores
        for (int i0 = lo; i0 < hi; i0 += 32 * kBatch) {
            int to[kBatch];
            float val[kBatch];
#pragma unroll
            for (int e = 0; e < kBatch; ++e) {
                const int i = i0 + e * 32 + lane;
                const unsigned u = i < hi ? rank(i) : 0u;
                const unsigned bm = __ballot_sync(0xffffffffu, i < hi && u > prefix);
                const unsigned bs = __ballot_sync(0xffffffffu, i < hi && u == prefix);
                const int my_more = more0 + __popc(bm & below), my_same = same0 + __popc(bs & below);
                const bool stays = (bm >> lane & 1) || ((bs >> lane & 1) && my_same < (int)need);
                to[e] = stays ? p.sinks + my_more + min(my_same, (int)need) : -1;
                val[e] = stays ? __ldg(w + first + i) : 0.0f;
                more0 += __popc(bm);
                same0 += __popc(bs);
            }
#pragma unroll
            for (int e = 0; e < kBatch; ++e)
                if (to[e] >= 0 && in_range(to[e], min(p.keep, p.slots), p.err)) {
                    const int i = first + i0 + e * 32 + lane;
                    kept[to[e]] = i;
                    nw[to[e]] = val[e];
                    if (np) np[to[e]] = pos ? __ldg(pos + i) : i;
                }
        }
    }
    for (int i = left + tid; i < p.keep; i += kSelectThreads) kept[i] = -1;
    for (int i = left + tid; i < p.slots; i += kSelectThreads) {
        nw[i] = 0.0f;
        if (np) np[i] = 0;
    }
}

// The kept rows to their new places.  A block has `width` 16-byte pieces of every row of one (sequence, head), of
// K or of V, and goes through the rows in their order: a row's place is never behind it, so with all of a
// batch of rows loaded before any of it is stored the move is right in place too, and the blocks need
// nothing from one another.  The next batch's key and page numbers are fetched while this one's rows
// are on their way.  Bound by DRAM: every byte is read and written once.  Measured with the selection, 16 caches of up to
// 16384 keys cut to 4096 (8 heads, D = 128): bf16 130 us (548 MB, 4.2 TB/s, of which the selection takes 20 us), fp32
// 214 us (5.1 TB/s).  Copies through a ring in shared memory took 140 us where this took 109.
constexpr int kMoveThreads = 256, kMoveRows = 4, kMoveBlocks = 4;   // blocks an SM
__global__ void __launch_bounds__(kMoveThreads, kMoveBlocks) evict_move_kernel(const __grid_constant__ EvictParams p, int width, int slices) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int per = kMoveThreads / width, mine = threadIdx.x / width;
    int at = blockIdx.x;
    const int slice = at % slices; at /= slices;
    const bool is_v = at & 1; at >>= 1;
    const int h = at % p.Hkv, b = at / p.Hkv;
    const int left = p.new_lens[b];
    const int byte = (slice * width + threadIdx.x % width) * 16;
    const int last = byte < p.row_bytes ? left : 0;          // threads behind the row's end have none
    char* base = (is_v ? p.v : p.k) + (is_v ? p.sv[1] : p.sk[1]) * h + byte;
    const long long sp = is_v ? p.sv[0] : p.sk[0], ss = is_v ? p.sv[2] : p.sk[2];
    const int* kept = p.kept + ((long long)b * p.Hkv + h) * p.keep;
    int key[kMoveRows];
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u) key[u] = u * per + mine < last ? kept[u * per + mine] : -1;
    for (int i0 = 0; i0 < left; i0 += per * kMoveRows) {
        uint4 r[kMoveRows];
        char* to[kMoveRows];
#pragma unroll
        for (int u = 0; u < kMoveRows; ++u) {
            const int i = i0 + u * per + mine;
            to[u] = nullptr;
            if (key[u] < 0) continue;
            const int si = page_index(p.div, key[u]), di = page_index(p.div, i);
            const int from_page = page_of(p.table, p.width, p.pages, p.err, b, si);
            const int to_page = page_of(p.out_table, p.out_width, p.pages, p.err, b, di);
            if (from_page < 0 || to_page < 0) continue;
            const char* from = base + from_page * sp + (key[u] - si * p.page_size) * ss;
            to[u] = base + to_page * sp + (i - di * p.page_size) * ss;
            if (from == to[u]) { to[u] = nullptr; continue; }
            r[u] = *reinterpret_cast<const uint4*>(from);
        }
#pragma unroll
        for (int u = 0; u < kMoveRows; ++u) {
            const int i = i0 + (kMoveRows + u) * per + mine;
            key[u] = i < last ? kept[i] : -1;
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kMoveRows; ++u)
            if (to[u]) *reinterpret_cast<uint4*>(to[u]) = r[u];
    }
}

}  // namespace dsdpa
