// Accumulated attention weights on the tensor cores: 16-bit storage, head dimensions up to 128.
//
// S^T = k q^T, 128 keys by up to 128 (token, head) rows, so that a thread has one key and adds up its row of
// weights without a word to another thread: weights = sum over the columns of exp2(s - lse).  Keys are shared out over the
// blocks like those of tree attention; every key has one writer.  With more than 128 rows a block goes
// through its keys once for every 128.  Bound by DRAM: the keys are read once, four bytes of weight read and
// written for each.  Roles: warps 0-3 and 4-7 take every second key tile's sums, 8-11 copy rows, 12 issues
// the matrix instructions.  Taken for more than 16 rows: 64 caches of up to 8192 keys, 5 tokens of 32 heads on 8 (20 rows),
// D = 128, bf16, take 133 us (3.8 TB/s; dsdpa_few.cuh, with 16 rows, 105 us).
#pragma once

#include "dsdpa_tree.cuh"

namespace dsdpa {

template <typename T, int HD, bool CAP, bool BIAS>
__global__ void __launch_bounds__(kTreeThreads, 1)
weights_kernel(const __grid_constant__ CacheParams p, const __grid_constant__ TreeSplit sp, int negate) {
    using L = TreeLayout<HD>;
    extern __shared__ char smem_raw[];
    const uint32_t smem = (smem_addr(smem_raw) + 1023u) & ~1023u;
    const uint32_t sm_q = smem, sm_ring = smem + 2 * L::kTileBytes, bars = sm_ring + L::kStages * L::kTileBytes;
    // bar_s, bar_r: a score buffer filled, read; bar_qe: a query tile and its columns' data free
    const uint32_t bar_s = bars, bar_r = bars + 32, bar_qe = bars + 64, bar_full = bars + 80, bar_empty = bar_full + 8 * L::kStages,
                   slot = bar_empty + 8 * L::kStages;
    __shared__ unsigned s_valid[kInfo][4];
    __shared__ float s_lse[2][kTreeRows], s_pos[2][BIAS ? kTreeRows : 1], s_slope[2][BIAS ? kTreeRows : 1];
    __shared__ unsigned long long s_above[2][kTreeRows];
    __shared__ TreeShare<kTreeThreads> share;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rows = p.T * p.group, passes = (rows + kTreeRows - 1) / kTreeRows;

    if (tid == 0) {
        for (int i = 0; i < 4; ++i) { mbar_init(bar_s + 8 * i, 1); mbar_init(bar_r + 8 * i, 4); }
        mbar_init(bar_qe, 9);          // the matrix instructions, and the eight warps that read the columns' data
        mbar_init(bar_qe + 8, 9);
        for (int i = 0; i < L::kStages; ++i) { mbar_init(bar_full + 8 * i, 4); mbar_init(bar_empty + 8 * i, 1); }
        fence_mbar_init();
    }
    if (warp == 12) tmem_alloc(slot, 512);
    find_share<TreeTile>(p, sp, share);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    uint32_t tmem;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(slot));
    TreeWalk<TreeTile> walk = share.walk<TreeTile>();
    // an item's passes over its rows; pass numbers run on over the items
    int pass = 0;

    if (warp == 12) {
        if (elect_one()) {
            int st = 0, ph = 0, n[2] = { 0, 0 };       // tiles of each side: it has two score buffers of its own
            bool ok = true;
            TreeItem it;
            while (ok && walk.next(p, sp, it))
                for (int r = 0; r < passes && ok; ++r, ++pass) {
                    const int cols = min(kTreeRows, rows - r * kTreeRows);
                    const uint32_t id = mma_desc<T>((cols + 15) & ~15, false, negate != 0);
                    const uint32_t q = sm_q + (pass & 1) * L::kTileBytes;
                    for (int i = 0; i < it.tiles; ++i) {
                        const int m = i & 1 ? n[1]++ : n[0]++, at = (i & 1) * 2 + (m & 1);
                        if (!(ok = mbar_wait_bounded(bar_full + 8 * st, ph, p.err) &&
                                   mbar_wait_bounded(bar_r + 8 * at, ((m >> 1) & 1) ^ 1, p.err))) break;
                        tc_fence_after();
                        mma_rows<HD>(tmem + at * kTreeRows, sm_ring + st * L::kTileBytes, q, kTreeRows, id);
                        mma_commit(bar_s + 8 * at);
                        mma_commit(bar_empty + 8 * st);
                        if (++st == L::kStages) { st = 0; ph ^= 1; }
                    }
                    if (ok) mma_commit(bar_qe + 8 * (pass & 1));
                }
        }
    } else if (warp >= 8) {
        const int w = warp - 8;
        int st = 0, ph = 1, entries = 0, handed = 0;
        bool ok = true;
        auto hand_over = [&](int up_to) {
            fence_proxy_async();
            __syncwarp();
            for (; handed < up_to; ++handed)
                if (lane == 0) mbar_arrive(bar_full + 8 * (handed % L::kStages));
        };
        auto lookup = [&](const TreeItem& it, int i) {          // not looked at yet: nothing waits for it here
            const int j = it.key0 + i * kTreeKeys + w * 32 + lane;
            return i < it.tiles && j < it.n + it.real ? table_entry(p.table, p.width, it.b, page_index(p.div, j)) : 0;
        };
        TreeItem it;
        while (ok && walk.next(p, sp, it))
            for (int r = 0; r < passes && ok; ++r, ++pass) {
                int page = lookup(it, 0);
                const int buf = pass & 1;
                // the pass before the last has to be over; it may need what has not been handed over yet
                if (!__all_sync(0xffffffffu, mbar_try_wait(bar_qe + 8 * buf, ((pass >> 1) & 1) ^ 1))) {
                    cp_async_wait<0>();
                    hand_over(entries);
                }
                if (!(ok = mbar_wait_bounded(bar_qe + 8 * buf, ((pass >> 1) & 1) ^ 1, p.err))) break;
                const int col = w * 32 + lane, gr = r * kTreeRows + col, t = gr / p.group, h = it.hk * p.group + gr % p.group;
                const bool valid = gr < rows;
                copy_rows<HD>(sm_q + buf * L::kTileBytes, w, lane, valid ? (const char*)row_of<T>(p.q, p.sq, it.b, h, t) : nullptr,
                              (const char*)p.q, p.D);
                // a column that does not count has an infinite lse: its weights are zero
                float lse = -kNegInf;
                unsigned long long above = 0;
                if (valid && t < it.real && !(p.take && !p.take[(long long)it.b * p.T + t])) {
                    lse = p.lse[((long long)it.b * p.Hq + h) * p.T + t];
                    if (lse == kNegInf) lse = -kNegInf;
                    above = tokens_above(p, it.b, t);
                }
                s_lse[buf][col] = lse;
                s_above[buf][col] = above;
                if (BIAS) {
                    s_pos[buf][col] = above ? (float)depth_of(above) : 0.0f;
                    s_slope[buf][col] = valid ? __ldg(p.slopes + h) * kLog2e : 0.0f;
                }
                for (int i = 0; i < it.tiles; ++i) {
                    const int j = it.key0 + i * kTreeKeys + w * 32 + lane, key = j - page_index(p.div, j) * p.page_size;
                    const int more = lookup(it, i + 1);
                    const char* src = nullptr;
                    if (j < it.n + it.real && (page = checked_page(page, p.pages, p.err)) >= 0)
                        src = (const char*)(row_of<T>(p.k, p.sk, 0, it.hk, key) + page * p.sk[0]);
                    if (!(ok = mbar_wait_bounded(bar_empty + 8 * st, ph, p.err))) break;
                    const unsigned there = __ballot_sync(0xffffffffu, src != nullptr);
                    if (lane == 0) s_valid[entries % kInfo][w] = there;
                    copy_rows<HD>(sm_ring + st * L::kTileBytes, w, lane, src, (const char*)p.k, p.D);
                    cp_async_commit();
                    if (++st == L::kStages) { st = 0; ph ^= 1; }
                    if (++entries - handed > L::kAhead) {
                        cp_async_wait<L::kAhead>();
                        hand_over(entries - L::kAhead);
                    }
                    page = more;
                }
            }
        cp_async_wait<0>();
        if (ok) hand_over(entries);
    } else {
        const int side = warp >> 2, quad = warp & 3;
        const uint32_t lanes = (uint32_t)quad << 21;
        ScoreConsts c;
        c.scale2 = fabsf(p.sm_scale) * kLog2e;
        c.cap_in = CAP ? 2.0f * fabsf(p.sm_scale) / p.cap : 0.0f;
        c.cap_out = CAP ? p.cap * kLog2e : 0.0f;
        const float unit = CAP ? c.cap_out : c.scale2;
        int n = 0, m = 0;          // key tiles of the block, and of this side
        bool ok = true;
        TreeItem it;
        while (ok && walk.next(p, sp, it))
            for (int r = 0; r < passes && ok; ++r, ++pass) {
                const int cols = min(kTreeRows, rows - r * kTreeRows), buf = pass & 1;
                float* out = p.weights + ((long long)it.b * p.Hkv + it.hk) * p.slots;
                for (int i = 0; i < it.tiles; ++i, ++n) {
                    if ((i & 1) != side) continue;       // the same thread in every pass
                    const int j = it.key0 + i * kTreeKeys + quad * 32 + lane, draft = j - it.n;
                    // a drafted key that the table has no room for is behind the row of weights too
                    const bool exists = draft < it.real && j < p.width * p.page_size;
                    const float old = exists && in_range(j, p.slots, p.err) ? out[j] : 0.0f;
                    float at = 0.0f;
                    if (BIAS && exists)
                        at = draft >= 0 ? (float)depth_of(tokens_above(p, it.b, draft)) : key_position(p, it.b, it.hk, j, first_position(p, it.b, it.n));
                    const int buffer = side * 2 + (m & 1);
                    if (!(ok = mbar_wait_bounded(bar_s + 8 * buffer, (m >> 1) & 1, p.err))) break;
                    ++m;
                    tc_fence_after();
                    const bool there = s_valid[n % kInfo][quad] >> lane & 1u;
                    const bool drafted = __any_sync(0xffffffffu, draft >= 0);
                    float sum = 0.0f;
#pragma unroll 1
                    for (int x = 0; x < cols; x += 16) {
                        float s[16], part[4] = { 0.0f, 0.0f, 0.0f, 0.0f };
                        tmem_ld16(tmem + buffer * kTreeRows + x + lanes, s);
                        tmem_wait_ld();
                        if (CAP) cap_scores(s, c);
#pragma unroll
                        for (int y = 0; y < 16; ++y) {
                            const float lse = s_lse[buf][x + y];
                            float v = fmaf(s[y], unit, -lse);
                            if (BIAS) v = fmaf(-s_slope[buf][x + y], fabsf(s_pos[buf][x + y] - at), v);
                            s[y] = fast_exp2(v);
                        }
                        // a column that does not count may meet a NaN product: its weight is zero all the same
#pragma unroll
                        for (int y = 0; y < 16; ++y) s[y] = s_lse[buf][x + y] == -kNegInf ? 0.0f : s[y];
                        if (drafted) {
#pragma unroll
                            for (int y = 0; y < 16; ++y) s[y] = draft < 0 || (s_above[buf][x + y] >> (draft & 63) & 1u) ? s[y] : 0.0f;
                        }
#pragma unroll
                        for (int y = 0; y < 16; ++y) part[y & 3] += s[y];
                        sum += (part[0] + part[1]) + (part[2] + part[3]);
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar_r + 8 * buffer);
                    if (exists && there && in_range(j, p.slots, p.err)) out[j] = old + sum;
                }
                // a warp without a tile in this pass must not run ahead: its next arrival would count for this phase
                ok = ok && mbar_wait_bounded(bar_qe + 8 * buf, ((pass >> 1) & 1) ^ 1, p.err);
                __syncwarp();
                if (ok && lane == 0) mbar_arrive(bar_qe + 8 * buf);
            }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 12) tmem_free(tmem, 512);
}

}  // namespace dsdpa
