// Attention of drafted tokens over a paged cache on the tensor cores: 16-bit storage, head dimensions up
// to 128.
//
// A unit's queries (up to 128 rows, dsdpa_share.cuh) are one operand, so that the cache is read once for all of them.
// A block's loads run ahead of its arithmetic, from one unit into the next.
// Inside a unit key tiles of 128 go in turn to two streams, each with its own running maximum, sum and
// accumulator (tensor memory holds both), joined at the end: one stream's softmax runs while the other's
// products do, which matters when a handful of rows leaves a single warp with all of the softmax.
// Taken for more than 16 rows (dsdpa_few.cuh has the others).  Measured, three caches of up to 65536 keys, 32 heads on 8, trees of
// 29 tokens (116 rows), D = 128, fp16: 149 us without cap or bias (4.5 TB/s), 168 us biased, 184 us capped, 207 us
// both, where reading the cache takes 103 us: bound by DRAM's latency and, with a cap, by the softmax's
// arithmetic.  Loads by TMA, a box for each page, were slower (254 -> 320 us then): boxes are issued one by one.
// Roles: warps 0-3 and 4-7 the streams' softmax, 8-11 copy rows (cp.async: any page size and stride, rows
// that are not there read as zero), 12 issues the matrix instructions.
#pragma once

#include "dsdpa_masked_fwd.cuh"
#include "dsdpa_share.cuh"

namespace dsdpa {

constexpr int kTreeThreads = 416;
constexpr int kTreeRows = 128, kTreeKeys = 128, kInfo = 16;
using TreeTile = ShareTile<kTreeRows, kTreeKeys>;

template <int HD>
struct TreeLayout {
    static constexpr int kTileBytes = 128 * HD * 2;
    static constexpr int kStages = HD == 128 ? 4 : 8;
    // Entries issued behind the one that a producer waits for: with it, three times 32 KB in flight cover the
    // latency, and the ring's other entries are the products' to work on.
    static constexpr int kAhead = HD == 128 ? 2 : 5;
    static constexpr int kSmem = 2 * kTileBytes + kStages * kTileBytes + 1024 + 512;
};

__device__ __forceinline__ void pair_barrier(int id) { asm volatile("bar.sync %0, 64;" :: "r"(id) : "memory"); }

// The 32 rows whose addresses the warp's lanes hold (null: zeros) into rows 32w .. 32w+31 of a tile, swizzled.
template <int HD>
__device__ __forceinline__ void copy_rows(uint32_t tile, int w, int lane, const char* row, const char* any, int D) {
    constexpr int kPer = HD / 8, kAt = 32 / kPer;          // 16-byte pieces of a row, rows of an instruction
    const int c = lane % kPer;
    // all exchanges first: the copies keep their order, and would have every one of them wait for an exchange
    const char* src[32 / kAt];
#pragma unroll
    for (int i = 0; i < 32 / kAt; ++i) src[i] = (const char*)__shfl_sync(0xffffffffu, (unsigned long long)row, i * kAt + lane / kPer);
    const uint32_t dst = tile + (c >> 3) * 128 * 128 + w * 32 * 128 + (lane / kPer) * 128;
#pragma unroll
    for (int i = 0; i < 32 / kAt; ++i) {
        const bool there = src[i] != nullptr && c * 8 < D;
        cp_async16(dst + i * kAt * 128 + (((c & 7) ^ ((i * kAt + lane / kPer) & 7)) << 4), there ? src[i] + c * 16 : any, there ? 16u : 0u);
    }
}

template <typename T, int HD, bool CAP, bool BIAS>
__global__ void __launch_bounds__(kTreeThreads, 1)
tree_kernel(const __grid_constant__ CacheParams p, const __grid_constant__ TreeSplit sp, int negate) {
    using L = TreeLayout<HD>;
    extern __shared__ char smem_raw[];
    const uint32_t smem = (smem_addr(smem_raw) + 1023u) & ~1023u;
    const uint32_t sm_q = smem, sm_ring = smem + 2 * L::kTileBytes, bars = sm_ring + L::kStages * L::kTileBytes;
    const uint32_t bar_s = bars, bar_p = bars + 16, bar_o = bars + 32, bar_qe = bars + 48, bar_full = bars + 64,
                   bar_empty = bar_full + 8 * L::kStages, slot = bar_empty + 8 * L::kStages;
    __shared__ unsigned s_valid[kInfo][4];                 // keys of a tile that are there
    __shared__ float s_at[BIAS ? kInfo : 1][kTreeKeys];    // their positions, from the first drafted token's on
    __shared__ float s_m[2][kTreeRows], s_l[2][kTreeRows]; // what the streams tell one another
    __shared__ unsigned s_odd[4][2];
    __shared__ TreeShare<kTreeThreads> share;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (tid == 0) {
        for (int t = 0; t < 2; ++t) {
            mbar_init(bar_s + 8 * t, 1);
            mbar_init(bar_p + 8 * t, 4);
            mbar_init(bar_o + 8 * t, 1);
            mbar_init(bar_qe + 8 * t, 1);
        }
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

    // With a bias the nearest keys, which lie last, come first: they have the large scores, and a row's reference point is
    // found once instead of moving with every tile.
    auto first_key = [](const TreeItem& it, int i) { return it.key0 + (BIAS ? it.tiles - 1 - i : i) * kTreeKeys; };
    // Ring entries of an item with n tiles, in the order in which the products take them:
    // K0 K1 V0 K2 V1 .. K(n-1) V(n-2) V(n-1); the query tile comes with K0.
    if (warp >= 12) {
        if (warp == 12 && elect_one()) {
            const uint32_t id_s = mma_desc<T>(kTreeKeys, false, negate != 0), id_o = mma_desc<T>(HD, true);
            int st = 0, ph = 0, pp[2] = { 0, 0 }, item = 0;
            bool ok = true;
            auto take = [&]() {
                const int at = st;
                if (!mbar_wait_bounded(bar_full + 8 * st, ph, p.err)) { ok = false; return 0; }
                tc_fence_after();
                if (++st == L::kStages) { st = 0; ph ^= 1; }
                return at;
            };
            TreeItem it;
            while (ok && walk.next(p, sp, it)) {
                if (it.tiles == 0) continue;
                auto score = [&](int i) {
                    const int e = take();
                    if (!ok) return;
                    mma_rows<HD>(tmem + (i & 1) * kTreeKeys, sm_q + (item & 1) * L::kTileBytes, sm_ring + e * L::kTileBytes, kTreeKeys, id_s);
                    mma_commit(bar_s + 8 * (i & 1));
                    mma_commit(bar_empty + 8 * e);
                    if (i + 1 == it.tiles) mma_commit(bar_qe + 8 * (item & 1));
                };
                score(0);
                if (it.tiles > 1 && ok) score(1);
                for (int i = 0; i < it.tiles && ok; ++i) {
                    const int t = i & 1, e = take();
                    if (!ok || !(ok = mbar_wait_bounded(bar_p + 8 * t, pp[t], p.err))) break;
                    pp[t] ^= 1;
                    tc_fence_after();
                    mma_weights<kTreeKeys>(tmem + 256 + t * HD, tmem + t * kTreeKeys, sm_ring + e * L::kTileBytes, id_o, i >= 2);
                    mma_commit(bar_o + 8 * t);
                    mma_commit(bar_empty + 8 * e);
                    if (i + 2 < it.tiles) score(i + 2);
                }
                ++item;
            }
        }
    } else if (warp >= 8) {
        const int w = warp - 8;
        int st = 0, ph = 1, item = 0, entries = 0, handed = 0, info = 0;
        bool ok = true;
        // an entry is handed over when its copies are there: kAhead entries after they were issued, or at once
        // where the products may need it before the next one can be issued
        auto hand_over = [&](int up_to) {
            fence_proxy_async();
            __syncwarp();
            for (; handed < up_to; ++handed)
                if (lane == 0) mbar_arrive(bar_full + 8 * (handed % L::kStages));
        };
        // Page numbers are asked for ahead of the rows they lead to: a tile's three tiles before, the next item's
        // first ones while this item's rows are copied.
        auto next_item = [&](TreeItem& it) {
            do {
                if (!walk.next(p, sp, it)) it.tiles = -1;
            } while (it.tiles == 0);
        };
        auto lookup = [&](const TreeItem& it, int i) {          // not looked at yet: nothing waits for it here
            const int j = first_key(it, i) + w * 32 + lane;
            return i < it.tiles && j < it.n + it.real ? table_entry(p.table, p.width, it.b, page_index(p.div, j)) : 0;
        };
        TreeItem it;
        next_item(it);
        int page[3] = { lookup(it, 0), lookup(it, 1), lookup(it, 2) };
        while (it.tiles > 0 && ok) {
            TreeItem then;
            next_item(then);
            const int after[3] = { lookup(then, 0), lookup(then, 1), lookup(then, 2) };
            auto entry = [&](int i, bool is_v, int pg) {
                const int j = first_key(it, i) + w * 32 + lane, key = j - page_index(p.div, j) * p.page_size;
                const char* src = nullptr;
                if (j < it.n + it.real && (pg = checked_page(pg, p.pages, p.err)) >= 0)
                    src = is_v ? (const char*)(row_of<T>(p.v, p.sv, 0, it.hk, key) + pg * p.sv[0])
                               : (const char*)(row_of<T>(p.k, p.sk, 0, it.hk, key) + pg * p.sk[0]);
                if (!mbar_wait_bounded(bar_empty + 8 * st, ph, p.err)) { ok = false; return; }
                if (i == 0 && !is_v) {
                    // this item's queries, where the last item's but one were: its products may still have to be begun
                    if (!__all_sync(0xffffffffu, mbar_try_wait(bar_qe + 8 * (item & 1), ((item >> 1) & 1) ^ 1))) {
                        cp_async_wait<0>();
                        hand_over(entries);
                    }
                    if (!mbar_wait_bounded(bar_qe + 8 * (item & 1), ((item >> 1) & 1) ^ 1, p.err)) { ok = false; return; }
                    const int r = it.row0 + w * 32 + lane;
                    const char* from = nullptr;
                    if (w * 32 + lane < it.rows)
                        from = (const char*)row_of<T>(p.q, p.sq, it.b, it.hk * p.group + r % p.group, r / p.group);
                    copy_rows<HD>(sm_q + (item & 1) * L::kTileBytes, w, lane, from, (const char*)p.q, p.D);
                }
                if (!is_v) {
                    const unsigned valid = __ballot_sync(0xffffffffu, src != nullptr);
                    if (lane == 0) s_valid[info][w] = valid;
                    if (BIAS) {
                        float pos = 0.0f;
                        if (src != nullptr)
                            pos = j >= it.n ? (float)depth_of(tokens_above(p, it.b, j - it.n)) : key_position(p, it.b, it.hk, j, first_position(p, it.b, it.n));
                        s_at[info][w * 32 + lane] = pos;
                    }
                    info = (info + 1) % kInfo;
                }
                copy_rows<HD>(sm_ring + st * L::kTileBytes, w, lane, src, is_v ? (const char*)p.v : (const char*)p.k, p.D);
                cp_async_commit();
                if (++st == L::kStages) { st = 0; ph ^= 1; }
                if (++entries - handed > L::kAhead) {
                    cp_async_wait<L::kAhead>();
                    hand_over(entries - L::kAhead);
                }
            };
            entry(0, false, page[0]);
            if (it.tiles > 1 && ok) entry(1, false, page[1]);
            for (int i = 0; i < it.tiles && ok; ++i) {
                const int more = lookup(it, i + 3);
                entry(i, true, page[0]);
                if (i + 2 < it.tiles && ok) entry(i + 2, false, page[2]);
                page[0] = page[1];
                page[1] = page[2];
                page[2] = more;
            }
            ++item;
            it = then;
            page[0] = after[0];
            page[1] = after[1];
            page[2] = after[2];
        }
        cp_async_wait<0>();
        if (ok) hand_over(entries);
    } else {
        const int tile = warp >> 2, quad = warp & 3, in_tile = quad * 32 + lane;
        const uint32_t lanes = (uint32_t)quad << 21, s_col = tmem + tile * kTreeKeys + lanes, o_col = tmem + 256 + tile * HD + lanes;
        ScoreConsts c;
        c.scale2 = positive_scale(p.sm_scale);
        c.cap_in = CAP ? 2.0f * fabsf(p.sm_scale) / p.cap : 0.0f;
        c.cap_out = CAP ? p.cap * kLog2e : 0.0f;
        const float unit = CAP ? c.cap_out : c.scale2;    // of what cap_scores, or the product, left: scores in base 2
        int done = 0, info = 0;           // key tiles of this stream, of the block, so far
        bool ok = true, again = false;
        TreeItem it;
        while (ok && walk.next(p, sp, it)) {
            const bool busy = quad * 32 < it.rows;        // this warp has rows
            const int gr = it.row0 + in_tile, t = gr / p.group, h = it.hk * p.group + gr % p.group;
            const bool valid = in_tile < it.rows, real = valid && t < it.real;
            unsigned long long above = real ? tokens_above(p, it.b, t) : 0ull;
            const float slope2 = BIAS && valid ? __ldg(p.slopes + h) * kLog2e : 0.0f;
            const float pos = BIAS && real ? (float)depth_of(above) : 0.0f;
            float m = kNegInf, l = 0.0f;
            int mine = 0;
            for (int i = tile; i < it.tiles; i += 2, ++mine) {
                if (!mbar_wait_bounded(bar_s + 8 * tile, (done + mine) & 1, p.err)) { ok = false; break; }
                tc_fence_after();
                if (busy) {
                    // 32 columns at a time, twice (for the maximum, for the weights): the code stays small, and with it the
                    // time that the two streams' warps wait for instructions
                    const int slot_i = (info + i) % kInfo, k0 = first_key(it, i);
                    const bool linear = BIAS && !p.positions && !p.start && k0 + kTreeKeys <= it.n;
                    float top = kNegInf;
#pragma unroll 1
                    for (int w = 0; w < 4; ++w) {
                        float s[32];
                        tmem_ld32(s_col + w * 32, s);
                        const int left = it.n - (k0 + w * 32);       // cached keys from this column on
                        const unsigned cached = left >= 32 ? ~0u : left > 0 ? (1u << left) - 1 : 0u;
                        const unsigned tree = left >= 32 ? 0u : left > 0 ? (unsigned)(above << left) : left > -64 ? (unsigned)(above >> -left) : 0u;
                        const unsigned see = real ? (cached | tree) & s_valid[slot_i][w] : 0u;
                        const bool whole = __all_sync(0xffffffffu, see == ~0u);
                        tmem_wait_ld();
                        if (CAP) cap_scores(s, c);
                        if (BIAS) {
                            // cached keys at their own numbers lie before every query that starts behind them
                            if (linear) {
                                add_bias(s, unit, slope2, pos - from_first(k0 + w * 32, it.n), true);
                            } else {
#pragma unroll
                                for (int x = 0; x < 32; ++x) s[x] = fmaf(-slope2, fabsf(pos - s_at[slot_i][w * 32 + x]), s[x] * unit);
                            }
                        }
                        if (!whole) {
#pragma unroll
                            for (int x = 0; x < 32; ++x) s[x] = see >> x & 1u ? s[x] : kNegInf;
                        }
                        if (CAP || BIAS || !whole) tmem_st32(s_col + w * 32, reinterpret_cast<const uint32_t*>(s));
                        float mx[4];
#pragma unroll
                        for (int x = 0; x < 4; ++x) mx[x] = s[x];
#pragma unroll
                        for (int x = 4; x < 32; ++x) mx[x & 3] = fmaxf(mx[x & 3], s[x]);
                        top = fmaxf(top, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
                    }
                    tmem_wait_st();
                    if (!BIAS) top *= unit;
                    const bool move = top > m + 8.0f || (m == kNegInf && top > kNegInf);
                    if (__any_sync(0xffffffffu, move)) {
                        const float f = move ? (m == kNegInf ? 0.0f : fast_exp2(m - top)) : 1.0f;
                        if (move) m = top;
                        l *= f;
                        if (mine > 0) {
                            if (!mbar_wait_bounded(bar_o + 8 * tile, (done + mine - 1) & 1, p.err)) { ok = false; break; }
                            tc_fence_after();
#pragma unroll 1
                            for (int x = 0; x < HD; x += 32) {
                                float o[32];
                                tmem_ld32(o_col + x, o);
                                tmem_wait_ld();
#pragma unroll
                                for (int y = 0; y < 32; ++y) o[y] *= f;
                                tmem_st32(o_col + x, reinterpret_cast<const uint32_t*>(o));
                            }
                        }
                    }
                    const float m0 = m == kNegInf ? 0.0f : m;
                    float2 sum[2] = { make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f) };
                    const float2 scale = make_float2(unit, unit), to = make_float2(-m0, -m0);
#pragma unroll 1
                    for (int w = 0; w < 4; ++w) {
                        float s[32];
                        uint32_t u[16];
                        tmem_ld32(s_col + w * 32, s);
                        tmem_wait_ld();
#pragma unroll
                        for (int y = 0; y < 32; y += 2) {
                            const float2 v = make_float2(s[y], s[y + 1]), a = BIAS ? add2(v, to) : fma2(v, scale, to);
                            const float2 e = make_float2(fast_exp2(a.x), fast_exp2(a.y));
                            sum[(y >> 1) & 1] = add2(sum[(y >> 1) & 1], e);
                            u[y / 2] = pack2<T>(e.x, e.y);
                        }
                        tmem_st16(s_col + w * 16, u);     // behind what has been read
                    }
                    l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                    tmem_wait_st();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_p + 8 * tile);
            }
            if (!ok) break;
            done += mine;
            info = (info + it.tiles) % kInfo;
            if (mine > 0 && !(ok = mbar_wait_bounded(bar_o + 8 * tile, (done - 1) & 1, p.err))) break;
            if (!busy) continue;                           // the same for a warp and its partner of the other stream
            tc_fence_after();
            // Both streams' results to the larger of the two reference points: the pair of warps that has the same rows
            // exchanges these, and takes a half of the columns each -- tensor memory has both accumulators.
            s_m[tile][in_tile] = m;
            s_l[tile][in_tile] = l;
            tc_fence_before();
            pair_barrier(1 + quad);
            tc_fence_after();
            const float m1 = s_m[tile ^ 1][in_tile], l1 = s_l[tile ^ 1][in_tile], top = fmaxf(m, m1), t0 = top == kNegInf ? 0.0f : top;
            const float f0 = fast_exp2(m - t0), f1 = fast_exp2(m1 - t0);
            // (in the order of the streams, so that both warps get the same)
            const float total = tile == 0 ? l * f0 + l1 * f1 : l1 * f1 + l * f0, inv = total != 0.0f ? 1.0f / total : 0.0f;
            const float lse = total != 0.0f ? t0 + log2f(total) : kNegInf;
            const float g0 = (tile == 0 ? f0 : f1) * inv, g1 = (tile == 0 ? f1 : f0) * inv;
            const long long row = ((long long)it.b * p.Hq + h) * p.T + t, part = (long long)it.part * sp.part_rows + in_tile;
            // a sum of 0 x over the results is NaN where one is not finite
            float nan0 = 0.0f * total, nan1 = 0.0f;
#pragma unroll 1
            for (int x = tile * (HD / 2); x < (tile + 1) * (HD / 2); x += 32) {
                float o[32] = {};
                if (it.tiles > 1) {
                    float z[32];
                    tmem_ld32(tmem + 256 + x + lanes, o);
                    tmem_ld32(tmem + 256 + HD + x + lanes, z);
                    tmem_wait_ld();
#pragma unroll
                    for (int y = 0; y < 32; ++y) o[y] = fmaf(o[y], g0, z[y] * g1);
                } else if (it.tiles > 0) {
                    tmem_ld32(tmem + 256 + x + lanes, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int y = 0; y < 32; ++y) o[y] *= g0;
                }
                if (inv == 0.0f) {
#pragma unroll
                    for (int y = 0; y < 32; ++y) o[y] = 0.0f;
                }
#pragma unroll
                for (int y = 0; y < 32; y += 2) {
                    nan0 = fmaf(o[y], 0.0f, nan0);
                    nan1 = fmaf(o[y + 1], 0.0f, nan1);
                }
                if (valid) {
#pragma unroll
                    for (int y = 0; y < 32; y += 8)
                        if (x + y < p.D) {
                            float v[8];
#pragma unroll
                            for (int z = 0; z < 8; ++z) v[z] = o[y + z];
                            if (it.part < 0) store8<T>((T*)p.out + row * p.D + x + y, v);
                            else if (in_range(part, sp.rows, p.err)) store8<float>(sp.part + part * p.D + x + y, v);
                        }
                }
            }
            if (tile == 0 && valid) {
                if (it.part < 0) p.lse[row] = lse;
                else if (in_range(part, sp.rows, p.err)) sp.part_lse[part] = lse;
            }
            // rows that something non-finite reached are marked by an lse of NaN, which no other row has, and done once more
            // behind the loop: the other roles wait for this warp here, with limits
            const float nan = nan0 + nan1;
            const unsigned odd = it.part < 0 ? __ballot_sync(0xffffffffu, valid && nan != nan) : 0u;
            if (lane == 0) s_odd[quad][tile] = odd;
            tc_fence_before();
            pair_barrier(1 + quad);                       // both have read the accumulators; then the next products may write them
            if (tile == 0) {
                const unsigned bad = s_odd[quad][0] | s_odd[quad][1];
                again = again || bad != 0u;
                if (bad >> lane & 1u) p.lse[row] = __int_as_float(0x7fffffff);
            }
        }
        if (ok && again) {
            walk = share.walk<TreeTile>();
            while (walk.next(p, sp, it)) {
                if (it.part >= 0) continue;               // tree_combine_kernel's
                const int gr = it.row0 + in_tile, t = gr / p.group, h = it.hk * p.group + gr % p.group;
                const bool valid = in_tile < it.rows;
                const float lse = valid ? p.lse[((long long)it.b * p.Hq + h) * p.T + t] : 0.0f;
                unsigned bad = __ballot_sync(0xffffffffu, lse != lse);
                while (bad) {                             // from the keys that the row sees alone
                    const int g = gr - lane + __ffs(bad) - 1;
                    bad &= bad - 1;
                    exact_row_tree<T>(p, it.b, it.hk * p.group + g % p.group, g / p.group);
                }
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 12) tmem_free(tmem, 512);
}

}  // namespace dsdpa
