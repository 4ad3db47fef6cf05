"""tree_sdpa, cache_weights and cache_evict against their definitions, and the three together over a few steps."""
import math

import pytest
import torch

import ops
import sequence_ref as ref

be = ops.backend
pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


class Cache:
    def __init__(self, lens, T, Hkv, D, page, dtype, seed=0, spare=2, extra=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.per = [-(-(max(n, 0) + T) // page) for n in lens]
        total = sum(self.per) + spare
        self.k, self.v = (torch.randn(total, Hkv, page, D, generator=g, device="cuda").to(dtype) for _ in range(2))
        order = torch.randperm(total, generator=g, device="cuda").int()
        self.table = torch.full((len(lens), max(max(self.per), 1) + extra), -1, dtype=torch.int32, device="cuda")
        at = 0
        for b, n in enumerate(self.per):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.spare = order[at:]
        self.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.page, self.slots = page, self.table.shape[1] * page
        self.g = g

    def q(self, H, T):
        return torch.randn(len(self.lens), H, T, self.k.shape[3], generator=self.g, device="cuda").to(self.k.dtype)


def random_tree(B, T, seed):
    g = torch.Generator().manual_seed(seed)
    return [[-1] + [int(torch.randint(max(-1, t - 5), t, (1,), generator=g)) for t in range(1, T)] for _ in range(B)]


def as_int(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def check(c, q, sm, parents=None, drafted=None, positions=None, start=None, take=None, **kw):
    more = dict(kw, parents=None if parents is None else as_int(parents), drafted=None if drafted is None else as_int(drafted),
                positions=positions, start=None if start is None else as_int(start))
    out, lse = be.tree_sdpa(q, c.k, c.v, c.table, c.lens, sm, **more)
    w = torch.rand(len(c.lens), c.k.shape[1], c.slots, generator=c.g, device="cuda")
    before = w.clone()
    assert be.cache_weights(w, q, lse, c.k, c.table, c.lens, sm, take=take, **more) is w
    H, T = q.shape[1], q.shape[2]
    Hkv = c.k.shape[1]
    for b, n in enumerate(c.lens.tolist()):
        n = max(n, 0)
        real = T if drafted is None else max(0, min(T, drafted[b]))
        assert (out[b, :, real:] == 0).all() and (lse[b, :, real:] == -math.inf).all()
        assert torch.equal(w[b, :, n + real:], before[b, :, n + real:])
        if real == 0:
            assert torch.equal(w[b], before[b])
            continue
        res, tol = ref.tree_one(q[b], c.k, c.v, c.table[b], n, sm, None if parents is None else parents[b], real,
                                positions=None if positions is None else positions[b], start=None if start is None else start[b], **kw)
        ref.assert_within(out[b, :, :real], res["out"], tol["out"], f"out of sequence {b}")
        ref.assert_within(lse[b, :, :real], res["lse"], tol["lse"], f"lse of sequence {b}")
        # weights: p from scores off by the bound of lse (which adds up the scores' and the sum's), once from each side
        p = weights_of(q[b], c, b, n, real, sm, None if parents is None else parents[b], positions, start, kw)
        if take is not None:
            p = p * take[b, :real, None]
        add = p.view(Hkv, -1, p.shape[-2], p.shape[-1])
        err = (add * (2 * tol["lse"].view(Hkv, -1, real, 1) + 2.0 ** -19)).sum((1, 2))
        want = before[b, :, :n + real].double() + add.sum((1, 2))
        ref.assert_within(w[b, :, :n + real], want, err + (H // Hkv * T + 2) * ref.E32 * want.abs(), f"weights of sequence {b}")
    return out, lse


def weights_of(q, c, b, n, real, sm, parents, positions, start, kw):
    """p in 64 bits: a value of 1 in one column at a time, all at once, read off as the output."""
    D = n + real
    H, T = q.shape[0], q.shape[1]
    seen, depth = ref.tree_seen(parents, T, n)
    seen, depth = seen[:real, :D].cuda(), depth[:real].cuda()
    g = H // c.k.shape[1]
    k = ref.rows_of(c.k, c.table[b], D).double().repeat_interleave(g, 0)
    x = sm * q[:, :real].double() @ k.transpose(-1, -2)
    cap = kw.get("softcap", 0.0)
    s = cap * torch.tanh(x / cap) if cap else x
    if kw.get("slopes") is not None:
        base = n if start is None else start[b]
        at = base + depth
        key = torch.arange(n, device="cuda").expand(c.k.shape[1], n) if positions is None else positions[b][:, :n].long()
        key = torch.cat([key, at.expand(c.k.shape[1], real)], 1).repeat_interleave(g, 0)
        s = s - kw["slopes"].double()[:, None, None] * (at[None, :, None] - key[:, None]).abs()
    return torch.softmax(torch.where(seen, s, torch.full_like(s, -math.inf)), -1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [8, 32, 64, 72, 128, 256])
@pytest.mark.parametrize("T", [1, 5])
def test_types_and_head_dims(dtype, D, T):
    c = Cache([37, 1, 200], T, 2, D, 16, dtype, seed=D + T)
    check(c, c.q(4, T), D ** -0.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [1, 7, 16, 64, 256])
@pytest.mark.parametrize("Hq,Hkv,T", [(1, 1, 1), (8, 1, 3), (32, 4, 1), (6, 2, 64), (12, 12, 17)])
def test_pages_heads_and_tokens(dtype, page, Hq, Hkv, T):
    c = Cache([0, 63, 64, 300, 129], T, Hkv, 64, page, dtype, seed=page, extra=3)
    check(c, c.q(Hq, T), 0.125, parents=random_tree(5, T, page) if T > 1 else None)


@pytest.mark.parametrize("dtype", TYPES)
def test_cap_bias_positions_and_ragged_tokens(dtype):
    T, Hkv = 9, 2
    lens = [150, 0, 2000, 31, 600]
    c = Cache(lens, T, Hkv, 64, 32, dtype, seed=20)
    slopes = torch.tensor([0.5, 0.1, 0.02, 0.004], device="cuda")
    q, tree = c.q(4, T), random_tree(5, T, 21)
    check(c, q, 0.3, parents=tree, slopes=slopes)
    positions = torch.sort(torch.randint(0, 5000, (5, Hkv, c.slots), generator=c.g, device="cuda"), -1).values.int()
    check(c, q, 0.3, parents=tree, slopes=slopes, softcap=8.0, positions=positions, start=[5000, 7, 5003, 5001, 6000])
    check(c, q, 0.3, parents=tree, drafted=[9, 0, 4, 1, 12], softcap=8.0)
    take = torch.rand(5, T, generator=c.g, device="cuda") < 0.5
    check(c, q, -0.3, drafted=[3, 9, 0, -2, 7], slopes=slopes, take=take)


@pytest.mark.parametrize("dtype", TYPES)
def test_long_caches(dtype):
    """Split over many blocks, and lengths around the ends of the pieces."""
    c = Cache([9000, 1023, 1024, 1025, 4095], 2, 2, 64, 64, dtype, seed=22)
    check(c, c.q(8, 2), 0.125)
    c = Cache([20011], 1, 1, 128, 16, dtype, seed=23)
    check(c, c.q(4, 1), 0.088, softcap=30.0)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("dtype", TYPES)
def test_what_is_not_seen_may_hold_anything(dtype, bad):
    T = 6
    c = Cache([70, 128], T, 2, 64, 32, dtype, seed=24)
    q = c.q(4, T)
    tree = [[-1, 0, 0, 1, 2, -1]] * 2
    want = be.tree_sdpa(q, c.k, c.v, c.table, c.lens, 0.125, parents=as_int(tree))
    for b, n in enumerate([70, 128]):                       # behind the last key, in pages that are in use
        last = c.table[b, (n + T - 1) // 32].item()
        c.k[last, :, (n + T - 1) % 32 + 1:] = bad
        c.v[last, :, (n + T - 1) % 32 + 1:] = bad
    c.k[c.spare.long()], c.v[c.spare.long()] = bad, bad
    got = be.tree_sdpa(q, c.k, c.v, c.table, c.lens, 0.125, parents=as_int(tree))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for b, n in enumerate([70, 128]):                       # token 5, which only token 5 sees
        at = n + 5
        c.k[c.table[b, at // 32].item(), :, at % 32] = bad
        c.v[c.table[b, at // 32].item(), :, at % 32] = bad
    out, lse = be.tree_sdpa(q, c.k, c.v, c.table, c.lens, 0.125, parents=as_int(tree))
    for b, n in enumerate([70, 128]):
        res, tol = ref.tree_one(q[b, :, :5], c.k, c.v, c.table[b], n, 0.125, tree[b][:5])
        ref.assert_within(out[b, :, :5], res["out"], tol["out"], "out")
        ref.assert_within(lse[b, :, :5], res["lse"], tol["lse"], "lse")
    w = torch.zeros(2, 2, c.slots, device="cuda")
    take = torch.ones(2, T, dtype=torch.bool, device="cuda")
    take[:, 5] = False
    be.cache_weights(w, q, lse, c.k, c.table, c.lens, 0.125, parents=as_int(tree), take=take)
    assert torch.isfinite(w).all()
    # each of the five taken tokens' weights sum to one for each of the two heads of a group
    assert ((w.sum(-1) - 10).abs() < 1e-3).all()


def test_strided_pages_and_queries():
    c = Cache([90, 33], 3, 2, 64, 16, torch.bfloat16, seed=25)
    q = c.q(4, 3)
    want = be.tree_sdpa(q, c.k, c.v, c.table, c.lens, 0.125)
    both = torch.stack([c.k.transpose(1, 2), c.v.transpose(1, 2)], 1).contiguous()      # [pages, 2, page, heads, D]
    k, v = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    wide = torch.full((2, 9), 7777, dtype=torch.int32, device="cuda")
    wide[:, :c.table.shape[1]] = c.table
    qt = q.transpose(1, 2).contiguous().transpose(1, 2)
    got = be.tree_sdpa(qt, k, v, wide, c.lens, 0.125)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_far_pages():
    """A pool of more than 2^31 elements: offsets pass 32 bits."""
    Hkv, page, D = 2, 512, 128
    pages = (1 << 31) // (Hkv * page * D) + 3
    k = torch.zeros(pages, Hkv, page, D, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    g = torch.Generator(device="cuda").manual_seed(26)
    for i in (0, pages - 1):
        k[i], v[i] = (torch.randn(Hkv, page, D, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    table, lens = as_int([[pages - 1, 0]]), as_int([700])
    q = torch.randn(1, 4, 1, D, generator=g, device="cuda").to(torch.bfloat16)
    out, lse = be.tree_sdpa(q, k, v, table, lens, 0.1)
    res, tol = ref.tree_one(q[0], k, v, table[0], 700, 0.1)
    ref.assert_within(out[0], res["out"], tol["out"], "out")
    w = torch.rand(1, Hkv, 2 * page, generator=g, device="cuda")
    target = as_int([[pages - 2]])
    new_lens, kept, _ = be.cache_evict(k, v, table, lens, w, 100, out_table=target)
    for h in range(Hkv):
        want = ref.evict_one(w[0, h].tolist(), 700, 100, 0, 0)
        assert kept[0, h].tolist() == want
        assert torch.equal(k[pages - 2, h, :100], ref.rows_of(k, table[0], 700)[h, torch.tensor(want, device="cuda")])


def test_bad_pages_and_parents_are_left_out_and_reported():
    cabi = be.cabi
    c = Cache([40, 40], 2, 1, 64, 16, torch.bfloat16, seed=27)
    q = c.q(2, 2)
    want = be.tree_sdpa(q, c.k, c.v, c.table, c.lens, 0.125)
    cabi.check(cabi.lib().dsdpa_device_error(0))
    for page in (-1, c.k.shape[0], 2 ** 31 - 1):
        broken = c.table.clone()
        broken[1, 1] = page
        out, lse = be.tree_sdpa(q, c.k, c.v, broken, c.lens, 0.125)
        assert cabi.lib().dsdpa_device_error(0) == cabi.ERR_DEVICE_BOUNDS
        assert cabi.lib().dsdpa_device_error(0) == cabi.OK
        assert torch.equal(out[0], want[0][0]) and torch.isfinite(out).all()
        keys = [n for n in range(42) if n // 16 != 1]                    # keys of the page count as absent
        k = ref.rows_of(c.k, c.table[1], 42)[:, keys]
        v = ref.rows_of(c.v, c.table[1], 42)[:, keys]
        seen = ref.tree_seen(None, 2, 40)[0][:, keys].cuda()
        res, tol = ref.attend(q[1:2], k[None].expand(1, 2, -1, -1), v[None].expand(1, 2, -1, -1), seen[None, None], seen[None, None], 0.125)
        ref.assert_within(out[1:2], res["out"], tol["out"], "out")
        w = torch.zeros(2, 1, c.slots, device="cuda")
        be.cache_weights(w, q, lse, c.k, broken, c.lens, 0.125)
        assert cabi.lib().dsdpa_device_error(0) == cabi.ERR_DEVICE_BOUNDS
        assert (w[1, :, 16:32] == 0).all() and (w[0, :, :42] != 0).all()
        k0, v0 = c.k.clone(), c.v.clone()
        be.cache_evict(k0, v0, broken, c.lens, torch.rand(2, 1, c.slots, device="cuda"), 30)
        assert cabi.lib().dsdpa_device_error(0) == cabi.ERR_DEVICE_BOUNDS
    too_long = as_int([40, 1000])
    out, _ = be.tree_sdpa(q, c.k, c.v, c.table, too_long, 0.125)
    assert cabi.lib().dsdpa_device_error(0) == cabi.ERR_DEVICE_BOUNDS
    assert torch.equal(out[0], want[0][0])
    out, _ = be.tree_sdpa(q, c.k, c.v, c.table, c.lens, 0.125, parents=as_int([[-1, 0], [-1, 1]]))     # its own parent
    assert cabi.lib().dsdpa_device_error(0) == cabi.ERR_DEVICE_BOUNDS
    roots = be.tree_sdpa(q, c.k, c.v, c.table, c.lens, 0.125, parents=as_int([[-1, 0], [-1, -1]]))
    assert torch.equal(out, roots[0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [5, 9, 20])
def test_parents_behind_the_last_token_are_not_looked_at(dtype, T):
    c = Cache([40, 7, 90], T, 2, 64, 16, dtype, seed=31)
    tree = random_tree(3, T, 32)
    for row, real in zip(tree, (T, 3, 1)):
        row[real:] = [-7] * (T - real)
    be.cabi.check(be.cabi.lib().dsdpa_device_error(0))
    check(c, c.q(4, T), 0.125, parents=tree, drafted=[T, 3, 1], slopes=torch.full((4,), 0.1, device="cuda"))
    assert be.cabi.lib().dsdpa_device_error(0) == be.cabi.OK


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("keep,sinks,recent", [(1, 0, 0), (50, 4, 10), (50, 20, 30), (64, 0, 64), (300, 3, 7), (5000, 4, 4)])
def test_evict(dtype, in_place, keep, sinks, recent):
    lens = [0, 1, 50, 51, 301, 4500]
    Hkv = 3
    c = Cache(lens, 0, Hkv, 40 if dtype != torch.float32 else 8, 16, dtype, seed=keep, spare=6 * 300)
    w = torch.rand(6, Hkv, c.slots, generator=c.g, device="cuda")
    w = torch.where(w < 0.4, torch.zeros_like(w), (w * 64).floor() / 64)                 # many ties
    w[5, 0, 100:130] = math.nan
    w[5, 1, 200:210] = math.inf
    w[5, 2, :4500] = -w[5, 2, :4500]
    pos = torch.randint(0, 9999, w.shape, generator=c.g, device="cuda").int()
    k0, v0, w0 = c.k.clone(), c.v.clone(), w.clone()
    width = -(-min(keep, c.slots) // 16)
    table = None if in_place else c.spare[:6 * width].view(6, width)
    new_lens, kept, nw, npos = be.cache_evict(c.k, c.v, c.table, c.lens, w, keep, sinks=sinks, recent=recent, out_table=table, positions=pos)
    assert torch.equal(torch.nan_to_num(w, nan=9.0), torch.nan_to_num(w0, nan=9.0)) and c.lens.tolist() == lens
    assert new_lens.tolist() == [min(n, keep) for n in lens]
    to = c.table if in_place else table
    untouched = torch.ones(c.k.shape[:3], dtype=torch.bool, device="cuda")
    for b, n in enumerate(lens):
        for h in range(Hkv):
            want = ref.evict_one(w0[b, h].tolist(), n, keep, sinks, recent)
            m = len(want)
            assert kept[b, h].tolist() == want + [-1] * (keep - m), (b, h)
            src = torch.tensor(want, dtype=torch.long, device="cuda")
            assert torch.equal(nw[b, h, :m].nan_to_num(nan=9.0), w0[b, h, src].nan_to_num(nan=9.0)) and (nw[b, h, m:] == 0).all()
            assert torch.equal(npos[b, h, :m], pos[b, h, src]) and (npos[b, h, m:] == 0).all()
            if m == 0:
                continue
            i = torch.arange(m, device="cuda")
            page = to[b].long()[i // 16]
            untouched[page, h, i % 16] = False
            for now, old in ((c.k, k0), (c.v, v0)):
                assert torch.equal(now[page, h, i % 16], ref.rows_of(old, c.table[b], n)[h, src])
    for now, old in ((c.k, k0), (c.v, v0)):
        assert torch.equal(now[untouched], old[untouched])


def test_decoding_with_eviction():
    """What a server does: decode, add up weights, evict when the cache is full, decode on -- with the positions that the
    kept keys had -- against plain lists of keys per head."""
    torch.manual_seed(28)
    B, H, Hkv, D, page, keep = 2, 4, 2, 64, 16, 40
    dtype, g = torch.bfloat16, H // Hkv
    c = Cache([60, 47], 12, Hkv, D, page, dtype, seed=28)
    slopes = torch.tensor([0.3, 0.1, 0.03, 0.01], device="cuda")
    lens, start = c.lens.clone(), c.lens.clone()
    pos = torch.arange(c.slots, dtype=torch.int32, device="cuda").expand(B, Hkv, -1).contiguous()
    weights = torch.zeros(B, Hkv, c.slots, device="cuda")
    keys = [[ref.rows_of(c.k, c.table[b], n)[h].clone() for h in range(Hkv)] for b, n in enumerate(lens.tolist())]
    vals = [[ref.rows_of(c.v, c.table[b], n)[h].clone() for h in range(Hkv)] for b, n in enumerate(lens.tolist())]
    at = [[list(range(n)) for _ in range(Hkv)] for n in lens.tolist()]
    for step in range(6):
        new_k, new_v = (torch.randn(B, Hkv, D, generator=c.g, device="cuda").to(dtype) for _ in range(2))
        q = torch.randn(B, H, 1, D, generator=c.g, device="cuda").to(dtype)
        for b, n in enumerate(lens.tolist()):
            where = c.table[b, n // page].item()
            c.k[where, :, n % page], c.v[where, :, n % page] = new_k[b], new_v[b]
            pos[b, :, n] = start[b]
            for h in range(Hkv):
                keys[b][h] = torch.cat([keys[b][h], new_k[b, h][None]])
                vals[b][h] = torch.cat([vals[b][h], new_v[b, h][None]])
                at[b][h].append(start[b].item())
        kw = dict(slopes=slopes, positions=pos, start=start)
        out, lse = be.tree_sdpa(q, c.k, c.v, c.table, lens, 0.125, **kw)
        be.cache_weights(weights, q, lse, c.k, c.table, lens, 0.125, **kw)
        for b in range(B):
            for h in range(H):
                kk, vv = keys[b][h // g], vals[b][h // g]
                dist = (start[b].item() - torch.tensor(at[b][h // g], device="cuda")).double()
                seen = torch.ones(1, 1, 1, len(kk), dtype=torch.bool, device="cuda")
                res, tol = ref.attend(q[b, h][None, None], kk[None, None], vv[None, None], seen, dist[None, None, None], 0.125, slopes=slopes[h:h + 1])
                ref.assert_within(out[b, h][None, None], res["out"], tol["out"], f"step {step}")
        lens, start = lens + 1, start + 1
        if step in (1, 4):
            lens, kept, weights, pos = be.cache_evict(c.k, c.v, c.table, lens, weights, keep, sinks=2, recent=8, positions=pos)
            for b in range(B):
                for h in range(Hkv):
                    idx = kept[b, h][kept[b, h] >= 0].long()
                    keys[b][h], vals[b][h] = keys[b][h][idx], vals[b][h][idx]
                    at[b][h] = [at[b][h][i] for i in idx.tolist()]
            assert lens.tolist() == [keep, keep]


def test_drafted_tree_equals_its_paths():
    """Every drafted token's result is that of decoding its path token by token."""
    T, n, page = 10, 75, 16
    c = Cache([n], T, 2, 64, page, torch.float32, seed=29)
    tree = random_tree(1, T, 30)
    q = c.q(4, T)
    out, lse = be.tree_sdpa(q, c.k, c.v, c.table, c.lens, 0.125, parents=as_int(tree))
    for t in range(T):
        path, at = [t], tree[0][t]
        while at >= 0:
            path.insert(0, at)
            at = tree[0][at]
        k, v = c.k.clone(), c.v.clone()
        for i, u in enumerate(path):
            a, z = c.table[0, (n + u) // page].item(), c.table[0, (n + i) // page].item()
            k[z, :, (n + i) % page], v[z, :, (n + i) % page] = c.k[a, :, (n + u) % page], c.v[a, :, (n + u) % page]
        one, l1 = be.tree_sdpa(q[:, :, t:t + 1], k, v, c.table, as_int([n + len(path) - 1]), 0.125)
        # two fp32 results of one definition, sums in another order
        assert (one[:, :, 0] - out[:, :, t]).abs().max() < 1e-5 and (l1[:, :, 0] - lse[:, :, t]).abs().max() < 1e-5


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_graph_of_a_step(dtype):
    """Lengths, tables and weights change between replays; two graphs live side by side."""
    c = Cache([500, 60], 1, 2, 64, 16, dtype, seed=31, spare=80)
    q = c.q(4, 1)
    w = torch.zeros(2, 2, c.slots, device="cuda")
    target = c.spare[:2 * 8].view(2, 8)
    be.tree_sdpa(q, c.k, c.v, c.table, c.lens, 0.125)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, lse = be.tree_sdpa(q, c.k, c.v, c.table, c.lens, 0.125)
            be.cache_weights(w, q, lse, c.k, c.table, c.lens, 0.125)
            ev = be.cache_evict(c.k, c.v, c.table, c.lens, w, 100, recent=3, out_table=target)
        graphs.append((graph, out, lse, ev))
    for n in ([500, 60], [3, 59], [499, 0]):
        c.lens.copy_(torch.tensor(n))
        for graph, out, lse, ev in graphs:
            w.zero_()
            graph.replay()
        want = be.tree_sdpa(q, c.k, c.v, c.table, c.lens, 0.125)
        ww = be.cache_weights(torch.zeros_like(w), q, want[1], c.k, c.table, c.lens, 0.125)
        we = be.cache_evict(c.k.clone(), c.v.clone(), c.table, c.lens, ww, 100, recent=3, out_table=target)
        for graph, out, lse, ev in graphs:
            assert torch.equal(out, want[0]) and torch.equal(lse, want[1]) and torch.equal(w, ww)
            assert all(torch.equal(a, b) for a, b in zip(ev, we))


def test_two_streams_at_once():
    c = Cache([3000, 2000], 4, 2, 64, 64, torch.bfloat16, seed=32)
    qs = [c.q(8, 4) for _ in range(2)]
    want = [be.tree_sdpa(q, c.k, c.v, c.table, c.lens, 0.125) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(be.tree_sdpa(qs[i], c.k, c.v, c.table, c.lens, 0.125))
    torch.cuda.synchronize()
    for i in range(2):
        for out, lse in got[i]:
            assert torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1])


@pytest.mark.parametrize("D", [8, 32, 40, 64, 96, 128])
@pytest.mark.parametrize("page,Hq,Hkv,T", [(16, 2, 2, 1), (7, 4, 1, 1), (64, 3, 1, 2), (1, 2, 1, 4), (48, 8, 1, 1)])
def test_few_rows_in_fp32(D, page, Hq, Hkv, T):
    """Up to eight rows over caches that are shared out between warps."""
    c = Cache([700, 0, 31, 1025, 256, 5], T, Hkv, D, page, torch.float32, seed=D + page)
    tree = random_tree(6, T, page) if T > 1 else None
    check(c, c.q(Hq, T), D ** -0.5, parents=tree)
    slopes = torch.linspace(0.3, 0.01, Hq, device="cuda")
    positions = torch.sort(torch.randint(0, 3000, (6, Hkv, c.slots), generator=c.g, device="cuda"), -1).values.int()
    take = torch.rand(6, T, generator=c.g, device="cuda") < 0.5
    check(c, c.q(Hq, T), 2 * D ** -0.5, parents=tree, drafted=[T, 0, 1, T, 1, T], softcap=6.0, slopes=slopes, take=take)
    check(c, c.q(Hq, T), -D ** -0.5, parents=tree, slopes=slopes, positions=positions, start=[3000, 1, 3001, 3005, 2999, 3000])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,T", [(8, 1), (4, 4), (1, 13), (16, 1), (2, 9), (1, 64)])
def test_short_caches_with_every_number_of_rows(dtype, D, Hq, T):
    """One block goes through a short cache; its shared memory grows with the rows."""
    c = Cache([300, 17, 0, 440], T, 1, D, 32, dtype, seed=D + T)
    check(c, c.q(Hq, T), D ** -0.5, parents=random_tree(4, T, 5) if T > 1 else None)
