"""Calls of the sequence operators at the ends of what their documentation allows, on every kernel that can take them:
rows from one to more than 128 to a key/value head, caches that one block goes through and caches that are cut."""
import copy
import math

import pytest
import torch

import ops
import sequence_ref as ref
from test_gpu_cache import Cache, as_int, check, random_tree

be = ops.backend
cabi = be.cabi
pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
# heads of a group and tokens: 1, 8, 12, 20, 64 and 160 rows
ROWS = [(1, 1), (2, 4), (4, 3), (4, 5), (1, 64), (4, 40)]


def present(c, b, n, T, table=None):
    """Numbers of sequence b's cached and drafted keys that lie in a page of its table."""
    table = c.table if table is None else table
    room = table.shape[1] * c.page
    return [j for j in range(min(n, room) + T) if j < room and 0 <= table[b, j // c.page].item() < c.k.shape[0]]


def among(c, q, b, n, keys, sm, table=None):
    """Results of sequence b's tokens (a chain) from those keys alone, the bounds, and p of [heads, T, keys]."""
    table = c.table if table is None else table
    n = min(n, table.shape[1] * c.page)
    T, g = q.shape[2], q.shape[1] // c.k.shape[1]
    at = torch.tensor(keys, dtype=torch.long, device="cuda")
    page = table[b].long()[at // c.page]
    k, v = (x[page, :, at % c.page].transpose(0, 1).repeat_interleave(g, 0)[None] for x in (c.k, c.v))
    seen = at[None, :] <= n + torch.arange(T, device="cuda")[:, None]
    res, tol = ref.attend(q[b][None], k, v, seen[None, None], (n + torch.arange(T, device="cuda")[:, None] - at).double()[None, None], sm)
    s = sm * q[b].double() @ k[0].double().transpose(-1, -2)
    p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
    return {x: t[0] for x, t in res.items()}, {x: t[0] for x, t in tol.items()}, p, at


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group,T", ROWS)
@pytest.mark.parametrize("pages", [4, 200])
def test_lengths_beyond_the_table(dtype, group, T, pages):
    """Drafted keys that the table has no room for, or a length that it cannot hold, with rows of weights that end where the
    table's room does: those keys are absent, the others are right, nobody else's weights change."""
    page, Hkv = 16, 2
    room = pages * page
    few = min(40, room - T)
    c = Cache([room - T, few, room - T], T, Hkv, 64, page, dtype, seed=T + pages)
    assert c.slots == room
    q = c.q(Hkv * group, T)
    lens = [room - T + (T + 1) // 2, few, room + 1000]
    out, lse = be.tree_sdpa(q, c.k, c.v, c.table, as_int(lens), 0.125)
    assert cabi.lib().dsdpa_device_error(0) == cabi.ERR_DEVICE_BOUNDS
    held = torch.rand(5, Hkv, room, generator=c.g, device="cuda")
    before = held.clone()
    be.cache_weights(held[1:4], q, lse, c.k, c.table, as_int(lens), 0.125)
    assert cabi.lib().dsdpa_device_error(0) == cabi.ERR_DEVICE_BOUNDS
    assert torch.equal(held[0], before[0]) and torch.equal(held[4], before[4])
    for b, n in enumerate(lens):
        keys = present(c, b, n, T)
        res, tol, p, at = among(c, q, b, n, keys, 0.125)
        ref.assert_within(out[b], res["out"], tol["out"], f"out of sequence {b}")
        ref.assert_within(lse[b], res["lse"], tol["lse"], f"lse of sequence {b}")
        add = p.view(Hkv, -1, *p.shape[-2:])
        err = (add * (2 * tol["lse"].view(Hkv, -1, T, 1) + 2.0 ** -19)).sum((1, 2))
        want = before[1 + b][:, at].double() + add.sum((1, 2))
        ref.assert_within(held[1 + b][:, at], want, err + (group * T + 2) * ref.E32 * want.abs(), f"weights of sequence {b}")
        other = torch.ones(room, dtype=torch.bool, device="cuda")
        other[at] = False
        assert torch.equal(held[1 + b][:, other], before[1 + b][:, other])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group,T", ROWS)
@pytest.mark.parametrize("B,n", [(3, 50), (170, 150), (3, 5000), (70, 2500)])
def test_non_finite_values_reach_the_rows_that_see_them_only(dtype, group, T, B, n):
    """More sequences than blocks and caches that are cut: a NaN in the last token's value and in one sequence's first value,
    and an infinity in a cached key's value of another sequence."""
    D, sm = 64, 0.125
    lens = [n + 7 * (b % 5) for b in range(B)]
    c = Cache(lens, T, 1, D, 32, dtype, seed=T + n)
    q = c.q(group, T)
    for b, m in enumerate(lens):
        if b % 3 != 2 or T == 1:
            at = m + T - 1
            c.v[c.table[b, at // 32].item(), :, at % 32] = math.nan
    c.v[c.table[1, 0].item(), :, 0, 3] = math.nan
    c.v[c.table[2, 1].item(), :, 1] = math.inf
    out, lse = be.tree_sdpa(q, c.k, c.v, c.table, c.lens, sm)
    for b, m in enumerate(lens):
        if b in (1, 2):
            bad = torch.zeros(D, dtype=torch.bool, device="cuda")
            bad[3 if b == 1 else slice(None)] = True
            assert not torch.isfinite(out[b, :, :, bad]).any()
            assert torch.isfinite(out[b, :, :T - 1, ~bad]).all()
        elif b % 3 != 2 or T == 1:
            assert torch.isnan(out[b, :, T - 1]).all()
    # the first sequences of the others, and the last one
    others = [b for b in range(B) if b not in (1, 2)]
    for b in others[:6] + others[-1:]:
        res, tol, _, _ = among(c, q, b, lens[b], list(range(lens[b] + T)), sm)
        ref.assert_within(lse[b], res["lse"], tol["lse"], f"lse of sequence {b}")
        if T > 1:
            rows = slice(0, T - 1) if b % 3 != 2 else slice(0, T)
            clean = copy.copy(c)
            clean.v = torch.nan_to_num(c.v, nan=0.0, posinf=0.0)
            res, tol, _, _ = among(clean, q, b, lens[b], list(range(lens[b] + T)), sm)
            ref.assert_within(out[b, :, rows], res["out"][:, rows], tol["out"][:, rows], f"out of sequence {b}")


def capped_bounds(cap, uncapped):
    """A capped form's results with bounds that have no term of the cap's own size: the scores' error is relative to them (the
    polynomial is good to 3 units of 2^-24, the general form, taken from 0.76 cap on, to 4), which is 8 E32 |y| of the 16 that
    the uncapped form's bound has.  For caps far above the scores the weights are the uncapped ones'."""
    return cap[0], uncapped[1]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("softcap", [2.0 ** 14, 1e6, 1e12])
@pytest.mark.parametrize("group,T", ROWS)
@pytest.mark.parametrize("n", [150, 3000])
def test_wide_caps_over_a_cache(dtype, softcap, group, T, n):
    """A cap far above the scores leaves them as they are, to their own rounding."""
    c = Cache([n, 40], T, 2, 64, 16, dtype, seed=T + n)
    q, sm = c.q(2 * group, T), 0.3
    out, lse = be.tree_sdpa(q, c.k, c.v, c.table, c.lens, sm, softcap=softcap)
    w = torch.zeros(2, 2, c.slots, device="cuda")
    be.cache_weights(w, q, lse, c.k, c.table, c.lens, sm, softcap=softcap)
    for b, m in enumerate([n, 40]):
        res, tol = capped_bounds(ref.tree_one(q[b], c.k, c.v, c.table[b], m, sm, softcap=softcap), ref.tree_one(q[b], c.k, c.v, c.table[b], m, sm))
        ref.assert_within(out[b], res["out"], tol["out"], "out")
        ref.assert_within(lse[b], res["lse"], tol["lse"], "lse")
        p = among(c, q, b, m, list(range(m + T)), sm)[2].view(2, -1, T, m + T)      # uncapped: off by (x / cap)^2 x / 3 < 1e-7
        want, err = p.sum((1, 2)), (p * (2 * tol["lse"].view(2, -1, T, 1) + 2.0 ** -19)).sum((1, 2))
        ref.assert_within(w[b, :, :m + T], want, err + (group * T + 2) * ref.E32 * want, "weights")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("causal", [False, True])
def test_one_score_above_a_wide_cap(dtype, D, causal):
    """One query's scores above the cap, the others' far below it: these keep the precision of their own size."""
    g = torch.Generator(device="cuda").manual_seed(D)
    q, k, v = (torch.randn(1, 2, 200, D, generator=g, device="cuda").to(dtype) for _ in range(3))
    q[:, :, 150] *= 4096
    cap, sm = 4096.0, 2 * D ** -0.5
    out, lse = be.masked_forward_raw(q, k, v, sm, causal=causal, softcap=cap)
    keep = [i for i in range(200) if i != 150]
    res, _ = ref.masked(q, k, v, sm, causal=causal, softcap=cap)
    _, tol = ref.masked(q, k, v, sm, causal=causal)
    for n, t in (("out", out), ("lse", lse)):
        ref.assert_within(t[:, :, keep], res[n][:, :, keep], tol[n][:, :, keep], n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("bias", [False, True])
def test_hidden_scores_above_the_cap_change_no_bit(dtype, D, bias):
    g = torch.Generator(device="cuda").manual_seed(D)
    q, k, v, do = (torch.randn(1, 2, 190, D, generator=g, device="cuda").to(dtype) for _ in range(4))
    kw = dict(causal=True, softcap=3.0, slopes=torch.tensor([0.1, 0.01], device="cuda") if bias else None)
    q *= 0.1

    def call():
        out, lse = be.masked_forward_raw(q, k, v, 0.2, **kw)
        return out, lse, be.masked_backward_raw(q, k, v, out, lse, do, 0.2, **kw)[0]
    want = call()
    for t in (q, k, v):
        t[:, :, 189] = 300.0                # the last token's key, which nobody else sees, and its own row
    for a, b in zip(call(), want):
        assert torch.equal(a[:, :, :189], b[:, :, :189])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group,T", ROWS[1:])
@pytest.mark.parametrize("n", [70, 3000])
def test_hidden_drafts_above_the_cap_change_no_bit(dtype, group, T, n):
    c = Cache([n], T, 1, 64, 16, dtype, seed=T)
    q = c.q(group, T) * 0.1
    take = torch.ones(1, T, dtype=torch.bool, device="cuda")
    take[:, -1] = False

    def call():
        out, lse = be.tree_sdpa(q, c.k, c.v, c.table, c.lens, 0.2, softcap=3.0)
        w = be.cache_weights(torch.zeros(1, 1, c.slots, device="cuda"), q, lse, c.k, c.table, c.lens, 0.2, softcap=3.0, take=take)
        return out[:, :, :-1], lse[:, :, :-1], w
    want = call()
    c.k[c.table[0, (n + T - 1) // 16].item(), :, (n + T - 1) % 16] = 300.0
    q[:, :, -1] = 300.0
    assert all(torch.equal(a, b) for a, b in zip(call(), want))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("where", ["dout", "dout element", "q", "out of nothing"])
@pytest.mark.parametrize("softcap", [0.0, 5.0])
def test_a_spoilt_query_spoils_what_it_sees_only(dtype, D, bad, where, softcap):
    """Documents, causal: one query whose gradient or row is not finite.  Its own dq and the keys that it sees are not finite,
    every other row is what it is without that query."""
    vis = be.visible_ranges([130, 100, 70], prefix=[20, 0, 0], device="cuda")
    g = torch.Generator(device="cuda").manual_seed(D)
    q, k, v, do = (torch.randn(1, h, 300, D, generator=g, device="cuda").to(dtype) for h in (4, 2, 2, 4))
    sm, at, head = D ** -0.5, 180, 1
    if where == "out of nothing":
        vis[at] = 0                                           # the spoilt query sees no key at all: nobody is reached
        do[0, head, at] = bad
    elif where == "dout element":
        do[0, head, at, 3] = bad
    elif where == "dout":
        do[0, head, at] = bad
    clean_q, clean_do = q.clone(), do.clone()
    if where == "q":
        q[0, head, at] = bad
    clean_do[0, head, at] = 0.0
    kw = dict(visible=vis, softcap=softcap)
    out, lse = be.masked_forward_raw(q, k, v, sm, **kw)
    dq, dk, dv = be.masked_backward_raw(q, k, v, out, lse, do, sm, **kw)
    res, tol = ref.masked(clean_q, k, v, sm, dout=clean_do, **kw)
    own = torch.zeros(1, 4, 300, dtype=torch.bool, device="cuda")
    own[0, head, at] = where != "out of nothing"
    # with a cap an infinite q gives scores of plus and minus the cap: a row like any other until its gradient
    rows = ~own
    for n, t in (("out", out), ("lse", lse), ("dq", dq)):
        ref.assert_within(t[rows], res[n][rows], tol[n][rows], n)
    seen = torch.zeros(1, 2, 300, dtype=torch.bool, device="cuda")
    if where != "out of nothing":
        seen[0, head // 2, vis[at, 0]:vis[at, 1]] = True
    for n, t in (("dk", dk), ("dv", dv)):
        ref.assert_within(t[~seen], res[n][~seen], tol[n][~seen], n)
    if where.startswith("dout"):
        assert not torch.isfinite(dk[seen]).any() and not torch.isfinite(dq[own]).any()
        assert not torch.isfinite(dv[seen][:, 3]).any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_an_infinite_value_spoils_one_column(dtype, D):
    g = torch.Generator(device="cuda").manual_seed(D)
    q, k, v, do = (torch.randn(1, h, 300, D, generator=g, device="cuda").to(dtype) for h in (4, 2, 2, 4))
    clean = v.clone()
    v[0, 1, 140, 5] = math.inf
    out, lse = be.masked_forward_raw(q, k, v, D ** -0.5, causal=True)
    res, tol = ref.masked(q, k, clean, D ** -0.5, causal=True)
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[0, 2:, 140:, 5] = True
    ref.assert_within(out[~bad], res["out"][~bad], tol["out"][~bad], "out")
    ref.assert_within(lse, res["lse"], tol["lse"], "lse")
    assert (out[bad] == math.inf).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("what", ["one row", "one element", "all of it", "an element of each row"])
def test_a_step_whose_loss_scale_overflowed_is_not_far_slower(dtype, what):
    """Infinite gradients are an everyday thing where a 16-bit loss is scaled: the pass is to take a few times a finite one's
    time, not hundreds of times it."""
    L = 4096 if dtype == torch.float16 else 2048
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v, do = (torch.randn(1, h, L, 64, generator=g, device="cuda").to(dtype) for h in (8, 2, 2, 8))
    out, lse = be.masked_forward_raw(q, k, v, 0.125, causal=True)

    def time():
        best = math.inf
        for _ in range(4):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            be.masked_backward_raw(q, k, v, out, lse, do, 0.125, causal=True)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        return best
    usual = time()
    if what == "one row":
        do[0, 3, L // 2] = math.inf
    elif what == "one element":
        do[0, 3, L // 2, 7] = math.inf
    elif what == "all of it":
        do.fill_(math.inf)
    else:
        do[..., 7] = math.inf
    assert time() < 40 * usual


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group,T", ROWS)
@pytest.mark.parametrize("n", [150, 3000])
@pytest.mark.parametrize("first", [0, 2 ** 30 + 1, 2 ** 31 - 1, -2 ** 31 + 5000])
def test_positions_far_from_zero(dtype, group, T, n, first):
    """Distances count, not positions: numbers that fp32 cannot tell apart, and ones next to the ends of int32."""
    c = Cache([n, 40], T, 2, 64, 16, dtype, seed=T + n)
    ago = torch.sort(torch.randint(0, 4000, (2, 2, c.slots), generator=c.g, device="cuda"), -1, descending=True).values
    positions = (first - ago).clamp_min(-2 ** 31).int()
    check(c, c.q(2 * group, T), 0.125, parents=random_tree(2, T, n) if T > 1 else None, positions=positions, start=[first, first - 1],
          slopes=torch.linspace(0.2, 0.001, 2 * group, device="cuda"))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
def test_weights_far_below_the_range_of_fp16(dtype, D):
    """Even weights of 277,309 keys, 60.5 of fp16's smallest steps each: dv is dout's sum over as many, to half a step of the
    weights and of the result."""
    Lk, Lq = 277309, 1024
    g = torch.Generator(device="cuda").manual_seed(D)
    q = torch.zeros(1, 1, Lq, D, dtype=dtype, device="cuda")
    k, v = (torch.randn(1, 1, Lk, D, generator=g, device="cuda").to(dtype) for _ in range(2))
    do = (torch.rand(1, 1, Lq, D, generator=g, device="cuda") + 1).mul(16).to(dtype)
    out, lse = be.masked_forward_raw(q, k, v, 0.125)
    dv = be.masked_backward_raw(q, k, v, out, lse, do, 0.125)[2]
    want = (do.double().sum(2, keepdim=True) / Lk).expand_as(dv)
    # lse is off by the sum of Lk weights (fp32, in groups of hundreds: 2^-20 is far above it) and a rounding near 18
    rel = 2 * ref.half_step(dtype) + 2.0 ** -20 + 18 * ref.E32 + (Lq + 8) * ref.E32
    ref.assert_within(dv, want, rel * want.abs(), "dv")


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("softcap", [0.0, 10.0])
def test_a_document_with_far_smaller_gradients_keeps_them(D, softcap):
    """fp16, two packed documents, the second one's dout 1e-5 of the first's: its gradients are those that it has alone, with the
    precision of the type.  dk's operand may round below the normal range: by half of fp16's smallest step at the scale of
    the key, which puts a bound of its row, 2 max |dout| |v|_1 + 2 max |delta|, between 2^13 and 2^14."""
    lens, sm = [150, 120], D ** -0.5
    vis = be.visible_ranges(lens, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(D)
    q, k, v, do = (torch.randn(1, h, 270, D, generator=g, device="cuda") for h in (4, 2, 2, 4))
    do[:, :, :150] *= 1000
    do[:, :, 150:] *= 0.01
    q, k, v, do = (t.half() for t in (q, k, v, do))
    kw = dict(softcap=softcap)
    out, lse = be.masked_forward_raw(q, k, v, sm, visible=vis, **kw)
    got = be.masked_backward_raw(q, k, v, out, lse, do, sm, visible=vis, **kw)
    for lo, hi in ((0, 150), (150, 270)):
        res, tol = ref.masked(*(t[:, :, lo:hi] for t in (q, k, v)), sm, causal=True, dout=do[:, :, lo:hi], **kw)
        most = do.double().abs().amax() * v[:, :, lo:hi].double().abs().sum(-1) + (out.double() * do.double()).sum(-1).abs().amax()
        tol["dk"] = tol["dk"] + sm * 2.0 ** -25 * (2 * most / 2.0 ** 13)[..., None] * q[:, :, lo:hi].double().abs().view(1, 2, 2, hi - lo, D).sum((2, 3))[:, :, None]
        for n, t in zip(("dq", "dk", "dv"), got):
            ref.assert_within(t[:, :, lo:hi], res[n], tol[n], f"{n} of the document from {lo} on")


def test_every_call_raises_what_the_device_recorded_where_that_is_asked_for(monkeypatch):
    c = Cache([40, 40], 2, 1, 64, 16, torch.bfloat16, seed=1)
    q, w = c.q(2, 2), torch.rand(2, 1, c.slots, device="cuda")
    out, lse = be.tree_sdpa(q, c.k, c.v, c.table, c.lens, 0.125)
    broken = c.table.clone()
    broken[1, 1] = -1
    monkeypatch.setattr(be.op, "check_device_errors", True)
    calls = [lambda t: be.tree_sdpa(q, c.k, c.v, t, c.lens, 0.125), lambda t: be.cache_weights(w, q, lse, c.k, t, c.lens, 0.125),
             lambda t: be.cache_evict(c.k.clone(), c.v.clone(), t, c.lens, w, 30)]
    for call in calls:
        call(c.table)
        with pytest.raises(cabi.DsdpaError, match="out of range"):
            call(broken)
        call(c.table)
    x = torch.randn(1, 2, 20, 64, device="cuda", requires_grad=True)
    be.masked_sdpa(x, x, x, causal=True).sum().backward()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group,T", ROWS)
@pytest.mark.parametrize("page,n", [(16, 100), (7, 100), (16, 3000), (64, 3001)])
def test_absent_pages(dtype, group, T, page, n):
    """Page numbers that are none, at the start, inside and at the end of a sequence: their keys count as absent, everywhere."""
    c = Cache([n, 50, n - 30], T, 2, 64, page, dtype, seed=T + n + page)
    q = c.q(2 * group, T)
    broken = c.table.clone()
    broken[0, 1], broken[0, (n + T - 1) // page], broken[2, 0] = -1, c.k.shape[0], 2 ** 31 - 1
    out, lse = be.tree_sdpa(q, c.k, c.v, broken, c.lens, 0.125)
    assert cabi.lib().dsdpa_device_error(0) == cabi.ERR_DEVICE_BOUNDS
    w = torch.rand(3, 2, c.slots, generator=c.g, device="cuda")
    before = w.clone()
    be.cache_weights(w, q, lse, c.k, broken, c.lens, 0.125)
    assert cabi.lib().dsdpa_device_error(0) == cabi.ERR_DEVICE_BOUNDS
    for b, m in enumerate(c.lens.tolist()):
        keys = present(c, b, m, T, broken)
        res, tol, p, at = among(c, q, b, m, keys, 0.125, broken)
        ref.assert_within(out[b], res["out"], tol["out"], f"out of sequence {b}")
        ref.assert_within(lse[b], res["lse"], tol["lse"], f"lse of sequence {b}")
        add = p.view(2, -1, *p.shape[-2:])
        want = before[b][:, at].double() + add.sum((1, 2))
        err = (add * (2 * tol["lse"].view(2, -1, T, 1) + 2.0 ** -19)).sum((1, 2))
        ref.assert_within(w[b][:, at], want, err + (group * T + 2) * ref.E32 * want, f"weights of sequence {b}")
        other = torch.ones(c.slots, dtype=torch.bool, device="cuda")
        other[at] = False
        assert torch.equal(w[b][:, other], before[b][:, other])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group,T", ROWS)
@pytest.mark.parametrize("n", [90, 3000])
def test_strides_of_pages_and_queries(dtype, group, T, n):
    """Keys and values interleaved in one pool, heads inside a slot, a wider table, queries of [B, T, heads, D] storage."""
    c = Cache([n, 33], T, 2, 64, 16, dtype, seed=T + n)
    q = c.q(2 * group, T)
    want = be.tree_sdpa(q, c.k, c.v, c.table, c.lens, 0.125)
    ww = be.cache_weights(torch.zeros(2, 2, c.slots, device="cuda"), q, want[1], c.k, c.table, c.lens, 0.125)
    both = torch.stack([c.k.transpose(1, 2), c.v.transpose(1, 2)], 1).contiguous()
    k, v = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    qt = q.transpose(1, 2).contiguous().transpose(1, 2)
    got = be.tree_sdpa(qt, k, v, c.table, c.lens, 0.125)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(be.cache_weights(torch.zeros(2, 2, c.slots, device="cuda"), qt, got[1], k, c.table, c.lens, 0.125), ww)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group,T", ROWS)
@pytest.mark.parametrize("longest", [200, 4000])
def test_graphs_of_trees(dtype, group, T, longest):
    """Lengths, trees, tables and queries change between the replays of two graphs that live side by side."""
    c = Cache([longest, 60, longest // 2], T, 2, 64, 16, dtype, seed=T)
    q, tree = c.q(2 * group, T), as_int(random_tree(3, T, 1))
    kw = dict(parents=tree if T > 1 else None, slopes=torch.full((2 * group,), 0.05, device="cuda"), softcap=20.0)
    w = torch.zeros(3, 2, c.slots, device="cuda")

    def step():
        out, lse = be.tree_sdpa(q, c.k, c.v, c.table, c.lens, 0.125, **kw)
        return out, lse, be.cache_weights(w, q, lse, c.k, c.table, c.lens, 0.125, **kw)
    step()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = step()
        graphs.append((graph, res))
    g = torch.Generator(device="cuda").manual_seed(2)
    for i, lens in enumerate([[longest, 60, 3], [0, 1, longest // 3], [longest - 1, 17, longest // 2]]):
        c.lens.copy_(torch.tensor(lens))
        tree.copy_(as_int(random_tree(3, T, 10 + i)))
        q.copy_(torch.randn(q.shape, generator=g, device="cuda"))
        c.table[0, :4] = c.table[0, :4].flip(0)
        for graph, (out, lse, _) in graphs:
            w.zero_()
            graph.replay()
            got = [t.clone() for t in (out, lse, w)]
            w.zero_()
            assert all(torch.equal(a, b) for a, b in zip(got, step()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group,T", ROWS)
def test_streams_at_once(dtype, group, T):
    c = Cache([3000, 900], T, 2, 64, 64, dtype, seed=T)
    qs = [c.q(2 * group, T) for _ in range(3)]

    def call(q):
        out, lse = be.tree_sdpa(q, c.k, c.v, c.table, c.lens, 0.125)
        return out, lse, be.cache_weights(torch.zeros(2, 2, c.slots, device="cuda"), q, lse, c.k, c.table, c.lens, 0.125)
    want = [call(q) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    got = [[] for _ in qs]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(qs[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i, runs in enumerate(got) for run in runs for a, b in zip(run, want[i]))


def test_far_pages_of_trees():
    """A pool of more than 2^31 elements under more than 16 rows."""
    Hkv, page, D, T = 2, 512, 128, 9
    pages = (1 << 31) // (Hkv * page * D) + 3
    k = torch.zeros(pages, Hkv, page, D, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    g = torch.Generator(device="cuda").manual_seed(3)
    for i in (0, pages - 1):
        k[i], v[i] = (torch.randn(Hkv, page, D, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    table, lens = as_int([[pages - 1, 0]]), as_int([700])
    q = torch.randn(1, 8, T, D, generator=g, device="cuda").to(torch.bfloat16)
    out, lse = be.tree_sdpa(q, k, v, table, lens, 0.1)
    res, tol = ref.tree_one(q[0], k, v, table[0], 700, 0.1)
    ref.assert_within(out[0], res["out"], tol["out"], "out")
    ref.assert_within(lse[0], res["lse"], tol["lse"], "lse")
    w = be.cache_weights(torch.zeros(1, Hkv, 2 * page, device="cuda"), q, lse, k, table, lens, 0.1)
    assert ((w.sum(-1) - 4 * T).abs() < 1e-3).all()


def few_key_bounds(q, k, v, do, sm, causal, cap, slopes):
    """dq, dk in 64 bits and their bounds where delta is the weighted mean of dp in fp32: as in sequence_ref.attend, but
    delta's own error is that of the weights, of the sums (N + 16 roundings of their terms) and of dp, with no rounding of out."""
    storage, (B, H, M, D), N, g = q.dtype, q.shape, k.shape[2], q.shape[1] // k.shape[1]
    u, e, a = ref.half_step(storage), ref.E32, abs(sm)
    x = dict(causal=causal, softcap=cap, slopes=slopes)
    res, tol = ref.masked(q, k, v, sm, dout=do, **x)
    seen = ref.seen_mask(B, M, N, causal, None, q.device)[:, None]
    dist = (torch.arange(M, device=q.device)[:, None] + (N - M) - torch.arange(N, device=q.device)).double().abs()
    q, do, k, v = q.double(), do.double(), k.double().repeat_interleave(g, 1), v.double().repeat_interleave(g, 1)
    s0 = sm * q @ k.transpose(-1, -2)
    y = cap * torch.tanh(s0 / cap) if cap else s0
    bias = slopes.double()[:, None, None] * dist if slopes is not None else torch.zeros_like(s0)
    off = (D + 4) * e * a * (q.abs() @ k.abs().transpose(-1, -2)) + 8 * e * ((y - bias).abs() + y.abs() + bias) + 8 * e * cap
    worst = 2 * torch.where(seen, off, torch.zeros_like(off)).amax(-1, keepdim=True)
    p = torch.softmax((y - bias).masked_fill(~seen, -math.inf), -1)
    dp = do @ v.transpose(-1, -2)
    c = dp - (p * dp).sum(-1, keepdim=True)
    slope = 1 - (y / cap) ** 2 if cap else torch.ones_like(y)
    err_dp = (D + 2) * e * (do.abs() @ v.abs().transpose(-1, -2))
    err_p = p * (2 * worst + 16 * e)
    err_delta = (p * (err_dp + (N + 16) * e * dp.abs()) + err_p * c.abs()).sum(-1, keepdim=True)
    ds = p * c * slope
    err_ds = p * (err_delta + err_dp + c.abs() * 16 * e) + err_p * c.abs() + (u + 4 * e) * ds.abs()
    if storage == torch.float16:
        err_ds = err_ds + torch.where(seen, 2.0 ** -22, 0.0) * do.abs().amax()
    dk = lambda z, w: a * (z.transpose(-1, -2) @ w).view(B, -1, g, N, D).sum(2)
    tol["dq"] = ref.stored(res["dq"], storage) + a * (err_ds @ k.abs() + (N + 4) * e * (ds.abs() @ k.abs()))
    tol["dk"] = ref.stored(res["dk"], storage) + dk(err_ds + (g * M + 4) * e * ds.abs(), q.abs())
    return res, tol


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [16, 64, 128, 256])
@pytest.mark.parametrize("Lq,Lk,causal", [(1, 1, True), (2, 2, True), (2, 2, False), (3, 3, True), (5, 4, False), (16, 16, True), (1, 64, False), (300, 2, False)])
@pytest.mark.parametrize("softcap,bias", [(0.0, False), (4.0, True)])
def test_gradients_of_rows_with_few_keys(dtype, D, Lq, Lk, causal, softcap, bias):
    """Rows with nearly all of their weight on one key: gradients are small differences of large numbers."""
    g = torch.Generator(device="cuda").manual_seed(D + Lq + Lk)
    q, k, v, do = (torch.randn(4, h, n, D, generator=g, device="cuda").to(dtype) for h, n in ((4, Lq), (2, Lk), (2, Lk), (4, Lq)))
    sm, slopes = 4 * D ** -0.5, torch.tensor([0.5, 0.1, 0.05, 0.01], device="cuda") if bias else None
    kw = dict(causal=causal, softcap=softcap, slopes=slopes)
    out, lse = be.masked_forward_raw(q, k, v, sm, **kw)
    dq, dk, dv = be.masked_backward_raw(q, k, v, out, lse, do, sm, **kw)
    res, tol = few_key_bounds(q, k, v, do, sm, causal, softcap, slopes)
    for n, t in (("dq", dq), ("dk", dk), ("dv", dv)):
        ref.assert_within(t, res[n], tol[n], n)
