"""masked_sdpa against its definition in 64 bits: types, head layouts, lengths, masks, strides; the bounds are
derived in sequence_ref.py."""
import math

import pytest
import torch

import ops
import sequence_ref as ref

be = ops.backend
pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(B, Hq, Hkv, Lq, Lk, D, dtype, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, k, v, do = (torch.randn(B, h, n, D, generator=g, device="cuda").mul(scale).to(dtype)
                   for h, n in ((Hq, Lq), (Hkv, Lk), (Hkv, Lk), (Hq, Lq)))
    return q, k, v, do


def alibi(H):
    return torch.exp2(-8.0 * torch.arange(1, H + 1, device="cuda", dtype=torch.float32) / H)


def check(q, k, v, do, sm, **kw):
    out, lse = be.masked_forward_raw(q, k, v, sm, **kw)
    dq, dk, dv = be.masked_backward_raw(q, k, v, out, lse, do, sm, **kw)
    res, tol = ref.masked(q, k, v, sm, dout=do, **kw)
    for n, t in (("out", out), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
        ref.assert_within(t, res[n], tol[n], n)
    return out, lse, dq, dk, dv


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [8, 16, 32, 64, 72, 128, 256])
@pytest.mark.parametrize("causal", [False, True])
def test_head_dims_and_types(dtype, D, causal):
    q, k, v, do = make(2, 4, 2, 150, 150, D, dtype, seed=D)
    check(q, k, v, do, D ** -0.5, causal=causal)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Lq,Lk", [(1, 1), (1, 300), (300, 1), (2, 129), (128, 128), (127, 257), (257, 127), (129, 640), (513, 513)])
@pytest.mark.parametrize("causal", [False, True])
def test_lengths(dtype, Lq, Lk, causal):
    q, k, v, do = make(1, 2, 1, Lq, Lk, 64, dtype, seed=Lq + Lk)
    check(q, k, v, do, 0.125, causal=causal)      # causal with Lq > Lk: the first queries see nothing


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (6, 2), (8, 1), (5, 5)])
def test_shared_heads(dtype, Hq, Hkv):
    q, k, v, do = make(3, Hq, Hkv, 77, 200, 64, dtype, seed=Hq)
    check(q, k, v, do, 0.125)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("softcap,bias", [(5.0, False), (0.0, True), (30.0, True)])
@pytest.mark.parametrize("D", [64, 128])
def test_cap_and_distance_bias(dtype, softcap, bias, D):
    q, k, v, do = make(2, 4, 2, 200, 333, D, dtype, seed=3)
    check(q, k, v, do, 3.0 * D ** -0.5, softcap=softcap, slopes=alibi(4) if bias else None, causal=softcap == 30.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sm", [0.0, -0.125, 2.0])
def test_scales(dtype, sm):
    q, k, v, do = make(1, 2, 2, 140, 140, 64, dtype, seed=4)
    check(q, k, v, do, sm, causal=True)
    check(q, k, v, do, sm, softcap=4.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_documents_prefixes_and_padding(dtype, D):
    lengths = [[100, 1, 130, 57], [300], [3, 200]]
    vis = be.visible_ranges(lengths, 317, prefix=[40, 250, 0], device="cuda")
    q, k, v, do = make(3, 4, 2, 317, 317, D, dtype, seed=5)
    out, lse, dq, dk, dv = check(q, k, v, do, D ** -0.5, visible=vis)
    for b, x in enumerate(lengths):
        n = sum(x)
        assert (out[b, :, n:] == 0).all() and (lse[b, :, n:] == -math.inf).all() and (dq[b, :, n:] == 0).all()
        assert (dk[b, :, n:] == 0).all() and (dv[b, :, n:] == 0).all()
    # the same ranges for every batch element, given once; and a window
    one = be.visible_ranges([150, 167], prefix=9, window=33, device="cuda")
    check(q, k, v, do, D ** -0.5, visible=one)
    check(q, k, v, do, D ** -0.5, visible=one[None].expand(3, -1, -1), softcap=20.0, slopes=alibi(4))


@pytest.mark.parametrize("dtype", TYPES)
def test_arbitrary_ranges(dtype):
    g = torch.Generator().manual_seed(6)
    lo = torch.randint(-5, 260, (2, 200, 1), generator=g)
    vis = torch.cat([lo, lo + torch.randint(-40, 150, (2, 200, 1), generator=g)], 2)
    vis[0, 3] = torch.tensor([-2 ** 31, 2 ** 31 - 1])
    vis[0, 4] = torch.tensor([2 ** 31 - 1, -2 ** 31])
    vis[1, 10:140] = 0                                       # a whole tile of rows that see nothing
    q, k, v, do = make(2, 2, 1, 200, 257, 64, dtype, seed=6)
    check(q, k, v, do, 0.125, visible=vis.int().cuda())
    check(q, k, v, do, 0.125, visible=vis.int().cuda(), causal=True)
    nothing = torch.zeros(2, 200, 2, dtype=torch.int32, device="cuda")
    for t in check(q, k, v, do, 0.125, visible=nothing):
        assert (t[torch.isfinite(t)] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("D", [64, 128])
def test_masked_places_may_hold_anything(dtype, bad, D):
    """Rows that nothing sees, and keys that a query does not see, hold NaN or infinity."""
    lengths, L = [[120, 60], [150]], 200
    vis = be.visible_ranges(lengths, L, device="cuda")
    q, k, v, do = make(2, 4, 2, L, L, D, dtype, seed=7)
    res, tol = ref.masked(q, k, v, D ** -0.5, visible=vis, dout=do)
    for b, x in enumerate(lengths):
        for t in (q, k, v, do):
            t[b, :, sum(x):] = bad
    check(q, k, v, do, D ** -0.5, visible=vis)
    # the last token's key and value spoil its own row only
    q, k, v, do = make(1, 2, 1, 200, 200, D, dtype, seed=8)
    k[:, :, 199], v[:, :, 199] = bad, bad
    out, lse = be.masked_forward_raw(q, k, v, 0.125, causal=True)
    res, tol = ref.masked(q[:, :, :199], k[:, :, :199], v[:, :, :199], 0.125, causal=True)
    ref.assert_within(out[:, :, :199], res["out"], tol["out"], "out")
    ref.assert_within(lse[:, :, :199], res["lse"], tol["lse"], "lse")
    if not (bad == -math.inf):
        assert not torch.isfinite(out[:, :, 199]).all()
    dq, dk, dv = be.masked_backward_raw(q, k, v, out, lse, do, 0.125, causal=True)
    assert torch.isfinite(dq[:, :, :199]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_inputs(dtype):
    """[B, L, heads, D] storage, a slice of fused projections, and layouts that have to be copied."""
    B, H, L, D = 2, 4, 150, 64
    g = torch.Generator(device="cuda").manual_seed(9)
    qkv = torch.randn(B, L, 3, H, D, generator=g, device="cuda").to(dtype)
    q, k, v = (qkv[:, :, n].transpose(1, 2) for n in range(3))
    do = torch.randn(B, L, H, D, generator=g, device="cuda").to(dtype).transpose(1, 2)
    out = check(q, k, v, do, 0.125, causal=True)[0]
    same = be.masked_forward_raw(q.contiguous(), k.contiguous(), v.contiguous(), 0.125, causal=True)[0]
    assert torch.equal(out, same)
    odd = torch.randn(B, H, L, D + 1, generator=g, device="cuda").to(dtype)[..., 1:]      # rows off any 16-byte boundary
    check(odd, k, v, do, 0.125)
    check(q, k[:, :1].expand(-1, 2, -1, -1), v[:1, :1].expand(2, 2, -1, -1), do, 0.125)     # broadcast heads and batch
    turned = torch.randn(B, H, D, L, generator=g, device="cuda").to(dtype).transpose(2, 3)
    check(turned, k, v, do, 0.125)


@pytest.mark.parametrize("dtype", TYPES)
def test_autograd(dtype):
    q, k, v, do = make(1, 4, 2, 90, 120, 64, dtype, seed=10)
    for t in (q, k, v):
        t.requires_grad_(True)
    kw = dict(causal=True, softcap=10.0, slopes=alibi(4))
    out = be.masked_sdpa(q, k, v, 0.125, **kw)
    out.backward(do)
    res, tol = ref.masked(q.detach(), k.detach(), v.detach(), 0.125, dout=do, **kw)
    for n, t in (("out", out), ("dq", q.grad), ("dk", k.grad), ("dv", v.grad)):
        ref.assert_within(t.detach(), res[n], tol[n], n)
    # a broadcast leaf gets the sum over its copies: torch adds four rounded results, three more roundings
    kv = torch.randn(1, 1, 120, 64, device="cuda", dtype=dtype, requires_grad=True)
    be.masked_sdpa(q.detach(), kv.expand(1, 4, -1, -1), v.detach()[:, :1].expand(1, 4, -1, -1), 0.125).backward(do)
    res, tol = ref.masked(q.detach(), kv.detach().expand(1, 4, -1, -1), v.detach()[:, :1].expand(1, 4, -1, -1), 0.125, dout=do)
    ref.assert_within(kv.grad[:, 0], res["dk"].sum(1), tol["dk"].sum(1) + 3 * ref.half_step(dtype) * res["dk"].abs().sum(1), "broadcast dk")
    with pytest.raises(RuntimeError):
        o = be.masked_sdpa(q, k, v, 0.125)
        g, = torch.autograd.grad(o, q, do, create_graph=True)
        g.sum().backward()


def ref_close(a, b, rel):
    return ((a.double() - b.double()).abs().max() <= rel * b.double().abs().max()).item()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_against_differences(dtype):
    """Central differences of sum(out dout) along random directions, in 32-bit storage; for bf16 the same inputs
    rounded, against the fp32 kernels' gradient (off by the roundings of p, ds and the results)."""
    kw = dict(causal=True, softcap=6.0, slopes=alibi(2))
    q, k, v, do = (t.to(dtype).float() for t in make(1, 2, 1, 70, 70, 32, torch.float32, seed=11))
    out, lse = be.masked_forward_raw(q, k, v, 0.3, **kw)
    grads = be.masked_backward_raw(q, k, v, out, lse, do, 0.3, **kw)
    if dtype is torch.bfloat16:
        low = [t.to(dtype) for t in (q, k, v)]
        o, l = be.masked_forward_raw(*low, 0.3, **kw)
        for a, b in zip(be.masked_backward_raw(*low, o, l, do.to(dtype), 0.3, **kw), grads):
            assert ref_close(a, b, 8 * ref.half_step(dtype))
        return
    g = torch.Generator(device="cuda").manual_seed(12)
    for n in range(3):
        x = [q, k, v]
        d = torch.randn(x[n].shape, generator=g, device="cuda")
        h = 2.0 ** -7

        def loss(step):
            y = [t.double() for t in x]
            y[n] = y[n] + step * d.double()
            return (ref.masked(*[t for t in y], 0.3, **kw)[0]["out"] * do.double()).sum().item()
        # fourth-order differences of the 64-bit form: their own error is about h^4 times a fifth derivative
        diff = (8 * (loss(h) - loss(-h)) - (loss(2 * h) - loss(-2 * h))) / (12 * h)
        want = (grads[n].double() * d.double()).sum().item()
        size = (grads[n].double() * d.double()).abs().sum().item()
        assert abs(diff - want) <= 1e-4 * size


@pytest.mark.parametrize("dtype", TYPES)
def test_two_runs_are_the_same_bits(dtype):
    q, k, v, do = make(2, 8, 2, 300, 300, 64, dtype, seed=13)
    kw = dict(causal=True, softcap=20.0)
    a = be.masked_forward_raw(q, k, v, 0.125, **kw)
    b = be.masked_forward_raw(q, k, v, 0.125, **kw)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    a, b = (be.masked_backward_raw(q, k, v, *a, do, 0.125, **kw) for _ in range(2))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_empty_calls():
    q, k, v, do = make(1, 2, 1, 5, 0, 64, torch.bfloat16)
    out, lse = be.masked_forward_raw(q, k, v)
    assert (out == 0).all() and (lse == -math.inf).all()
    dq, dk, dv = be.masked_backward_raw(q, k, v, out, lse, do)
    assert (dq == 0).all() and dk.shape == k.shape
    q, k, v, do = make(1, 2, 1, 0, 5, 64, torch.bfloat16)
    out, lse = be.masked_forward_raw(q, k, v)
    dq, dk, dv = be.masked_backward_raw(q, k, v, out, lse, do)
    assert out.shape == q.shape and (dk == 0).all() and (dv == 0).all()
    q, k, v, do = make(0, 2, 1, 5, 5, 64, torch.bfloat16)
    out, lse = be.masked_forward_raw(q, k, v)
    assert [t.shape for t in be.masked_backward_raw(q, k, v, out, lse, do)] == [q.shape, k.shape, v.shape]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_side_stream_and_graph(dtype):
    q, k, v, do = make(1, 4, 2, 260, 260, 64, dtype, seed=14)
    want = be.masked_forward_raw(q, k, v, 0.125, causal=True)
    grads = be.masked_backward_raw(q, k, v, *want, do, 0.125, causal=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = be.masked_forward_raw(q, k, v, 0.125, causal=True)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = be.masked_forward_raw(q, k, v, 0.125, causal=True)
        more = be.masked_backward_raw(q, k, v, out, lse, do, 0.125, causal=True)
    for t in (q, k, v, do):
        t.mul_(0.5)
    graph.replay()
    new = be.masked_forward_raw(q, k, v, 0.125, causal=True)
    assert torch.equal(out, new[0]) and torch.equal(lse, new[1])
    again = be.masked_backward_raw(q, k, v, *new, do, 0.125, causal=True)
    assert all(torch.equal(a, b) for a, b in zip(more, again))
    assert not torch.equal(again[0], grads[0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", [1e-4, 200.0])
def test_small_and_large_gradients(dtype, size):
    """A loss that is scaled far up or down: ds leaves the range of fp16 before the results do."""
    q, k, v, do = make(1, 2, 1, 200, 200, 64, dtype, seed=15)
    do = (do.float() * size).to(dtype)
    check(q, k, v, do, 0.125, causal=True)


def test_long_rows_keep_their_precision():
    """Far keys with a steep bias, and a row whose maximum moves late."""
    q, k, v, do = make(1, 1, 1, 4, 9001, 64, torch.bfloat16, seed=16)
    k[:, :, -1] *= 4
    check(q, k, v, do, 0.5, slopes=torch.tensor([0.01], device="cuda"))
    check(q, k, v, do, 0.5, causal=True)


def test_threads_of_their_own():
    """A thread whose first CUDA call this is (an autograd engine starts such threads), all memory coming from the cache."""
    import threading
    q, k, v, do = make(1, 2, 1, 200, 200, 64, torch.float16, seed=17)
    want = be.masked_forward_raw(q, k, v, 0.125, causal=True)
    grads = be.masked_backward_raw(q, k, v, *want, do, 0.125, causal=True)
    for _ in range(3):
        [t.clone() for t in (q, k, v, do, *want)]
    torch.cuda.synchronize()
    got = []

    def work():
        try:
            out = be.masked_forward_raw(q, k, v, 0.125, causal=True)
            got.append((out, be.masked_backward_raw(q, k, v, *out, do, 0.125, causal=True)))
        except Exception as e:
            got.append(e)
    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert len(got) == 4
    for g in got:
        assert not isinstance(g, Exception), g
        assert all(torch.equal(a, b) for a, b in zip(g[0] + g[1], want + grads))


def test_no_query_heads():
    q, k, v, do = make(1, 0, 2, 5, 7, 64, torch.bfloat16)
    out, lse = be.masked_forward_raw(q, k, v)
    dq, dk, dv = be.masked_backward_raw(q, k, v, out, lse, do)
    assert out.shape == dq.shape == q.shape and (dk == 0).all() and (dv == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_without_gradients_the_same_result(dtype):
    q, k, v, _ = make(2, 4, 2, 130, 130, 32, dtype, seed=18)
    out = be.masked_sdpa(q, k, v, causal=True, softcap=20.0)
    assert not out.requires_grad
    leaf = q.clone().requires_grad_()
    with torch.no_grad():
        quiet = be.masked_sdpa(leaf, k, v, causal=True, softcap=20.0)
    loud = be.masked_sdpa(leaf, k, v, causal=True, softcap=20.0)
    assert not quiet.requires_grad and loud.requires_grad
    assert torch.equal(out, quiet) and torch.equal(out, loud)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scale", [0.05, 3.0], ids=["below the cap", "above the cap"])
@pytest.mark.parametrize("causal", [False, True])
def test_caps_over_whole_and_cut_tiles(dtype, scale, causal):
    """Scores on either side of the cap, over key tiles that every row of a query tile sees and over ones that some do not."""
    q, k, v, do = make(1, 2, 1, 390, 650, 64, dtype, seed=19)
    check(q, k, v, do, scale, causal=causal, softcap=4.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_steep_bias_over_many_tiles(dtype):
    """Nearest keys first: every row's maximum is in its first tile, which a window may have taken away."""
    q, k, v, do = make(1, 2, 1, 300, 1500, 64, dtype, seed=20)
    slopes = torch.tensor([0.25, 0.002], device="cuda")
    check(q, k, v, do, 0.125, causal=True, slopes=slopes)
    i = torch.arange(300, device="cuda", dtype=torch.int32)
    visible = torch.stack([torch.zeros_like(i), (i * 5 - 200).clamp(min=0)], -1)
    check(q, k, v, do, 0.125, slopes=slopes, visible=visible, softcap=3.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_step_in_a_graph(dtype):
    """Forward and backward through autograd, captured once and replayed with other inputs."""
    q, k, v, do = make(1, 4, 2, 150, 150, 64, dtype, seed=21)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]

    def step():
        out = be.masked_sdpa(*leaves, causal=True, softcap=10.0)
        return (out.detach(), *torch.autograd.grad(out, leaves, do))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.no_grad():
        for t in leaves:
            t.mul_(0.5)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, step()))
