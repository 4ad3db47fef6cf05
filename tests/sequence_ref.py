"""Plain 64-bit forms of the sequence-attention and cache operators, with how far a kernel's results may be off.

Every bound is elementwise and adds up what the arithmetic allows, u being half a step of the storage type and
e = 2^-24 half a step of fp32:
  * a result is rounded once to storage: u |result|, or half the type's smallest step (2^-25 for fp16) where
    that is more;
  * the weights p (and ds) are rounded to storage before they are multiplied with rows: u sum |p| |row|
    (not for fp32 storage);
  * a sum of n products in fp32 is off by at most n e sum |products|;
  * a score is off by ds = (D + 4) e |sm_scale| sum |q k| (products, scaling) + 8 e (|s| + bias) + 8 e cap (tanh, the
    rounding of the parts), which changes its weight by the factor 1 + 2 ds; exp2 and the final division
    add 8 e (exp2.approx is good to 2 units in the last place, and so is the reciprocal);
  * the backward takes delta = out.dout from the rounded out: u sum |out dout|, times p in ds, and products
    that went into delta and dp carry their own n e.
"""
import math

import torch

E32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def stored(x, dtype):
    """What rounding x to dtype may add."""
    return half_step(dtype) * x.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def seen_mask(B, Lq, Lk, causal, visible, device="cpu"):
    i = torch.arange(Lq, device=device)[:, None] + (Lk - Lq)
    j = torch.arange(Lk, device=device)[None, :]
    seen = torch.ones(B, Lq, Lk, dtype=torch.bool, device=device)
    if causal:
        seen &= j <= i
    if visible is not None:
        v = visible if visible.dim() == 3 else visible[None]
        seen &= (j >= v[..., :1]) & (j < v[..., 1:])
    return seen


def clean(x, used):
    """x with the rows that nothing sees set to zero: they may hold anything."""
    return torch.where(used[..., None], x.double(), torch.zeros((), dtype=torch.float64, device=x.device))


def attend(q, k, v, seen, dist, sm_scale, cap=0.0, slopes=None, dout=None, storage=None):
    """q [B,H,M,D], k and v [B,H,N,D] (a key head per query head), seen [B,1 or H,M,N], dist [..,M,N].
    Returns {"out", "lse"[, "dq", "dk", "dv"]} and the same keys' bounds."""
    storage = storage or q.dtype
    u = half_step(storage)
    narrow = 0.0 if storage == torch.float32 else u
    q, k, v = q.double(), k.double(), v.double()
    D, N, M = q.shape[-1], k.shape[-2], q.shape[-2]
    x = sm_scale * q @ k.transpose(-1, -2)
    off = (D + 4) * E32 * abs(sm_scale) * (q.abs() @ k.abs().transpose(-1, -2))
    y = cap * torch.tanh(x / cap) if cap > 0 else x
    s = y
    bias = torch.zeros((), dtype=torch.float64, device=q.device)
    if slopes is not None:
        bias = slopes.double()[:, None, None] * dist.abs()
        s = s - bias
    off = off + 8 * E32 * (s.abs() + y.abs() + bias.abs()) + 8 * E32 * cap
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    off = torch.where(seen, off, torch.zeros_like(off))
    lse = torch.logsumexp(s, -1)
    p = torch.where(seen, torch.exp(s - torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)[..., None]), torch.zeros_like(s))
    worst = 2 * off.amax(-1, keepdim=True) if N else torch.zeros_like(s[..., :0])
    worst = worst if N else torch.zeros(*s.shape[:-1], 1, dtype=s.dtype, device=s.device)
    out = p @ v
    av = p @ v.abs()
    res = {"out": out, "lse": lse / math.log(2.0)}
    # the weights' own error meets |v| twice: in the sum and, through the total, in the division
    tol = {"out": stored(out, storage) + (narrow + 2 * worst + (N + 16) * E32) * av,
           "lse": (worst[..., 0] + (N + 16) * E32) * 1.5 + 4 * E32 * torch.nan_to_num(res["lse"], neginf=0.0).abs()}
    if dout is None:
        return res, tol
    do = dout.double()
    dp = do @ v.transpose(-1, -2)
    delta = (out * do).sum(-1, keepdim=True)
    slope_y = 1.0 - (y / cap) ** 2 if cap > 0 else torch.ones_like(y)
    ds = p * (dp - delta) * slope_y
    # delta's and dp's own error, and the error of p and of the derivative of the cap
    err_delta = (u + D * E32) * (out.abs() * do.abs()).sum(-1, keepdim=True) + (tol["out"] * do.abs()).sum(-1, keepdim=True)
    err_dp = (D + 2) * E32 * (do.abs() @ v.abs().transpose(-1, -2))
    err_p = p * (2 * worst + 16 * E32)
    err_ds = p * (err_delta + err_dp + (dp - delta).abs() * 16 * E32) + err_p * (dp - delta).abs()
    dv = p.transpose(-1, -2) @ do
    dq, dk = sm_scale * ds @ k, sm_scale * ds.transpose(-1, -2) @ q
    err_ds = err_ds + (narrow + 4 * E32) * ds.abs()
    err_pr = err_p + narrow * p
    if storage == torch.float16:
        # values below fp16's normal range are off by half its smallest step: relative to 1 for p, and for ds to the
        # largest |dout| (the kernels scale by a power of two of it, up to a factor of 4)
        big = do.abs().amax(dim=(-1, -2), keepdim=True)
        err_pr = err_pr + torch.where(seen, 2.0 ** -24, 0.0)
        err_ds = err_ds + torch.where(seen, 2.0 ** -22, 0.0) * big
        tol["out"] = tol["out"] + 2.0 ** -24 * (seen.double() @ v.abs())
    a = abs(sm_scale)
    res |= {"dq": dq, "dk": dk, "dv": dv}
    tol |= {"dv": stored(dv, storage) + err_pr.transpose(-1, -2) @ do.abs() + M * E32 * (p.transpose(-1, -2) @ do.abs()),
            "dq": stored(dq, storage) + a * (err_ds @ k.abs() + (N + 4) * E32 * (ds.abs() @ k.abs())),
            "dk": stored(dk, storage) + a * (err_ds.transpose(-1, -2) @ q.abs() + (M + 4) * E32 * (ds.abs().transpose(-1, -2) @ q.abs()))}
    return res, tol


def masked(q, k, v, sm_scale, causal=False, visible=None, softcap=0.0, slopes=None, dout=None):
    """masked_sdpa in 64 bits; rows that nothing sees may hold anything."""
    B, Hq, Lq, D = q.shape
    Hkv, Lk = k.shape[1], k.shape[2]
    g = Hq // Hkv
    seen = seen_mask(B, Lq, Lk, causal, visible, q.device)
    dist = (torch.arange(Lq, device=q.device)[:, None] + (Lk - Lq) - torch.arange(Lk, device=q.device)).double()
    rows, cols = seen.any(-1)[:, None].expand(B, Hq, Lq), seen.any(-2)[:, None].expand(B, Hkv, Lk)
    storage = q.dtype
    qc, kc, vc = clean(q, rows), clean(k, cols), clean(v, cols)
    do = clean(dout, rows) if dout is not None else None
    res, tol = attend(qc, kc.repeat_interleave(g, 1), vc.repeat_interleave(g, 1), seen[:, None], dist, sm_scale, softcap, slopes, do, storage)
    if dout is not None:
        for n in ("dk", "dv"):
            extra = half_step(storage) + (g + 2) * E32
            res[n] = res[n].view(B, Hkv, g, Lk, D).sum(2)
            tol[n] = tol[n].view(B, Hkv, g, Lk, D).sum(2) + extra * res[n].abs()
    return res, tol


def rows_of(pages, table_row, n):
    """Keys 0 .. n-1 of a sequence: [heads, n, D]."""
    size = pages.shape[2]
    s = torch.arange(n, device=pages.device)
    return pages[table_row.long()[s // size], :, s % size].transpose(0, 1)


def tree_seen(parents, T, n):
    """[T, n + T] and the tokens' depths, from a list of parents (None: a chain)."""
    up = []
    for t in range(T):
        above = t - 1 if parents is None else parents[t]
        up.append(({t} | up[above]) if above >= 0 else {t})
    seen = torch.ones(T, n + T, dtype=torch.bool)
    for t in range(T):
        for s in range(T):
            seen[t, n + s] = s in up[t]
    return seen, torch.tensor([len(x) - 1 for x in up])


def tree_one(q, k_pages, v_pages, table_row, n, sm_scale, parents=None, drafted=None, softcap=0.0, slopes=None, positions=None, start=None):
    """One sequence of tree_sdpa: q [H, T, D].  Returns res, tol and p [H, real, n + real]."""
    H, T, D = q.shape
    real = T if drafted is None else max(0, min(T, drafted))
    Hkv = k_pages.shape[1]
    g = H // Hkv
    seen, depth = tree_seen(parents, T, n)
    seen, depth = seen[:real, :n + real].to(q.device), depth[:real].to(q.device)
    k, v = rows_of(k_pages, table_row, n + real), rows_of(v_pages, table_row, n + real)
    base = n if start is None else start
    at = base + depth
    key_at = torch.arange(n, device=q.device).expand(Hkv, n) if positions is None else positions[:, :n].long()
    key_at = torch.cat([key_at, at.expand(Hkv, real)], 1).repeat_interleave(g, 0)
    dist = (at[None, :, None] - key_at[:, None, :]).double()
    res, tol = attend(q[None, :, :real], k[None].repeat_interleave(g, 1), v[None].repeat_interleave(g, 1), seen[None, None], dist[None],
                      sm_scale, softcap, slopes)
    return {n_: t[0] for n_, t in res.items()}, {n_: t[0] for n_, t in tol.items()}


def evict_one(weights, n, keep, sinks, recent):
    """Kept key numbers of one (sequence, head), ascending; weights is a list of floats."""
    if n <= keep:
        return list(range(n))
    middle = list(range(sinks, n - recent))
    rank = {i: (-math.inf, 0) if math.isnan(weights[i]) else (weights[i], 1) for i in middle}
    middle.sort(key=lambda i: (-rank[i][1], -rank[i][0] if rank[i][1] else 0.0, i))
    return sorted(list(range(sinks)) + middle[:keep - sinks - recent] + list(range(n - recent, n)))


def assert_within(got, want, tol, what):
    got, want, tol = got.double(), want.double(), tol.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), f"{what}: infinities differ"
    d = torch.where(inf, torch.zeros_like(want), (got - want).abs())
    tol = torch.where(inf, torch.ones_like(tol), tol) + 1e-30
    assert torch.isfinite(d).all(), f"{what}: {(~torch.isfinite(d)).sum().item()} values are not finite"
    if d.numel():
        r = (d / tol).max().item()
        assert r <= 1.0, f"{what}: off by {r:.3g} times the bound (largest difference {d.max().item():.3g})"
