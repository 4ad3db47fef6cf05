"""Cases of the sequence-attention and key/value-cache operators: what is timed, and what their results are held to.

``listed()`` names the cases, ``draw()`` gives more of the same ranges, ``prepare()`` makes what a program holds before the
call, ``run()`` is one call: of the package's operators where ``own`` is true, else of their plain form in elementary
torch operations.  ``exact()`` restates the definitions in 64 bits.

Definitions (heads of a group g share a key/value head h; positions count from 0):

    x = sm_scale q.k        y = cap tanh(x / cap) where cap > 0, else x        s = y - slope |position(q) - position(k)|
    p = softmax(s) over the visible keys        out = p v        lse = log2 sum exp(s)
    a query that sees no key: out = 0, lse = -inf
"""
import math
import random

import torch

own = False

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_LOG2E = 1.4426950408889634


# ---- the cases ----------------------------------------------------------------------------------------------------
def _masked(name, dtype, B, Hq, Hkv, Lq, Lk, D, grad, causal=True, docs=0, prefix=0, pad=0.0, softcap=0.0, slopes=False):
    return dict(name=name, op="masked_sdpa", dtype=dtype, B=B, Hq=Hq, Hkv=Hkv, Lq=Lq, Lk=Lk, D=D, grad=grad, causal=causal,
                docs=docs, prefix=prefix, pad=pad, softcap=softcap, slopes=slopes)


def _cache(name, op, dtype, B, Hq, Hkv, T, D, longest, page, spread=0.5, softcap=0.0, slopes=False, keep=0, recent=0):
    return dict(name=name, op=op, dtype=dtype, B=B, Hq=Hq, Hkv=Hkv, T=T, D=D, longest=longest, page=page, spread=spread,
                softcap=softcap, slopes=slopes, keep=keep, recent=recent)


def listed():
    return [
        # one 14x14 feature map as a short sequence, forward only: a call whose time is its launch
        _masked("masked short forward", "bfloat16", 1, 16, 16, 196, 196, 32, False, causal=False),
        # training in 32 bits on the 88x32 feature map, an image prefix in front of causal text, scores capped
        _masked("masked fp32 prefix training", "float32", 1, 8, 8, 2816, 2816, 32, True, docs=1, prefix=700, softcap=30.0),
        # training on padded sequences of 28x28 image tokens and text, odd length, capped scores, heads of their own
        _masked("masked prefix training", "bfloat16", 4, 16, 16, 1571, 1571, 64, True, docs=1, prefix=784, pad=0.4, softcap=30.0),
        # training on packed documents, four query heads to a key head: the largest call
        _masked("masked document training", "bfloat16", 1, 32, 8, 8192, 8192, 128, True, docs=9),
        # a prompt's second piece against what came before it, with a bias by distance, forward only
        _masked("masked biased prompt", "float16", 2, 16, 4, 2048, 6101, 128, False, slopes=True),
        # one sequence, one token, a short cache: latency
        _cache("tree single token short", "tree_sdpa", "bfloat16", 1, 16, 16, 1, 64, 300, 16),
        # a full batch of sequences of all lengths, one token each: the cache is read once
        _cache("tree token batch", "tree_sdpa", "bfloat16", 64, 32, 8, 1, 128, 8192, 64, spread=1.0),
        # trees of drafted tokens over long caches, capped scores, a bias by distance, odd sizes
        _cache("tree drafted long", "tree_sdpa", "float16", 3, 32, 8, 29, 128, 65536, 32, softcap=50.0, slopes=True),
        # weights gathered while a batch decodes
        _cache("weights token batch", "cache_weights", "bfloat16", 64, 32, 8, 1, 128, 8192, 64, spread=1.0),
        # weights of the last tokens of a prompt, 32 bits
        _cache("weights window fp32", "cache_weights", "float32", 3, 8, 8, 17, 64, 2000, 16),
        # a small cache cut down to a quarter
        _cache("evict short fp32", "cache_evict", "float32", 2, 8, 8, 0, 32, 1001, 16, keep=257, recent=32),
        # long caches of many sequences cut down
        _cache("evict long", "cache_evict", "bfloat16", 16, 32, 8, 0, 128, 16384, 64, keep=4096, recent=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    op = rng.choice(["masked_sdpa", "masked_sdpa", "tree_sdpa", "tree_sdpa", "cache_weights", "cache_evict"])
    D = rng.choice([16, 32, 64, 64, 128, 128])
    Hkv = rng.choice([1, 2, 4, 8])
    Hq = Hkv * rng.choice([1, 2, 4])
    softcap = rng.choice([0.0, 0.0, 20.0, 50.0])
    slopes = rng.random() < 0.3
    if op == "masked_sdpa":
        grad = rng.random() < 0.6
        Lq = _log(rng, 1, 4096)
        Lk = Lq if grad or rng.random() < 0.5 else Lq + _log(rng, 1, 4096)
        docs = rng.choice([0, 1, 1, rng.randint(2, 7)]) if Lq == Lk else 0
        prefix = rng.randint(1, Lq) if docs and rng.random() < 0.6 else 0
        pad = round(rng.uniform(0.1, 0.6), 2) if docs == 1 else 0.0
        B = max(1, min(rng.randint(1, 6), (1 << 25) // (Lq * Lk * 2)))
        c = _masked("", dtype, B, Hq, Hkv, Lq, Lk, D, grad, causal=rng.random() < 0.7, docs=docs, prefix=prefix, pad=pad,
                    softcap=softcap, slopes=slopes)
    else:
        longest = _log(rng, 32, 16384)
        B = max(1, min(_log(rng, 1, 48), (1 << 21) // (longest * Hkv)))
        T = 0 if op == "cache_evict" else rng.choice([1, 1, rng.randint(2, 16), rng.randint(17, 64)])
        keep = _log(rng, 8, longest) if op == "cache_evict" else 0
        c = _cache("", op, dtype, B, Hq, Hkv, T, D, longest, rng.choice([8, 16, 32, 64, 128]), spread=round(rng.uniform(0.0, 1.0), 2),
                   softcap=softcap, slopes=slopes, keep=keep, recent=rng.randint(0, keep // 2) if keep else 0)
        if op == "cache_evict":
            c["softcap"], c["slopes"] = 0.0, False
    del c["name"]
    return c


# ---- what a case fixes, whatever the seed --------------------------------------------------------------------------
def _ranges(c):
    """The keys [lo, hi) that each query may see, as nested lists [B][Lq][2], or None where the case has no such mask."""
    if not c["docs"]:
        return None
    L, rows = c["Lq"], []
    for b in range(c["B"]):
        rng = random.Random(1000 * c["docs"] + 10 * b + L)
        used = L - int(L * c["pad"] * b / c["B"])          # rows behind it are padding: they see nothing
        cuts = sorted(rng.sample(range(1, used), min(c["docs"], used) - 1)) if used > 1 else []
        row = []
        for lo, end in zip([0] + cuts, cuts + [used]):
            # a document's first tokens (an image) see one another, the rest see what lies before them
            row += [[lo, end if not c["causal"] else min(end, max(i + 1, lo + c["prefix"]))] for i in range(lo, end)]
        rows.append(row + [[0, 0]] * (L - used))
    return rows


def _lens(c):
    rng = random.Random(c["longest"] + 7 * c["B"])
    return [c["longest"]] + [max(1, int(c["longest"] * (1.0 - c["spread"] * rng.random()))) for _ in range(c["B"] - 1)]


def _parents(c):
    """A tree of drafted tokens for each sequence: token t hangs under an earlier one, or (-1) under the cached text."""
    out = []
    for b in range(c["B"]):
        rng = random.Random(31 * b + c["T"])
        out.append([-1] + [rng.randint(max(-1, t - 6), t - 1) for t in range(1, c["T"])])
    return out


def _alibi(H, device):
    return torch.exp2(-8.0 * torch.arange(1, H + 1, device=device, dtype=torch.float32) / H)


# ---- inputs --------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = _TYPES[c["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev, dtype=torch.float32 if dt == torch.float32 else dt)

    st = {"case": c, "sm_scale": c["D"] ** -0.5, "slopes": _alibi(c["Hq"], dev) if c["slopes"] else None}
    if c["op"] == "masked_sdpa":
        st["q"] = normal(c["B"], c["Hq"], c["Lq"], c["D"])
        st["k"], st["v"] = normal(c["B"], c["Hkv"], c["Lk"], c["D"]), normal(c["B"], c["Hkv"], c["Lk"], c["D"])
        r = _ranges(c)
        st["visible"] = None if r is None else torch.tensor(r, dtype=torch.int32).to(dev)
        # with ranges the causal part is in them already (a prefix sees forward)
        st["causal"] = bool(c["causal"]) and r is None
        if c["grad"]:
            for n in "qkv":
                st[n].requires_grad_(True)
            st["dout"] = normal(c["B"], c["Hq"], c["Lq"], c["D"])
        return st
    lens, T, page = _lens(c), c["T"], c["page"]
    per = [-(-(n + T) // page) for n in lens]
    width = max(per)
    new = -(-c["keep"] // page) if c["op"] == "cache_evict" else 0        # pages that take the kept rows
    total = sum(per) + new * c["B"]
    order = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    table = torch.full((c["B"], width), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    st["page_table"], st["lens"] = table, torch.tensor(lens, dtype=torch.int32, device=dev)
    st["k_pages"] = normal(total, c["Hkv"], page, c["D"])
    slots = width * page
    if c["op"] == "cache_evict":
        st["v_pages"] = normal(total, c["Hkv"], page, c["D"])
        st["out_table"] = order[at:].view(c["B"], new).contiguous()
        # accumulated weights: a few heavy keys, many light ones, many that no query has looked at (ties)
        w = torch.rand(c["B"], c["Hkv"], slots, generator=g, device=dev)
        st["weights"] = torch.where(w < 0.3, torch.zeros_like(w), torch.pow(w, 12.0))
        return st
    st["q"] = normal(c["B"], c["Hq"], T, c["D"])
    st["parents"] = torch.tensor(_parents(c), dtype=torch.int32).to(dev) if T > 1 else None
    if c["op"] == "tree_sdpa":
        st["v_pages"] = normal(total, c["Hkv"], page, c["D"])
    else:
        st["weights"] = torch.zeros(c["B"], c["Hkv"], slots, device=dev)
        st["lse"] = torch.logsumexp(_tree_scores(st), -1) * _LOG2E
    return st


# ---- the plain forms -----------------------------------------------------------------------------------------------
def _capped(x, cap):
    return cap * torch.tanh(x / cap) if cap > 0 else x


def _shared(x, Hq):
    """Each key head once for every query head of its group."""
    return x.float().repeat_interleave(Hq // x.shape[1], dim=1)


def _plain_masked(st):
    c = st["case"]
    q, Hq, cap = st["q"].detach().float(), c["Hq"], c["softcap"]
    k, v = _shared(st["k"].detach(), Hq), _shared(st["v"].detach(), Hq)
    at = torch.arange(c["Lq"], device=q.device) + (c["Lk"] - c["Lq"])
    to = torch.arange(c["Lk"], device=q.device)
    seen = torch.ones(1, 1, c["Lq"], c["Lk"], dtype=torch.bool, device=q.device)
    if st["causal"]:
        seen = seen & (to <= at[:, None])
    if st["visible"] is not None:
        r = st["visible"][:, None, :, :, None]
        seen = seen & (to >= r[..., 0, :]) & (to < r[..., 1, :])
    s = _capped(torch.matmul(q, k.transpose(-1, -2)) * st["sm_scale"], cap)
    slope = (1.0 - (s / cap) ** 2).mul_(st["sm_scale"]) if cap > 0 and c["grad"] else st["sm_scale"]
    if st["slopes"] is not None:
        s = s - st["slopes"][:, None, None] * (at[:, None] - to).abs()
    s = s.masked_fill_(~seen, -math.inf)
    top = s.amax(-1, keepdim=True).clamp_min(-3.0e38)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(total.clamp_min(1e-38))
    out = torch.matmul(p, v)
    if not c["grad"]:
        return {"out": out.to(st["q"].dtype), "lse": ((top + total.log()) * _LOG2E).masked_fill(total == 0, -math.inf)[..., 0]}
    do = st["dout"].float()
    dv = torch.matmul(p.transpose(-1, -2), do)
    dp = torch.matmul(do, v.transpose(-1, -2))
    ds = dp.sub_((out * do).sum(-1, keepdim=True)).mul_(p).mul_(slope)
    dq, dk = torch.matmul(ds, k), torch.matmul(ds.transpose(-1, -2), q)
    dk, dv = (t.view(c["B"], c["Hkv"], -1, c["Lk"], c["D"]).sum(2) for t in (dk, dv))
    return {n: t.to(st["q"].dtype) for n, t in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv))}


def _rows(pages, table):
    """A paged cache as [B, heads, slots, ...]; slots of absent pages repeat page 0 and are masked by the callers."""
    x = pages[table.clamp_min(0).long()]
    x = x.transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[-1])


def _tree_scores(st):
    """s of every drafted token with every slot of its cache, -inf where it does not see it: [B, Hq, T, slots], fp32."""
    c, T = st["case"], st["case"]["T"]
    k = _shared(_rows(st["k_pages"], st["page_table"]), c["Hq"])
    s = _capped(torch.matmul(st["q"].float(), k.transpose(-1, -2)) * st["sm_scale"], c["softcap"])
    slot, n = torch.arange(k.shape[2], device=k.device), st["lens"].long()
    eye = torch.eye(T, device=k.device)
    own_token = torch.arange(T, device=k.device)
    up = eye.expand(c["B"], T, T) if st["parents"] is None else eye + (st["parents"].long()[:, :, None] == own_token).float()
    above = (torch.linalg.matrix_power(up.double(), T) > 0)                           # [B, T, T]: u is t or above t
    draft = slot - n[:, None]                                                        # [B, slots]
    seen_draft = above.gather(2, draft.clamp(0, T - 1)[:, None, :].expand(-1, T, -1)) & ((draft >= 0) & (draft < T))[:, None, :]
    seen = (draft < 0)[:, None, :] | seen_draft
    if st["slopes"] is not None:
        depth = above.sum(-1) - 1                                                    # tokens above t in its tree
        at = n[:, None] + depth
        to = torch.where(draft < 0, slot, n[:, None] + depth.gather(1, draft.clamp(0, T - 1)))
        s = s - st["slopes"][:, None, None] * (at[:, :, None] - to[:, None, :]).abs()[:, None]
    return s.masked_fill_(~seen[:, None], -math.inf)


def _plain_tree(st):
    s = _tree_scores(st)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.div_(total), _shared(_rows(st["v_pages"], st["page_table"]), st["case"]["Hq"]))
    return {"out": out.to(st["q"].dtype), "lse": ((top + total.log()) * _LOG2E)[..., 0]}


def _plain_weights(st):
    c = st["case"]
    p = torch.exp2(_tree_scores(st) * _LOG2E - st["lse"][..., None])
    st["weights"] += p.view(c["B"], c["Hkv"], -1, p.shape[-1]).sum(2)
    return {"weights": st["weights"]}


def _plain_evict(st):
    c, n, w = st["case"], st["lens"].long(), st["weights"]
    slot = torch.arange(w.shape[2], device=w.device)
    rank = torch.where((slot >= (n - c["recent"])[:, None])[:, None], math.inf, w)
    rank = torch.where((slot < n[:, None])[:, None], rank, -math.inf)
    heavy = rank.sort(dim=-1, descending=True, stable=True).indices[..., :c["keep"]]
    left = n.clamp_max(c["keep"])
    i = torch.arange(heavy.shape[2], device=w.device)
    valid = (i < left[:, None])[:, None]
    kept = torch.where(valid, heavy, w.shape[2]).sort(dim=-1).values
    src = kept.clamp_max(w.shape[2] - 1)
    new_w = torch.zeros_like(w)
    new_w[..., :heavy.shape[2]] = torch.where(valid, w.gather(2, src), 0.0)
    page = c["page"]
    b = torch.arange(c["B"], device=w.device)[:, None, None]
    h = torch.arange(c["Hkv"], device=w.device)[None, :, None]
    to = st["out_table"][:, i // page].long()[:, None]
    there = torch.where(valid, (to * c["Hkv"] + h) * page + i % page, -1).reshape(-1)
    here = ((st["page_table"][b, src // page].long() * c["Hkv"] + h) * page + src % page).reshape(-1)
    here, there = here[there >= 0], there[there >= 0]
    for_k, for_v = st["k_pages"].view(-1, c["D"]), st["v_pages"].view(-1, c["D"])
    for_k[there], for_v[there] = for_k[here], for_v[here]
    return {"lens": left.int(), "kept": torch.where(valid, kept, -1).int(), "weights": new_w, "k_pages": st["k_pages"], "v_pages": st["v_pages"]}


def run(state):
    st, c = state, state["case"]
    if own:
        return _own(st, c)
    return {"masked_sdpa": _plain_masked, "tree_sdpa": _plain_tree, "cache_weights": _plain_weights, "cache_evict": _plain_evict}[c["op"]](st)


def _own(st, c):
    from ops import backend as be
    if c["op"] == "masked_sdpa":
        more = dict(causal=st["causal"], visible=st["visible"], softcap=c["softcap"], slopes=st["slopes"])
        if not c["grad"]:
            out, lse = be.masked_forward_raw(st["q"], st["k"], st["v"], st["sm_scale"], **more)
            return {"out": out, "lse": lse}
        out = be.masked_sdpa(st["q"], st["k"], st["v"], st["sm_scale"], **more)
        dq, dk, dv = torch.autograd.grad(out, (st["q"], st["k"], st["v"]), st["dout"])
        return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}
    if c["op"] == "cache_evict":
        lens, kept, weights = be.cache_evict(st["k_pages"], st["v_pages"], st["page_table"], st["lens"], st["weights"], c["keep"],
                                             recent=c["recent"], out_table=st["out_table"])
        return {"lens": lens, "kept": kept, "weights": weights, "k_pages": st["k_pages"], "v_pages": st["v_pages"]}
    more = dict(parents=st["parents"], softcap=c["softcap"], slopes=st["slopes"])
    if c["op"] == "tree_sdpa":
        out, lse = be.tree_sdpa(st["q"], st["k_pages"], st["v_pages"], st["page_table"], st["lens"], st["sm_scale"], **more)
        return {"out": out, "lse": lse}
    be.cache_weights(st["weights"], st["q"], st["lse"], st["k_pages"], st["page_table"], st["lens"], st["sm_scale"], **more)
    return {"weights": st["weights"]}


# ---- what one pass cannot do without -------------------------------------------------------------------------------
def work(case):
    c = case
    e = 4 if c["dtype"] == "float32" else 2
    if c["op"] == "masked_sdpa":
        r = _ranges(c)
        if r is not None:
            pairs = sum(hi - lo for row in r for lo, hi in row)
        elif c["causal"]:
            pairs = c["B"] * sum(i + 1 + c["Lk"] - c["Lq"] for i in range(c["Lq"]))
        else:
            pairs = c["B"] * c["Lq"] * c["Lk"]
        nq, nk = c["B"] * c["Hq"] * c["Lq"] * c["D"], c["B"] * c["Hkv"] * c["Lk"] * c["D"]
        ranges = 0 if r is None else 8 * c["B"] * c["Lq"]
        # forward: q, k, v in, out (and lse) out; training adds dout in and dq, dk, dv out
        moved = (2 * nq + 2 * nk) * e + ranges + (0 if c["grad"] else 4 * c["B"] * c["Hq"] * c["Lq"])
        moved += (2 * nq + 2 * nk) * e if c["grad"] else 0
        return {"bytes": moved, "flops": (14 if c["grad"] else 4) * pairs * c["Hq"] * c["D"]}
    lens = _lens(c)
    if c["op"] == "cache_evict":
        rows = sum(min(n, c["keep"]) for n in lens) * c["Hkv"]
        return {"bytes": 4 * c["Hkv"] * sum(lens) + 4 * rows * c["D"] * e + 8 * rows, "flops": 0}
    keys = sum(n + c["T"] for n in lens) * c["Hkv"] * c["D"]
    pairs = sum(n * c["T"] + (c["T"] * (c["T"] + 1)) // 2 for n in lens)
    q = c["B"] * c["Hq"] * c["T"] * c["D"]
    if c["op"] == "tree_sdpa":
        return {"bytes": (2 * keys + 2 * q) * e + 4 * q // c["D"], "flops": 4 * pairs * c["Hq"] * c["D"]}
    return {"bytes": (keys + q) * e + 8 * keys // c["D"], "flops": 2 * pairs * c["Hq"] * c["D"]}


# ---- the definitions in 64 bits, head by head ----------------------------------------------------------------------
def _exact_head(x, seen, dist, cap, slope):
    y = cap * torch.tanh(x / cap) if cap > 0 else x
    s = y if slope is None else y - slope * dist
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    lse = torch.logsumexp(s, -1)
    p = torch.where(seen, torch.exp(s - torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)[:, None]), torch.zeros_like(s))
    return p, lse / math.log(2.0), y


def _exact_masked(st, c):
    q, k, v = (st[n].detach().double() for n in "qkv")
    dev, cap, group = q.device, c["softcap"], c["Hq"] // c["Hkv"]
    i = torch.arange(c["Lq"], device=dev)[:, None] + c["Lk"] - c["Lq"]
    j = torch.arange(c["Lk"], device=dev)[None, :]
    out, lse = torch.zeros_like(q), torch.zeros(q.shape[:3], dtype=torch.float64, device=dev)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b in range(c["B"]):
        seen = (j <= i) if st["causal"] else torch.ones(c["Lq"], c["Lk"], dtype=torch.bool, device=dev)
        if st["visible"] is not None:
            seen = seen & (j >= st["visible"][b, :, :1]) & (j < st["visible"][b, :, 1:])
        for h in range(c["Hq"]):
            n = h // group
            slope = None if st["slopes"] is None else st["slopes"][h].double()
            p, lse[b, h], y = _exact_head(q[b, h] @ k[b, n].T * st["sm_scale"], seen, (i - j).abs(), cap, slope)
            out[b, h] = p @ v[b, n]
            if c["grad"]:
                do = st["dout"][b, h].double()
                dv[b, n] += p.T @ do
                ds = p * (do @ v[b, n].T - (out[b, h] * do).sum(-1, keepdim=True))
                if cap > 0:
                    ds = ds * (1.0 - (y / cap) ** 2)
                dq[b, h] = ds @ k[b, n] * st["sm_scale"]
                dk[b, n] += ds.T @ q[b, h] * st["sm_scale"]
    return {"out": out, "dq": dq, "dk": dk, "dv": dv} if c["grad"] else {"out": out, "lse": lse}


def _exact_cache(st, c):
    q, group, cap, T = st["q"].double(), c["Hq"] // c["Hkv"], c["softcap"], c["T"]
    tree = _parents(c)
    out, lse = torch.zeros_like(q), torch.zeros(q.shape[:3], dtype=torch.float64, device=q.device)
    weights = torch.zeros(c["B"], c["Hkv"], st["page_table"].shape[1] * c["page"], dtype=torch.float64, device=q.device)
    for b, n in enumerate(_lens(c)):
        up = []
        for t in range(T):
            p = tree[b][t] if T > 1 else -1
            up.append(({t} | up[p]) if p >= 0 else {t})
        seen = torch.ones(T, n + T, dtype=torch.bool)
        for t in range(T):
            for u in range(T):
                seen[t, n + u] = u in up[t]
        depth = torch.tensor([len(u) - 1 for u in up], dtype=torch.float64)
        key_at = torch.cat([torch.arange(n, dtype=torch.float64), n + depth])
        dist = ((n + depth)[:, None] - key_at).abs().to(q.device)
        seen = seen.to(q.device)
        s = torch.arange(n + T, device=q.device)
        page, slot = st["page_table"][b].long()[s // c["page"]], s % c["page"]
        for h in range(c["Hq"]):
            k = st["k_pages"][page, h // group, slot].double()
            slope = None if st["slopes"] is None else st["slopes"][h].double()
            x = q[b, h] @ k.T * st["sm_scale"]
            p, lse[b, h], y = _exact_head(x, seen, dist, cap, slope)
            if c["op"] == "tree_sdpa":
                out[b, h] = p @ st["v_pages"][page, h // group, slot].double()
            else:
                # against the lse that the call is given, a float that was rounded
                p = p * torch.exp2(lse[b, h] - st["lse"][b, h].double())[:, None]
                weights[b, h // group, :n + T] += p.sum(0)
    return {"out": out, "lse": lse} if c["op"] == "tree_sdpa" else {"weights": weights}


def _exact_evict(st, c):
    keep, page = c["keep"], c["page"]
    w = st["weights"].cpu()
    kept = torch.full((c["B"], c["Hkv"], keep), -1, dtype=torch.int64)
    new_w = torch.zeros(w.shape, dtype=torch.float64)
    new_k, new_v = st["k_pages"].double(), st["v_pages"].double()
    for b, n in enumerate(_lens(c)):
        for h in range(c["Hkv"]):
            if n <= keep:
                chosen = torch.arange(n)
            else:
                first = n - c["recent"]
                order = torch.argsort(-w[b, h, :first].double(), stable=True)[:keep - c["recent"]]
                chosen = torch.cat([torch.sort(order).values, torch.arange(first, n)])
            m = len(chosen)
            kept[b, h, :m] = chosen
            new_w[b, h, :m] = w[b, h, chosen].double()
            i, src = torch.arange(m, device=new_k.device), chosen.to(new_k.device)
            a, z = st["page_table"][b].long()[src // page], st["out_table"][b].long()[i // page]
            new_k[z, h, i % page] = st["k_pages"][a, h, src % page].double()
            new_v[z, h, i % page] = st["v_pages"][a, h, src % page].double()
    dev = st["weights"].device
    return {"lens": st["lens"].long().clamp_max(keep), "kept": kept.to(dev), "weights": new_w.to(dev), "k_pages": new_k, "v_pages": new_v}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "masked_sdpa":
        return _exact_masked(st, case)
    return _exact_evict(st, case) if case["op"] == "cache_evict" else _exact_cache(st, case)
