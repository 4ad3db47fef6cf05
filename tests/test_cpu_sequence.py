"""Host side of the sequence-attention and cache operators: the C structs, the argument checks that answer before any CUDA
call, the refusals of the Python front end, and the ranges that visible_ranges makes."""
import ctypes
import re
from pathlib import Path

import pytest
import torch

import ops
import sequence_ref as ref

be = ops.backend
cabi = be.cabi
HEADER = (Path(__file__).resolve().parent.parent / "include" / "dsdpa.h").read_text()


def struct_fields(name):
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), HEADER, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    out = []
    for decl in body.split(";"):
        decl = decl.strip()
        if not decl:
            continue
        names = re.sub(r"^(const )?(unsigned char|long long|unsigned|int|float|void)\s*\*?", "", decl)
        out += [re.sub(r"\[.*\]", "", n).strip(" *") for n in names.split(",")]
    return out


@pytest.mark.parametrize("name,mirror,size", [("dsdpa_masked_problem", cabi.MaskedProblem, 40 + 24 * 8 + 8),
                                              ("dsdpa_cache_problem", cabi.CacheProblem, 56 + 72), ("dsdpa_cache_tree", cabi.CacheTree, 40)])
def test_structs_match_the_header(name, mirror, size):
    assert struct_fields(name) == [f[0] for f in mirror._fields_]
    assert ctypes.sizeof(mirror) == size


def test_packed_problems_are_the_structs():
    """The front end packs the structs instead of filling their mirrors."""
    n = [f[0] for f in cabi.MaskedProblem._fields_]
    got = cabi.MaskedProblem.from_buffer_copy(be.masked._PROBLEM.pack(*range(1, 11), *range(100, 125)))
    assert be.masked._PROBLEM.size == ctypes.sizeof(cabi.MaskedProblem)
    assert [getattr(got, x) for x in n[:10]] == list(range(1, 11))
    assert [v for x in n[10:18] for v in getattr(got, x)] + [got.stride_visible] == list(range(100, 125))
    n = [f[0] for f in cabi.CacheProblem._fields_]
    got = cabi.CacheProblem.from_buffer_copy(be.cache._PROBLEM.pack(*range(1, 14), *range(100, 109)))
    assert be.cache._PROBLEM.size == ctypes.sizeof(cabi.CacheProblem)
    assert [getattr(got, x) for x in n[:13]] == list(range(1, 14))
    assert [v for x in n[13:] for v in getattr(got, x)] == list(range(100, 109))


def masked_problem(**kw):
    base = dict(B=1, Hq=4, Hkv=2, Lq=10, Lk=12, D=64, sm_scale=0.125, softcap=0.0, dtype=cabi.BF16, flags=0)
    base.update(kw)
    p = cabi.MaskedProblem(*[base[f[0]] for f in cabi.MaskedProblem._fields_[:10]])
    for n in ("q", "k", "v", "out", "dout", "dq", "dk", "dv"):
        setattr(p, "stride_" + n, (ctypes.c_longlong * 3)(12 * 64 * 4, 12 * 64, 64))
    return p


OK = ctypes.c_void_p(4096)
ODD = ctypes.c_void_p(4100)


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=3), cabi.ERR_BAD_DTYPE), (dict(D=12), cabi.ERR_BAD_HEAD_DIM), (dict(D=0), cabi.ERR_BAD_HEAD_DIM), (dict(D=264), cabi.ERR_BAD_HEAD_DIM),
    (dict(B=0), cabi.ERR_BAD_SHAPE), (dict(Hq=5), cabi.ERR_BAD_SHAPE), (dict(Hkv=0), cabi.ERR_BAD_SHAPE), (dict(Lq=-1), cabi.ERR_BAD_SHAPE),
    (dict(Lk=(1 << 24) + 1), cabi.ERR_BAD_SHAPE), (dict(flags=2), cabi.ERR_BAD_FLAGS), (dict(sm_scale=float("inf")), cabi.ERR_BAD_SHAPE),
    (dict(softcap=float("nan")), cabi.ERR_BAD_SHAPE)])
def test_bad_masked_problems(kw, status):
    L, p = cabi.lib(), masked_problem(**kw)
    assert L.dsdpa_masked_forward(ctypes.byref(p), *[OK] * 7, 0, None) == status
    assert L.dsdpa_masked_backward(ctypes.byref(p), *[OK] * 12, 1 << 30, 0, None) == status
    assert L.dsdpa_masked_backward_workspace_bytes(ctypes.byref(p)) == 0


def test_masked_pointers():
    L, p = cabi.lib(), masked_problem()
    fwd = [OK, OK, OK, None, None, OK, OK]
    for i in (0, 1, 2, 5, 6):
        a = list(fwd)
        a[i] = None
        assert L.dsdpa_masked_forward(ctypes.byref(p), *a, 0, None) == cabi.ERR_NULL_POINTER
    for i in (0, 1, 2, 5):
        a = list(fwd)
        a[i] = ODD
        assert L.dsdpa_masked_forward(ctypes.byref(p), *a, 0, None) == cabi.ERR_MISALIGNED
    assert L.dsdpa_masked_forward(ctypes.byref(p), OK, OK, OK, ODD, None, OK, OK, 0, None) == cabi.ERR_MISALIGNED
    p.stride_k = (ctypes.c_longlong * 3)(12 * 64 * 4, 12 * 64, 63)
    assert L.dsdpa_masked_forward(ctypes.byref(p), *fwd, 0, None) == cabi.ERR_MISALIGNED
    p = masked_problem()
    need = L.dsdpa_masked_backward_workspace_bytes(ctypes.byref(p))
    assert need > 0
    bwd = [OK, OK, OK, None, None, OK, OK, OK, OK, OK, OK]
    assert L.dsdpa_masked_backward(ctypes.byref(p), *bwd, OK, need - 1, 0, None) == cabi.ERR_WORKSPACE
    assert L.dsdpa_masked_backward(ctypes.byref(p), *bwd, None, need, 0, None) == cabi.ERR_WORKSPACE
    assert L.dsdpa_masked_forward(None, *fwd, 0, None) == cabi.ERR_NULL_POINTER
    # nothing to do: no CUDA call
    assert L.dsdpa_masked_forward(ctypes.byref(masked_problem(Lq=0)), *[None] * 7, 0, None) == cabi.OK


def cache_problem(**kw):
    base = dict(B=2, Hq=4, Hkv=2, T=3, D=64, pages=9, page_size=16, table_width=4, slots=64, sm_scale=0.125, softcap=0.0, dtype=cabi.F16, flags=0)
    base.update(kw)
    p = cabi.CacheProblem(*[base[f[0]] for f in cabi.CacheProblem._fields_[:13]])
    for n in ("q", "k", "v"):
        setattr(p, "stride_" + n, (ctypes.c_longlong * 3)(2 * 16 * 64, 16 * 64, 64))
    return p


def tree_status(p, tree=None, ptrs=None):
    return cabi.lib().dsdpa_tree_forward(ctypes.byref(p), ctypes.byref(tree) if tree else None, *(ptrs or [OK] * 8), 1 << 40, 0, None)


def weights_status(p, tree=None, ptrs=None):
    return cabi.lib().dsdpa_cache_weights(ctypes.byref(p), ctypes.byref(tree) if tree else None, *(ptrs or [OK] * 7), 0, None)


def evict_status(p, keep=20, sinks=1, recent=2, out_width=4, ptrs=None, more=(OK, OK, ctypes.c_void_p(8192), None)):
    return cabi.lib().dsdpa_cache_evict(ctypes.byref(p), *(ptrs or [OK, OK, OK, OK, OK, None]), keep, sinks, recent, OK, out_width, *more, 0, None)


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=-1), cabi.ERR_BAD_DTYPE), (dict(D=4), cabi.ERR_BAD_HEAD_DIM), (dict(B=0), cabi.ERR_BAD_SHAPE), (dict(pages=0), cabi.ERR_BAD_SHAPE),
    (dict(page_size=0), cabi.ERR_BAD_SHAPE), (dict(table_width=0), cabi.ERR_BAD_SHAPE), (dict(table_width=1 << 27), cabi.ERR_BAD_SHAPE), (dict(flags=1), cabi.ERR_BAD_FLAGS)])
def test_bad_cache_problems(kw, status):
    p = cache_problem(**kw)
    assert tree_status(p) == status and weights_status(p) == status and evict_status(p) == status


def test_bad_token_problems():
    for kw, status in ((dict(Hq=3), cabi.ERR_BAD_SHAPE), (dict(T=0), cabi.ERR_BAD_SHAPE), (dict(T=65), cabi.ERR_TOO_LARGE),
                       (dict(sm_scale=float("nan")), cabi.ERR_BAD_SHAPE), (dict(softcap=float("inf")), cabi.ERR_BAD_SHAPE)):
        assert tree_status(cache_problem(**kw)) == status and weights_status(cache_problem(**kw)) == status
    assert weights_status(cache_problem(slots=63)) == cabi.ERR_BAD_SHAPE
    assert tree_status(cache_problem(slots=63), cabi.CacheTree(None, None, 4096, None, None)) == cabi.ERR_BAD_SHAPE
    assert tree_status(cache_problem(), cabi.CacheTree(4097, None, None, None, None)) == cabi.ERR_MISALIGNED
    for i in range(7):
        ptrs = [OK] * 8
        ptrs[i] = None
        assert tree_status(cache_problem(), None, ptrs) == cabi.ERR_NULL_POINTER
        if i != 5:
            assert weights_status(cache_problem(), None, ptrs[:7]) == cabi.ERR_NULL_POINTER
    for i in range(3):
        ptrs = [OK] * 8
        ptrs[i] = ODD
        assert tree_status(cache_problem(), None, ptrs) == cabi.ERR_MISALIGNED
    p = cache_problem()
    p.stride_v = (ctypes.c_longlong * 3)(2 * 16 * 64, 16 * 64, 60)
    assert tree_status(p) == cabi.ERR_MISALIGNED


def test_bad_evictions():
    p = cache_problem()
    for kw in (dict(keep=0), dict(sinks=-1), dict(recent=-1), dict(sinks=21), dict(sinks=15, recent=6), dict(out_width=1), dict(out_width=0),
               dict(recent=2 ** 31 - 1, sinks=5)):
        assert evict_status(p, **kw) == cabi.ERR_BAD_SHAPE, kw
    assert evict_status(cache_problem(slots=60)) == cabi.ERR_BAD_SHAPE
    assert evict_status(p, ptrs=[OK, OK, OK, OK, None, None]) == cabi.ERR_NULL_POINTER
    assert evict_status(p, ptrs=[ODD, OK, OK, OK, OK, None]) == cabi.ERR_MISALIGNED
    assert evict_status(p, more=(OK, OK, OK, None)) == cabi.ERR_BAD_SHAPE      # new weights over the old ones


def test_front_end_refuses_cpu_tensors():
    q = torch.zeros(1, 2, 4, 64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        be.masked_sdpa(q, q, q)
    pages, table, lens = torch.zeros(3, 2, 16, 64), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        be.tree_sdpa(q, pages, pages, table, lens)
    with pytest.raises(RuntimeError, match="no CPU path"):
        be.cache_weights(torch.zeros(1, 2, 32), q, torch.zeros(1, 2, 4), pages, table, lens)
    with pytest.raises(RuntimeError, match="no CPU path"):
        be.cache_evict(pages, pages, table, lens, torch.zeros(1, 2, 32), 4)


def test_visible_ranges():
    v = be.visible_ranges([3, 2], 7, prefix=2)
    assert v.tolist() == [[0, 2], [0, 2], [0, 3], [3, 5], [3, 5], [0, 0], [0, 0]]
    assert be.visible_ranges([3, 2], causal=False).tolist() == [[0, 3]] * 3 + [[3, 5]] * 2
    assert be.visible_ranges([4], window=2).tolist() == [[0, 1], [0, 2], [1, 3], [2, 4]]
    assert be.visible_ranges([4], window=2, prefix=3).tolist() == [[0, 3], [0, 3], [0, 3], [2, 4]]
    assert be.visible_ranges([2], prefix=9).tolist() == [[0, 2], [0, 2]]
    assert be.visible_ranges([0, 1, 0]).tolist() == [[0, 1]]
    assert be.visible_ranges([], 2).tolist() == [[0, 0], [0, 0]]
    b = be.visible_ranges([[1, 2], [2]], prefix=[[0, 2], 0])
    assert b.tolist() == [[[0, 1], [1, 3], [1, 3]], [[0, 1], [0, 2], [0, 0]]]
    assert b.dtype == torch.int32
    for bad in (dict(lengths=[3], total=2), dict(lengths=[-1]), dict(lengths=[3], window=0), dict(lengths=[3], prefix=[1, 2]), dict(lengths=[3], prefix=-1)):
        with pytest.raises(ValueError):
            be.visible_ranges(**bad)


def test_reference_forms_agree_with_torch():
    """The 64-bit forms themselves, against autograd over torch's softmax."""
    torch.manual_seed(0)
    q, k, v, do = torch.randn(2, 4, 9, 8), torch.randn(2, 2, 11, 8), torch.randn(2, 2, 11, 8), torch.randn(2, 4, 9, 8)
    vis = torch.randint(0, 6, (2, 9, 1))
    vis = torch.cat([vis, vis + 5], 2).int()
    slopes = torch.tensor([0.1, 0.2, 0.3, 0.4])
    res, tol = ref.masked(q, k, v, 0.7, visible=vis, causal=False, softcap=3.0, slopes=slopes, dout=do)
    x = [t.double().requires_grad_(True) for t in (q, k, v)]
    s = 3.0 * torch.tanh(0.7 * x[0] @ x[1].repeat_interleave(2, 1).transpose(-1, -2) / 3.0)
    d = (torch.arange(9)[:, None] + 2 - torch.arange(11)).abs()
    s = s - slopes.double()[:, None, None] * d
    seen = ref.seen_mask(2, 9, 11, False, vis)[:, None]
    out = torch.softmax(s.masked_fill(~seen, float("-inf")), -1) @ x[2].repeat_interleave(2, 1)
    out.backward(do.double())
    for n, t in (("out", out), ("dq", x[0].grad), ("dk", x[1].grad), ("dv", x[2].grad)):
        assert (res[n] - t.detach()).abs().max() < 1e-12 and (tol[n] >= 0).all() and (tol[n] > 0).any()
    assert ref.evict_one([5.0, 1.0, float("nan"), 1.0, 9.0, 2.0], 6, 3, 0, 1) == [0, 4, 5]
    assert ref.evict_one([0.0] * 5, 5, 3, 1, 1) == [0, 1, 4]
