"""Serving from a paged key/value cache: ``tree_sdpa``, ``cache_weights``, ``cache_evict``.

The cache is a pool of pages, k_pages and v_pages [pages, kv_heads, page_size, D] (any strides with rows
contiguous and 16-byte aligned), and for every sequence a row of page numbers: its key number n lies in
slot ``n % page_size`` of page ``page_table[b, n // page_size]``.  ``lens[b]`` keys are cached; the T drafted
tokens' own keys are to be in the cache behind them, as keys ``lens[b] .. lens[b] + T - 1``.
Formulas and limits are in ``include/dsdpa.h``.  Nothing here waits for the device; a page number or a parent
out of range is left out on the device and reported by ``cabi.lib().dsdpa_device_error(device)``.
"""
from __future__ import annotations

import ctypes

import torch

from . import cabi, masked, op


def _check_int(t, shape, device, what, name):
    if t is not None and (t.dtype != torch.int32 or tuple(t.shape) != tuple(shape) or t.device != device):
        raise ValueError(f"{name}: {what} must be int32 {list(shape)} on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _check_pages(k_pages, v_pages, page_table, lens, name):
    for t in (k_pages, v_pages, page_table, lens):
        if t is not None and not t.is_cuda:
            raise RuntimeError(f"{name}: tensors must live on a CUDA device (there is no CPU path)")
    if k_pages.dim() != 4 or (v_pages is not None and v_pages.shape != k_pages.shape):
        raise ValueError(f"{name}: k_pages and v_pages must be [pages, kv_heads, page_size, D], the same")
    if k_pages.dtype not in op._DTYPES:
        raise NotImplementedError(f"{name}: unsupported dtype {k_pages.dtype}")
    if v_pages is not None and (v_pages.dtype != k_pages.dtype or v_pages.device != k_pages.device):
        raise ValueError(f"{name}: k_pages and v_pages differ in dtype or device")
    if k_pages.numel() == 0:
        raise ValueError(f"{name}: the pool of pages is empty")
    if k_pages.shape[3] % 8 or not 8 <= k_pages.shape[3] <= 256:
        raise ValueError(f"{name}: head dim {k_pages.shape[3]} is not a multiple of 8 in 8 .. 256")
    for t in (k_pages, v_pages):
        # a copy would cost more than the call, and an eviction has to write where the caller looks
        if t is not None and not masked._usable(t):
            raise ValueError(f"{name}: rows of the pages must be contiguous and start on 16-byte boundaries")
    if page_table.dim() != 2 or page_table.shape[1] == 0:
        raise ValueError(f"{name}: page_table must be int32 [B, pages of a sequence]")
    _check_int(page_table, page_table.shape, k_pages.device, "page_table", name)
    _check_int(lens, page_table.shape[:1], k_pages.device, "lens", name)


def _problem(q, k_pages, v_pages, page_table, sm_scale, softcap, slots):
    prob = cabi.CacheProblem()
    prob.B, prob.Hkv = page_table.shape[0], k_pages.shape[1]
    prob.pages, prob.page_size, prob.D = k_pages.shape[0], k_pages.shape[2], k_pages.shape[3]
    prob.table_width, prob.slots, prob.dtype = page_table.shape[1], slots, op._DTYPES[k_pages.dtype]
    prob.stride_k = (ctypes.c_longlong * 3)(*k_pages.stride()[:3])
    if v_pages is not None:
        prob.stride_v = (ctypes.c_longlong * 3)(*v_pages.stride()[:3])
    if q is not None:
        prob.Hq, prob.T, prob.sm_scale, prob.softcap = q.shape[1], q.shape[2], float(sm_scale), float(softcap)
        prob.stride_q = (ctypes.c_longlong * 3)(*q.stride()[:3])
    return prob


def _tokens(q, k_pages, page_table, sm_scale, softcap, parents, drafted, slopes, positions, start, name):
    """Checks what describes the drafted tokens; returns the C struct and the tensors it points into."""
    if not q.is_cuda:
        raise RuntimeError(f"{name}: tensors must live on a CUDA device (there is no CPU path)")
    if q.dim() != 4 or q.shape[0] != page_table.shape[0] or q.shape[3] != k_pages.shape[3]:
        raise ValueError(f"{name}: q must be [B, heads, T, D], got {tuple(q.shape)}")
    B, Hq, T, _ = q.shape
    if q.dtype != k_pages.dtype or q.device != k_pages.device:
        raise ValueError(f"{name}: q and the pages differ in dtype or device")
    if Hq % k_pages.shape[1]:
        raise ValueError(f"{name}: {Hq} query heads are no multiple of {k_pages.shape[1]} key/value heads")
    if T > cabi.TREE_MAX:
        raise ValueError(f"{name}: {T} drafted tokens, at most {cabi.TREE_MAX}")
    masked._check_numbers(sm_scale, softcap, name)
    masked._check_slopes(slopes, Hq, q.device, name)
    _check_int(parents, (B, T), q.device, "parents", name)
    _check_int(drafted, (B,), q.device, "drafted", name)
    _check_int(start, (B,), q.device, "start", name)
    slots = page_table.shape[1] * k_pages.shape[2]
    if positions is not None:
        _check_int(positions, (B, k_pages.shape[1], positions.shape[-1]), q.device, "positions", name)
        if positions.shape[2] < slots:
            raise ValueError(f"{name}: positions must be int32 [B, kv_heads, {slots} or more]")
    held = [t.contiguous() if t is not None else None for t in (parents, drafted, positions, start, slopes)]
    return cabi.CacheTree(*(t.data_ptr() if t is not None else None for t in held)), held


def tree_sdpa(q, k_pages, v_pages, page_table, lens, sm_scale=None, *, parents=None, drafted=None, softcap=0.0, slopes=None,
              positions=None, start=None):
    """Attention of T drafted tokens (1 to 64; one is ordinary decoding) over a paged cache.

    q [B, heads, T, D].  Token t sees the ``lens[b]`` cached keys, itself and the tokens above it:
    ``parents`` int32 [B, T] names the earlier token that t follows, -1 for none; without it t follows t - 1.
    ``drafted`` int32 [B]: how many of a sequence's T tokens are real (default all); the rest give zeros.
    ``softcap`` and ``slopes`` as for ``masked_sdpa``; distances are between positions: a cached key's is its
    number, or ``positions`` int32 [B, kv_heads, slots]; a token without parent has ``start[b]`` (default
    ``lens[b]``) and every other one its parent's plus 1.
    Returns ``(out [B, heads, T, D], lse fp32 [B, heads, T] in base 2)``.  No gradients."""
    name = "tree_sdpa"
    sm_scale = q.shape[-1] ** -0.5 if sm_scale is None else float(sm_scale)
    _check_pages(k_pages, v_pages, page_table, lens, name)
    tree, held = _tokens(q, k_pages, page_table, sm_scale, softcap, parents, drafted, slopes, positions, start, name)
    q, k_pages, v_pages = masked._as_rows(q), k_pages.detach(), v_pages.detach()
    out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    lse = torch.empty(q.shape[:3], device=q.device, dtype=torch.float32)
    if out.numel() == 0:
        return out, lse
    page_table, lens = page_table.contiguous(), lens.contiguous()
    prob = _problem(q, k_pages, v_pages, page_table, sm_scale, softcap, positions.shape[2] if positions is not None else 0)
    L, p = cabi.lib(), op._ptr
    n = int(L.dsdpa_tree_workspace_bytes(ctypes.byref(prob)))
    ws = torch.empty(n, device=q.device, dtype=torch.uint8) if n else None
    stream = torch.cuda.current_stream(q.device).cuda_stream
    cabi.check(L.dsdpa_tree_forward(ctypes.byref(prob), ctypes.byref(tree), p(q), p(k_pages), p(v_pages), p(page_table), p(lens),
                                    p(out), p(lse), p(ws), n, q.device.index, ctypes.c_void_p(stream)))
    return out, lse


def cache_weights(weights, q, lse, k_pages, page_table, lens, sm_scale=None, *, parents=None, drafted=None, take=None,
                  softcap=0.0, slopes=None, positions=None, start=None):
    """Adds to ``weights`` fp32 [B, kv_heads, slots], in place, what every key was looked at: its softmax weights summed
    over the query heads that share it and over the tokens (``take`` bool [B, T]: over those only, e.g. the
    drafted tokens that were accepted).  ``lse`` is what ``tree_sdpa`` returned for the same arguments;
    slots is at least ``page_table.shape[1] * page_size``.  Returns ``weights``."""
    name = "cache_weights"
    sm_scale = q.shape[-1] ** -0.5 if sm_scale is None else float(sm_scale)
    _check_pages(k_pages, None, page_table, lens, name)
    tree, held = _tokens(q, k_pages, page_table, sm_scale, softcap, parents, drafted, slopes, positions, start, name)
    _check_weights(weights, k_pages, page_table, name)
    if lse.shape != q.shape[:3] or lse.dtype != torch.float32 or lse.device != q.device:
        raise ValueError(f"{name}: lse must be the fp32 [B, heads, T] of tree_sdpa")
    if take is not None and (take.dtype != torch.bool or take.shape != (q.shape[0], q.shape[2]) or take.device != q.device):
        raise ValueError(f"{name}: take must be bool [B, T] on {q.device}")
    if positions is not None and positions.shape[2] != weights.shape[2]:
        raise ValueError(f"{name}: positions and weights differ in their slots")
    if q.numel() == 0:
        return weights
    q, k_pages, lse, page_table, lens = masked._as_rows(q), k_pages.detach(), lse.contiguous(), page_table.contiguous(), lens.contiguous()
    take = take.contiguous() if take is not None else None
    prob = _problem(q, k_pages, None, page_table, sm_scale, softcap, weights.shape[2])
    p = op._ptr
    stream = torch.cuda.current_stream(q.device).cuda_stream
    cabi.check(cabi.lib().dsdpa_cache_weights(ctypes.byref(prob), ctypes.byref(tree), p(q), p(lse), p(k_pages), p(page_table),
                                              p(lens), p(take), p(weights), q.device.index, ctypes.c_void_p(stream)))
    return weights


def _check_weights(weights, k_pages, page_table, name):
    B, Hkv, slots = page_table.shape[0], k_pages.shape[1], page_table.shape[1] * k_pages.shape[2]
    if weights.dtype != torch.float32 or weights.dim() != 3 or weights.shape[:2] != (B, Hkv) or weights.shape[2] < slots or \
            weights.device != k_pages.device or not weights.is_contiguous() or weights.requires_grad:
        raise ValueError(f"{name}: weights must be a contiguous fp32 [{B}, {Hkv}, {slots} or more] on {k_pages.device}, without gradient")


def cache_evict(k_pages, v_pages, page_table, lens, weights, keep, *, sinks=0, recent=0, out_table=None, positions=None):
    """Cuts sequences longer than ``keep`` keys down to ``keep``, for every key/value head by itself: the first
    ``sinks``, the last ``recent`` and the heaviest between them (equal weights: the lowest number), in their order.

    The kept rows of k_pages and v_pages move to keys ``0 .. new_lens - 1``: in place, or into the pages of
    ``out_table`` int32 [B, n], which must hold no key of the sequences.  In place, the sequences must not
    share pages.  Returns ``(new_lens int32 [B], kept int32 [B, kv_heads, keep], new_weights)``: ``kept`` has the
    numbers of the kept keys, -1 behind the last; ``new_weights`` is ``weights`` of the kept keys, 0 behind.
    With ``positions`` (int32, of weights' shape) a fourth result: positions of the kept keys, 0 behind."""
    name = "cache_evict"
    _check_pages(k_pages, v_pages, page_table, lens, name)
    _check_weights(weights, k_pages, page_table, name)
    if not (isinstance(keep, int) and isinstance(sinks, int) and isinstance(recent, int)) or \
            keep < 1 or sinks < 0 or recent < 0 or sinks + recent > keep:
        raise ValueError(f"{name}: keep {keep} must be positive and hold sinks {sinks} and recent {recent}")
    if positions is not None:
        _check_int(positions, weights.shape, k_pages.device, "positions", name)
        positions = positions.contiguous()
    B, Hkv = page_table.shape[0], k_pages.shape[1]
    if keep > (1 << 30):
        raise ValueError(f"{name}: keep {keep} is too large")
    if out_table is not None:
        _check_int(out_table, (B, out_table.shape[-1]), k_pages.device, "out_table", name)
        if out_table.shape[1] * k_pages.shape[2] < min(keep, page_table.shape[1] * k_pages.shape[2]):
            raise ValueError(f"{name}: out_table has no room for {keep} keys")
    page_table, lens = page_table.contiguous(), lens.contiguous()
    out_table = page_table if out_table is None else out_table.contiguous()
    kept = torch.empty(B, Hkv, keep, device=k_pages.device, dtype=torch.int32)
    new_lens = torch.empty_like(lens)
    new_weights = torch.empty_like(weights)
    new_positions = torch.empty_like(positions) if positions is not None else None
    if B:
        prob = _problem(None, k_pages, v_pages, page_table, 0.0, 0.0, weights.shape[2])
        p = op._ptr
        stream = torch.cuda.current_stream(k_pages.device).cuda_stream
        cabi.check(cabi.lib().dsdpa_cache_evict(
            ctypes.byref(prob), p(k_pages), p(v_pages), p(page_table), p(lens), p(weights), p(positions), keep, sinks, recent,
            p(out_table), out_table.shape[1], p(kept), p(new_lens), p(new_weights), p(new_positions),
            k_pages.device.index, ctypes.c_void_p(stream)))
    return (new_lens, kept, new_weights) if positions is None else (new_lens, kept, new_weights, new_positions)
