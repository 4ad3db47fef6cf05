"""Serving from a paged key/value cache: ``tree_sdpa``, ``cache_weights``, ``cache_evict``.

The cache is a pool of pages, k_pages and v_pages [pages, kv_heads, page_size, D] (any strides with rows
contiguous and 16-byte aligned), and for every sequence a row of page numbers: its key number n lies in
slot ``n % page_size`` of page ``page_table[b, n // page_size]``.  ``lens[b]`` keys are cached; the T drafted
tokens' own keys are to be in the cache behind them, as keys ``lens[b] .. lens[b] + T - 1``.
Formulas and limits are in ``include/dsdpa.h``.  Nothing here waits for the device; a page number or a parent
out of range is left out on the device and reported by ``cabi.lib().dsdpa_device_error(device)``; with
``op.check_device_errors`` every call waits for the device, asks it and raises.
"""
from __future__ import annotations

import struct

import torch

from . import cabi, masked, op


_PROBLEM = struct.Struct("=9i2fiI4x9q")          # struct dsdpa_cache_problem, packed


def _check_int(t, shape, device, what, name):
    if t is not None and (t.dtype is not torch.int32 or t.shape != shape or t.get_device() != device):
        raise ValueError(f"{name}: {what} must be int32 {list(shape)} on cuda:{device}, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _check_pages(k_pages, v_pages, page_table, lens, name):
    dev = k_pages.get_device()
    if dev < 0 or page_table.get_device() < 0 or lens.get_device() < 0 or (v_pages is not None and v_pages.get_device() < 0):
        raise RuntimeError(f"{name}: tensors must live on a CUDA device (there is no CPU path)")
    shape = k_pages.shape
    if len(shape) != 4 or (v_pages is not None and v_pages.shape != shape):
        raise ValueError(f"{name}: k_pages and v_pages must be [pages, kv_heads, page_size, D], the same")
    if k_pages.dtype not in op._DTYPES:
        raise NotImplementedError(f"{name}: unsupported dtype {k_pages.dtype}")
    if v_pages is not None and (v_pages.dtype is not k_pages.dtype or v_pages.get_device() != dev):
        raise ValueError(f"{name}: k_pages and v_pages differ in dtype or device")
    if 0 in shape:
        raise ValueError(f"{name}: the pool of pages is empty")
    if shape[3] % 8 or not 8 <= shape[3] <= 256:
        raise ValueError(f"{name}: head dim {shape[3]} is not a multiple of 8 in 8 .. 256")
    # a copy would cost more than the call, and an eviction has to write where the caller looks
    if not masked._usable(k_pages) or (v_pages is not None and not masked._usable(v_pages)):
        raise ValueError(f"{name}: rows of the pages must be contiguous and start on 16-byte boundaries")
    table = page_table.shape
    if len(table) != 2 or table[1] == 0:
        raise ValueError(f"{name}: page_table must be int32 [B, pages of a sequence]")
    _check_int(page_table, table, dev, "page_table", name)
    _check_int(lens, table[:1], dev, "lens", name)
    return dev


def _problem(q, k_pages, v_pages, page_table, sm_scale, softcap, slots):
    pages, Hkv, size, D = k_pages.shape
    kt = k_pages.stride()
    vt = (0, 0, 0) if v_pages is None else v_pages.stride()
    Hq, T, qt = (0, 0, (0, 0, 0)) if q is None else (q.shape[1], q.shape[2], q.stride())
    B, width = page_table.shape
    return _PROBLEM.pack(B, Hq, Hkv, T, D, pages, size, width, slots, sm_scale, softcap, op._DTYPES[k_pages.dtype], 0,
                         qt[0], qt[1], qt[2], kt[0], kt[1], kt[2], vt[0], vt[1], vt[2])


def _tokens(q, k_pages, page_table, sm_scale, softcap, parents, drafted, slopes, positions, start, dev, name):
    """Checks what describes the drafted tokens; returns dsdpa_cache_tree's pointers, packed (None: all NULL), and the
    tensors they point into."""
    shape = q.shape
    if q.get_device() < 0:
        raise RuntimeError(f"{name}: tensors must live on a CUDA device (there is no CPU path)")
    if len(shape) != 4 or shape[0] != page_table.shape[0] or shape[3] != k_pages.shape[3]:
        raise ValueError(f"{name}: q must be [B, heads, T, D], got {tuple(shape)}")
    B, Hq, T, _ = shape
    if q.dtype is not k_pages.dtype or q.get_device() != dev:
        raise ValueError(f"{name}: q and the pages differ in dtype or device")
    Hkv = k_pages.shape[1]
    if Hq % Hkv:
        raise ValueError(f"{name}: {Hq} query heads are no multiple of {Hkv} key/value heads")
    if T > cabi.TREE_MAX:
        raise ValueError(f"{name}: {T} drafted tokens, at most {cabi.TREE_MAX}")
    if not masked._sound(sm_scale, softcap):
        masked._check_numbers(sm_scale, softcap, name)
    if parents is None and drafted is None and positions is None and start is None and slopes is None:
        return None, None
    masked._check_slopes(slopes, Hq, q.device, name)
    _check_int(parents, (B, T), dev, "parents", name)
    _check_int(drafted, (B,), dev, "drafted", name)
    _check_int(start, (B,), dev, "start", name)
    if positions is not None:
        slots = page_table.shape[1] * k_pages.shape[2]
        _check_int(positions, (B, Hkv, *positions.shape[2:3]), dev, "positions", name)
        if positions.dim() != 3 or positions.shape[2] < slots:
            raise ValueError(f"{name}: positions must be int32 [B, kv_heads, {slots} or more]")
    held = [None if t is None else t.contiguous() for t in (parents, drafted, positions, start, slopes)]
    return struct.pack("=5Q", *(0 if t is None else t.data_ptr() for t in held)), held


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
    sm_scale, softcap = q.shape[-1] ** -0.5 if sm_scale is None else float(sm_scale), float(softcap)
    dev = _check_pages(k_pages, v_pages, page_table, lens, name)
    tree, held = _tokens(q, k_pages, page_table, sm_scale, softcap, parents, drafted, slopes, positions, start, dev, name)
    q = masked._as_rows(q)
    B, Hq, T, _ = q.shape
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = q.new_empty((B, Hq, T), dtype=torch.float32)
    if not B * Hq * T:
        return out, lse
    page_table, lens = page_table.contiguous(), lens.contiguous()
    prob = _problem(q, k_pages, v_pages, page_table, sm_scale, softcap, positions.shape[2] if positions is not None else 0)
    L = cabi.lib()
    n = L.dsdpa_tree_workspace_bytes(prob)
    ws = q.new_empty(n, dtype=torch.uint8) if n else None
    st = L.dsdpa_tree_forward(prob, tree, q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), page_table.data_ptr(), lens.data_ptr(),
                              out.data_ptr(), lse.data_ptr(), None if ws is None else ws.data_ptr(), n, dev, masked._raw_stream(dev))
    masked._done(st, dev)
    return out, lse


def cache_weights(weights, q, lse, k_pages, page_table, lens, sm_scale=None, *, parents=None, drafted=None, take=None,
                  softcap=0.0, slopes=None, positions=None, start=None):
    """Adds to ``weights`` fp32 [B, kv_heads, slots], in place, what every key was looked at: its softmax weights summed
    over the query heads that share it and over the tokens (``take`` bool [B, T]: over those only, e.g. the
    drafted tokens that were accepted).  ``lse`` is what ``tree_sdpa`` returned for the same arguments;
    slots is at least ``page_table.shape[1] * page_size``.  Returns ``weights``."""
    name = "cache_weights"
    sm_scale, softcap = q.shape[-1] ** -0.5 if sm_scale is None else float(sm_scale), float(softcap)
    dev = _check_pages(k_pages, None, page_table, lens, name)
    tree, held = _tokens(q, k_pages, page_table, sm_scale, softcap, parents, drafted, slopes, positions, start, dev, name)
    _check_weights(weights, k_pages, page_table, dev, name)
    if lse.shape != q.shape[:3] or lse.dtype is not torch.float32 or lse.get_device() != dev:
        raise ValueError(f"{name}: lse must be the fp32 [B, heads, T] of tree_sdpa")
    if take is not None and (take.dtype is not torch.bool or take.shape != (q.shape[0], q.shape[2]) or take.get_device() != dev):
        raise ValueError(f"{name}: take must be bool [B, T] on {q.device}")
    if positions is not None and positions.shape[2] != weights.shape[2]:
        raise ValueError(f"{name}: positions and weights differ in their slots")
    if 0 in q.shape:
        return weights
    q, lse, page_table, lens = masked._as_rows(q), lse.contiguous(), page_table.contiguous(), lens.contiguous()
    if take is not None:
        take = take.contiguous()
    prob = _problem(q, k_pages, None, page_table, sm_scale, softcap, weights.shape[2])
    st = cabi.lib().dsdpa_cache_weights(prob, tree, q.data_ptr(), lse.data_ptr(), k_pages.data_ptr(), page_table.data_ptr(), lens.data_ptr(),
                                        None if take is None else take.data_ptr(), weights.data_ptr(), dev, masked._raw_stream(dev))
    masked._done(st, dev)
    return weights


def _check_weights(weights, k_pages, page_table, dev, name):
    B, Hkv, slots = page_table.shape[0], k_pages.shape[1], page_table.shape[1] * k_pages.shape[2]
    shape = weights.shape
    if weights.dtype is not torch.float32 or len(shape) != 3 or shape[0] != B or shape[1] != Hkv or shape[2] < slots or \
            weights.get_device() != dev or not weights.is_contiguous() or weights.requires_grad:
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
    dev = _check_pages(k_pages, v_pages, page_table, lens, name)
    _check_weights(weights, k_pages, page_table, dev, name)
    if not (isinstance(keep, int) and isinstance(sinks, int) and isinstance(recent, int)) or \
            keep < 1 or sinks < 0 or recent < 0 or sinks + recent > keep:
        raise ValueError(f"{name}: keep {keep} must be positive and hold sinks {sinks} and recent {recent}")
    if keep > (1 << 30):
        raise ValueError(f"{name}: keep {keep} is too large")
    if positions is not None:
        _check_int(positions, weights.shape, dev, "positions", name)
        positions = positions.contiguous()
    B, Hkv = page_table.shape[0], k_pages.shape[1]
    if out_table is not None:
        _check_int(out_table, (B, *out_table.shape[1:2]), dev, "out_table", name)
        if out_table.dim() != 2 or out_table.shape[1] * k_pages.shape[2] < min(keep, page_table.shape[1] * k_pages.shape[2]):
            raise ValueError(f"{name}: out_table has no room for {keep} keys")
    page_table, lens = page_table.contiguous(), lens.contiguous()
    out_table = page_table if out_table is None else out_table.contiguous()
    kept = lens.new_empty((B, Hkv, keep))
    new_lens, new_weights = torch.empty_like(lens), torch.empty_like(weights)
    new_positions = torch.empty_like(positions) if positions is not None else None
    if B:
        prob = _problem(None, k_pages, v_pages, page_table, 0.0, 0.0, weights.shape[2])
        st = cabi.lib().dsdpa_cache_evict(
            prob, k_pages.data_ptr(), v_pages.data_ptr(), page_table.data_ptr(), lens.data_ptr(), weights.data_ptr(),
            None if positions is None else positions.data_ptr(), keep, sinks, recent, out_table.data_ptr(), out_table.shape[1],
            kept.data_ptr(), new_lens.data_ptr(), new_weights.data_ptr(), None if positions is None else new_positions.data_ptr(),
            dev, masked._raw_stream(dev))
        masked._done(st, dev)
    return (new_lens, kept, new_weights) if positions is None else (new_lens, kept, new_weights, new_positions)
