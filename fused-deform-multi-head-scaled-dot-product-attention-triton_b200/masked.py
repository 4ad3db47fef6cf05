"""Attention over a sequence: ``masked_sdpa(q, k, v, sm_scale, ...)``.

Scores may be capped by a tanh and get a bias that falls with distance; which keys a query sees is given
as one range of keys per query (documents, prefixes, windows, padding: ``visible_ranges``) and ``causal``.
The device work is libdeform_sdpa.so's, through the C ABI of ``include/dsdpa.h``, which has the formulas.
"""
from __future__ import annotations

import struct

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import cabi, op


_raw_stream = torch._C._cuda_getCurrentRawStream     # of a device index; torch.cuda.current_stream makes an object first
_PROBLEM = struct.Struct("=6i2fiI25q")                # struct dsdpa_masked_problem, packed: a call spends its time in the host


def _usable(t):
    """Rows contiguous and 16-byte aligned, no dimension broadcast: what the kernels read as it lies.  Rows are known to
    have a multiple of 8 elements."""
    if t.data_ptr() % 16:
        return False
    if t.is_contiguous():
        return True
    e = t.element_size()
    return (t.stride(-1) == 1 and
            all(n < 2 or (st > 0 and st * e % 16 == 0) for st, n in zip(t.stride()[:-1], t.shape[:-1])))


def _as_rows(t):
    if _usable(t):
        return t
    t = t.detach().contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _check_inputs(q, k, v, sm_scale, softcap, visible, slopes, name):
    if not (q.is_cuda and k.is_cuda and v.is_cuda):
        raise RuntimeError(f"{name}: tensors must live on a CUDA device (there is no CPU path)")
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError(f"{name}: q must be [B, heads, Lq, D], k and v [B, kv_heads, Lk, D]")
    if k.shape != v.shape:
        raise ValueError(f"{name}: k and v shapes differ: {tuple(k.shape)}, {tuple(v.shape)}")
    if not (q.dtype == k.dtype == v.dtype):
        raise ValueError(f"{name}: q, k, v dtypes differ")
    if q.dtype not in op._DTYPES:
        raise NotImplementedError(f"{name}: unsupported dtype {q.dtype}")
    if not (q.device == k.device == v.device):
        raise ValueError(f"{name}: tensors are on different devices")
    B, Hq, Lq, D = q.shape
    if k.shape[0] != B or k.shape[3] != D:
        raise ValueError(f"{name}: q {tuple(q.shape)} and k {tuple(k.shape)} do not fit")
    if k.shape[1] == 0 or Hq % k.shape[1]:
        raise ValueError(f"{name}: {Hq} query heads are no multiple of {k.shape[1]} key/value heads")
    if D % 8 or not 8 <= D <= 256:
        raise ValueError(f"{name}: head dim {D} is not a multiple of 8 in 8 .. 256")
    _check_numbers(sm_scale, softcap, name)
    _check_slopes(slopes, Hq, q.device, name)
    if visible is not None:
        if visible.dtype != torch.int32 or visible.shape[-2:] != (Lq, 2) or \
                not (visible.dim() == 2 or (visible.dim() == 3 and visible.shape[0] in (1, B))):
            raise ValueError(f"{name}: visible must be int32 [B, Lq, 2] (or [Lq, 2]), got {visible.dtype} {tuple(visible.shape)}")
        if visible.device != q.device:
            raise ValueError(f"{name}: visible is on another device")


_LEAST, _MOST = torch.finfo(torch.float32).tiny, torch.finfo(torch.float32).max


def _sound(sm_scale, softcap):
    """What the kernels' fp32 can carry: sm_scale itself, softcap log2(e) and 2 |sm_scale| / softcap."""
    return -_MOST <= sm_scale <= _MOST and (softcap == 0.0 or (
        _LEAST <= softcap <= _MOST / 2 and (sm_scale == 0.0 or _LEAST <= 2.0 * abs(sm_scale) / softcap <= _MOST)))


def _check_numbers(sm_scale, softcap, name):
    if not _sound(sm_scale, softcap):
        raise ValueError(f"{name}: sm_scale {sm_scale} must be a finite fp32 number and softcap {softcap} 0 or a positive one, "
                         "neither so far from the other that 2 sm_scale / softcap leaves fp32")


def _check_slopes(slopes, heads, device, name):
    if slopes is None:
        return
    if slopes.requires_grad:
        raise ValueError(f"{name}: slopes get no gradient; pass slopes.detach()")
    if slopes.dtype != torch.float32 or tuple(slopes.shape) != (heads,) or slopes.device != device:
        raise ValueError(f"{name}: slopes must be fp32 [{heads}] on {device}")


def _mask_args(visible, slopes):
    """visible and slopes as the library takes them, and the batch stride of visible."""
    if slopes is not None:
        slopes = slopes.contiguous()
    if visible is None:
        return None, slopes, 0
    if visible.dim() == 2:
        visible = visible.unsqueeze(0)
    if visible.shape[0] == 1 or visible.stride(0) == 0:
        visible = visible[:1]
    visible = visible.contiguous()
    if visible.data_ptr() % 8:
        visible = visible.clone()
    return visible, slopes, 0 if visible.shape[0] == 1 else visible.stride(0)


def _plain(q, k, v, visible, slopes):
    """The usual arguments, seen at a glance; whatever else comes is looked at by _check_inputs."""
    dev, dt = q.get_device(), q.dtype
    if dev < 0 or k.get_device() != dev or v.get_device() != dev or k.dtype is not dt or v.dtype is not dt or dt not in op._DTYPES:
        return False
    qs, ks = q.shape, k.shape
    if len(qs) != 4 or len(ks) != 4 or v.shape != ks or qs[0] != ks[0] or qs[3] != ks[3] or ks[1] == 0 or qs[1] % ks[1] or \
            qs[3] % 8 or not 8 <= qs[3] <= 256:
        return False
    if visible is not None and (visible.dtype is not torch.int32 or visible.shape != (qs[0], qs[2], 2) or visible.get_device() != dev):
        return False
    return slopes is None or (slopes.dtype is torch.float32 and slopes.shape == (qs[1],) and slopes.get_device() == dev and
                              not slopes.requires_grad)


def _numbers(q, sm_scale, softcap):
    sm_scale = q.shape[-1] ** -0.5 if sm_scale is None else float(sm_scale)
    softcap = float(softcap)
    if not _sound(sm_scale, softcap):
        _check_numbers(sm_scale, softcap, "masked_sdpa")
    return sm_scale, softcap


def _done(st, device):
    """After a call of the library: its status, and with ``op.check_device_errors`` what the kernels recorded."""
    if st:
        cabi.check(st)
    if op.check_device_errors:
        cabi.check(cabi.lib().dsdpa_device_error(device))


def masked_forward_raw(q, k, v, sm_scale=None, *, causal=False, visible=None, softcap=0.0, slopes=None):
    """Forward through the C ABI.  Returns ``(out, lse)``, lse fp32 [B, heads, Lq] in base 2; no autograd.

    Arguments as for ``masked_sdpa``."""
    sm_scale, softcap = _numbers(q, sm_scale, softcap)
    if not _plain(q, k, v, visible, slopes):
        _check_inputs(q, k, v, sm_scale, softcap, visible, slopes, "masked_sdpa")
    q, k, v = _as_rows(q), _as_rows(k), _as_rows(v)
    B, Hq, Lq, D = q.shape
    out = torch.empty_like(q)
    lse = q.new_empty((B, Hq, Lq), dtype=torch.float32)
    if not B * Hq * Lq:
        return out, lse
    visible, slopes, stride = _mask_args(visible, slopes)
    qt, kt, vt, ot = q.stride(), k.stride(), v.stride(), out.stride()
    prob = _PROBLEM.pack(B, Hq, k.shape[1], Lq, k.shape[2], D, sm_scale, softcap, op._DTYPES[q.dtype], cabi.MASKED_CAUSAL if causal else 0,
                         qt[0], qt[1], qt[2], kt[0], kt[1], kt[2], vt[0], vt[1], vt[2], ot[0], ot[1], ot[2],
                         0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, stride)
    dev = q.get_device()
    st = cabi.lib().dsdpa_masked_forward(prob, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                         None if visible is None else visible.data_ptr(), None if slopes is None else slopes.data_ptr(),
                                         out.data_ptr(), lse.data_ptr(), dev, _raw_stream(dev))
    _done(st, dev)
    return out, lse


def masked_backward_raw(q, k, v, out, lse, dout, sm_scale=None, *, causal=False, visible=None, softcap=0.0, slopes=None):
    """Backward through the C ABI.  Returns ``(dq, dk, dv)``; ``out`` and ``lse`` are the forward's."""
    sm_scale, softcap = _numbers(q, sm_scale, softcap)
    if not _plain(q, k, v, visible, slopes):
        _check_inputs(q, k, v, sm_scale, softcap, visible, slopes, "masked_sdpa")
    dev = q.get_device()
    if out.shape != q.shape or dout.shape != q.shape or lse.shape != q.shape[:3]:
        raise ValueError("masked_sdpa: out, dout and lse must have the shapes of the forward's results")
    if out.dtype != q.dtype or lse.dtype != torch.float32 or out.get_device() != dev or lse.get_device() != dev or dout.get_device() != dev:
        raise ValueError("masked_sdpa: out and lse must be the forward's results")
    if dout.dtype != q.dtype:
        dout = dout.to(q.dtype)
    q, k, v, out, dout, lse = _as_rows(q), _as_rows(k), _as_rows(v), _as_rows(out), _as_rows(dout), lse.contiguous()
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    B, Hq, Lq, D = q.shape
    Hkv, Lk = k.shape[1], k.shape[2]
    if not B * Hq or not (Lq or Lk):
        return dq, dk.zero_(), dv.zero_()
    visible, slopes, stride = _mask_args(visible, slopes)
    rows = []
    for t in (q, k, v, out, dout, dq, dk, dv):
        rows += t.stride()[:3]
    prob = _PROBLEM.pack(B, Hq, Hkv, Lq, Lk, D, sm_scale, softcap, op._DTYPES[q.dtype], cabi.MASKED_CAUSAL if causal else 0, *rows, stride)
    L = cabi.lib()
    n = L.dsdpa_masked_backward_workspace_bytes(prob)
    ws = q.new_empty(n, dtype=torch.uint8) if n else None
    st = L.dsdpa_masked_backward(prob, q.data_ptr(), k.data_ptr(), v.data_ptr(), None if visible is None else visible.data_ptr(),
                                 None if slopes is None else slopes.data_ptr(), out.data_ptr(), lse.data_ptr(), dout.data_ptr(),
                                 dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), None if ws is None else ws.data_ptr(), n, dev, _raw_stream(dev))
    _done(st, dev)
    return dq, dk, dv


def _grads(ctx, dout):
    q, k, v, out, lse, visible, slopes = ctx.saved_tensors
    dq, dk, dv = masked_backward_raw(q, k, v, out, lse, dout, ctx.sm_scale, causal=ctx.causal, visible=visible,
                                     softcap=ctx.softcap, slopes=slopes)
    return dq, dk, dv, None, None, None, None, None


_grads_once = once_differentiable(_grads)


class _MaskedSDPA(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, sm_scale, causal, visible, softcap, slopes):
        out, lse = masked_forward_raw(q, k, v, sm_scale, causal=causal, visible=visible, softcap=softcap, slopes=slopes)
        ctx.save_for_backward(q, k, v, out, lse, visible, slopes)
        ctx.sm_scale, ctx.causal, ctx.softcap = sm_scale, causal, softcap
        return out

    @staticmethod
    def backward(ctx, dout):
        # gradients of gradients are refused where somebody asks for them
        return _grads_once(ctx, dout) if torch.is_grad_enabled() else _grads(ctx, dout)


def masked_sdpa(q, k, v, sm_scale=None, *, causal=False, visible=None, softcap=0.0, slopes=None):
    """Attention of q [B, heads, Lq, D] over k, v [B, kv_heads, Lk, D]; returns out, of q's shape.

    ``sm_scale``: factor of q.k, ``D ** -0.5`` by default.  ``causal``: query i sees keys up to ``i + Lk - Lq``.
    ``visible``: int32 [B, Lq, 2] (or [Lq, 2], the same for every batch element): query i sees keys
    ``lo <= j < hi`` only.  ``softcap``: scores become ``softcap * tanh(score / softcap)``; 0: none.
    ``slopes``: fp32 [heads]; ``slopes[h] * |i + Lk - Lq - j|`` is taken off the (capped) scores.
    Query heads in groups of ``heads // kv_heads`` share a key/value head.  D is a multiple of 8 up to 256.
    A query that sees no key gives zeros; keys it does not see have no part in its result, whatever they
    hold.  Gradients for q, k and v, bit-reproducible."""
    if not (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)) and forward_ad._current_level < 0:
        return masked_forward_raw(q, k, v, sm_scale, causal=causal, visible=visible, softcap=softcap, slopes=slopes)[0]
    sm_scale = q.shape[-1] ** -0.5 if sm_scale is None else float(sm_scale)
    return _MaskedSDPA.apply(q, k, v, sm_scale, bool(causal), visible, float(softcap), slopes)


def visible_ranges(lengths, total=None, *, prefix=0, causal=True, window=None, device=None):
    """``visible`` of ``masked_sdpa`` for self-attention over packed documents: int32 [total, 2] from the lengths of
    the documents that lie one behind the other (a list, or a list of such lists for a batch: [B, total, 2]).

    A token sees its own document only: all of it, or with ``causal`` what lies before it and itself.  The
    first ``prefix`` tokens of every document (a number, or one per document) see one another in any case.
    ``window``: not further back than that many tokens, itself among them.  Tokens behind the last document,
    up to ``total``, are padding and see nothing."""
    if len(lengths) and isinstance(lengths[0], (list, tuple)):
        if total is None:
            total = max(sum(x) for x in lengths)
        each = prefix if isinstance(prefix, (list, tuple)) else [prefix] * len(lengths)
        if len(each) != len(lengths):
            raise ValueError("visible_ranges: prefix does not fit the batch")
        return torch.stack([visible_ranges(x, total, prefix=f, causal=causal, window=window, device=device)
                            for x, f in zip(lengths, each)])
    used = sum(lengths)
    total = used if total is None else int(total)
    if any(n < 0 for n in lengths) or used > total:
        raise ValueError(f"visible_ranges: lengths {lengths} do not fit {total} tokens")
    if window is not None and window < 1:
        raise ValueError("visible_ranges: window must be at least 1")
    fixes = list(prefix) if isinstance(prefix, (list, tuple)) else [prefix] * len(lengths)
    if len(fixes) != len(lengths) or any(f < 0 for f in fixes):
        raise ValueError("visible_ranges: prefix must be one number, or one per document, not negative")
    n = torch.tensor(list(lengths), dtype=torch.int64)
    start = torch.repeat_interleave(torch.cumsum(n, 0) - n, n)
    end = start + torch.repeat_interleave(n, n)
    fix = torch.minimum(start + torch.repeat_interleave(torch.tensor(fixes, dtype=torch.int64), n), end)
    at = torch.arange(used)
    hi = torch.maximum(at + 1, torch.where(at < fix, fix, start)) if causal else end
    lo = start if window is None else torch.where(at < fix, start, torch.maximum(start, at + 1 - window))
    out = torch.zeros(total, 2, dtype=torch.int32)
    out[:used, 0], out[:used, 1] = lo.int(), hi.int()
    return out.to(device) if device is not None else out
