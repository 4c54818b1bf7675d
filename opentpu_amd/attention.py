"""Attention between a decoder's linears for a batch of sequences that share a prompt, and the cache it
reads: `shared` (the prefix's keys and values multiplied once by the queries of all sequences, each
sequence's own cache by its own, one softmax over both) and `evict` (slots of the own caches freed by
accumulated attention weight).

Device tensors, bfloat16 or float16; every call is queued on the current torch stream and allocates its
work area from torch's allocator on that stream."""
from __future__ import annotations

from . import _lib as X

_TYPES = {}                                     # torch dtype -> the ABI's type, once torch is loaded


def _types():
    if not _TYPES:
        T = X.torch()
        _TYPES.update({T.float32: X.F32, T.bfloat16: X.BF16, T.float16: X.F16})
    return _TYPES


def _check(who: str, name: str, t, dtype, shape, device, dense: bool = False):
    """t is a device tensor of this type and shape whose columns are adjacent (dense: contiguous)."""
    if t.dtype != dtype or tuple(t.shape) != tuple(shape) or t.device != device:
        raise ValueError(f"{who}: {name} is {t.dtype} {list(t.shape)} on {t.device}, needs {dtype} {list(shape)} on {device}")
    if dense:
        if not t.is_contiguous():
            raise ValueError(f"{who}: {name} must be contiguous")
    elif t.numel() and t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{who}: the columns of {name} must be adjacent")


def shared(q, prefix_k, prefix_v, k, v, lens, *, scale: float | None = None, weights=None, out=None):
    """Attention of q [B, Lq, Hq, D] over the shared prefix [P, Hkv, D] and each sequence's own cache
    k, v [B, T, Hkv, D], of which lens [B] (int32) tokens are in use, the Lq newest the queries' own:
    query i of sequence b sees the whole prefix and own tokens 0 .. lens[b] - Lq + i.  Returns out
    [B, Lq, Hq, D] in q's type; a query that sees no key gives 0.

    Hq is a multiple of Hkv, D a multiple of 8 up to 256.  scale: D ** -0.5 unless given.  prefix_k and
    prefix_v may be None, so may k, v and lens together.  weights (float32 [B, Hkv, T], contiguous): each
    own token's softmax weights, summed over the queries and the query heads of its head, are added to
    it.  out: a tensor to write to, which must overlap no input."""
    kinds = _types()
    if q.dim() != 4 or not q.is_cuda or kinds.get(q.dtype, X.F32) == X.F32:
        raise ValueError(f"shared: q is {q.dtype} {list(q.shape)} on {q.device}, needs [B, Lq, Hq, D] in bfloat16 or float16")
    B, Lq, Hq, D = q.shape
    dt, dev = q.dtype, q.device
    if (prefix_k is None) != (prefix_v is None) or (k is None) != (v is None) or (k is None) != (lens is None):
        raise ValueError("shared: prefix_k and prefix_v go together, so do k, v and lens")
    if prefix_k is None and k is None:
        raise ValueError("shared: neither a prefix nor a cache")
    P = T = 0
    Hkv = (k if prefix_k is None else prefix_k).shape[-2]
    _check("shared", "q", q, dt, (B, Lq, Hq, D), dev)
    pk = pv = kp = vp = lp = None
    ps = ks = vs = (0, 0, 0)
    pvs = (0, 0)
    if prefix_k is not None:
        P = prefix_k.shape[0]
        _check("shared", "prefix_k", prefix_k, dt, (P, Hkv, D), dev)
        _check("shared", "prefix_v", prefix_v, dt, (P, Hkv, D), dev)
        pk, pv, ps, pvs = prefix_k.data_ptr(), prefix_v.data_ptr(), prefix_k.stride(), prefix_v.stride()
    if k is not None:
        T = k.shape[1]
        _check("shared", "k", k, dt, (B, T, Hkv, D), dev)
        _check("shared", "v", v, dt, (B, T, Hkv, D), dev)
        _check("shared", "lens", lens, X.torch().int32, (B,), dev, True)
        kp, vp, lp, ks, vs = k.data_ptr(), v.data_ptr(), lens.data_ptr(), k.stride(), v.stride()
    if weights is not None:
        _check("shared", "weights", weights, X.torch().float32, (B, Hkv, T), dev, True)
    if out is None:
        out = X.torch().empty((B, Lq, Hq, D), dtype=dt, device=dev)
    else:
        _check("shared", "out", out, dt, (B, Lq, Hq, D), dev)
    if out.numel() == 0:
        return out
    nbytes = X.load().otpu_attn_work_bytes(B, Lq, Hq, Hkv, D, P, T)
    work = X.torch().empty((max(nbytes, 1),), dtype=X.torch().uint8, device=dev)
    qs, os = q.stride(), out.stride()
    X.call("otpu_attn_shared", q.data_ptr(), qs[0], qs[1], qs[2], pk, ps[0], ps[1], pv, pvs[0], pvs[1], P, kp, ks[0],
           ks[1], ks[2], vp, vs[0], vs[1], vs[2], lp, T, B, Lq, Hq, Hkv, D, kinds[dt],
           D ** -0.5 if scale is None else scale, out.data_ptr(), os[0], os[1], os[2], X.ptr(weights), work.data_ptr(),
           nbytes, X.stream())
    return out


def evict(k, v, weights, pos, lens, budget: int, recent: int = 0, *, out=None):
    """Frees slots of the caches k, v [B, T, H, D] in place: where lens[b] > budget, each head keeps `budget`
    slots, those of its `recent` newest positions first, then those of the largest accumulated weights, the
    lower slot where they are equal.  Slots below budget that go are overwritten by the slots past it
    that stay (both in slot order), so slots keep no order of positions.

    weights float32 and pos int32 [B, H, T] (contiguous): each slot's accumulated weight (`shared` adds to
    it) and its token's position.  lens int32 [B].  Returns the new (weights, pos, lens); slots past the new
    length have weight 0 and position -1.  out: the three tensors to write them to; (weights, pos, lens)
    themselves may be given."""
    kinds = _types()
    if k.dim() != 4 or not k.is_cuda or k.dtype not in kinds:
        raise ValueError(f"evict: k is {k.dtype} {list(k.shape)} on {k.device}, needs [B, T, H, D] in bfloat16, float16 or float32")
    B, T, H, D = k.shape
    t, dev, e = X.torch(), k.device, k.element_size()
    _check("evict", "k", k, k.dtype, (B, T, H, D), dev)
    _check("evict", "v", v, k.dtype, (B, T, H, D), dev)
    if out is None:
        out = (t.empty_like(weights), t.empty_like(pos), t.empty_like(lens))
    for name, x, dt, shape in (("weights", weights, t.float32, (B, H, T)), ("pos", pos, t.int32, (B, H, T)),
                               ("lens", lens, t.int32, (B,))):
        _check("evict", name, x, dt, shape, dev, True)
    for name, x, dt, shape in zip(("out[0]", "out[1]", "out[2]"), out, (t.float32, t.int32, t.int32),
                                  ((B, H, T), (B, H, T), (B,))):
        _check("evict", name, x, dt, shape, dev, True)
    nbytes = X.load().otpu_kv_evict_work_bytes(B, T, H, budget)
    work = t.empty((max(nbytes, 1),), dtype=t.uint8, device=dev)
    X.call("otpu_kv_evict", k.data_ptr(), *(e * s for s in k.stride()[:3]), v.data_ptr(), *(e * s for s in v.stride()[:3]),
           e * D, weights.data_ptr(), pos.data_ptr(), lens.data_ptr(), B, T, H, budget, recent, out[0].data_ptr(),
           out[1].data_ptr(), out[2].data_ptr(), work.data_ptr(), nbytes, X.stream())
    return out


__all__ = ["shared", "evict"]
