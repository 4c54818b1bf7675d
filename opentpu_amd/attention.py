"""Attention between a decoder's linears for a batch of sequences that share a prompt, and the cache it
reads: `shared` (the prefix's keys and values multiplied once by the queries of all sequences, each
sequence's own cache by its own, one softmax over both) and `evict` (slots of the own caches freed by
accumulated attention weight).

Tensors of the current device, bfloat16 or float16; every call is queued on the current torch stream and allocates its
work area from torch's allocator on that stream."""
from __future__ import annotations

import functools
import operator

from . import _lib as X

_TYPES = {}                                     # torch dtype -> the ABI's type, once torch is loaded


def _types():
    if not _TYPES:
        T = X.torch()
        _TYPES.update({T.float32: X.F32, T.bfloat16: X.BF16, T.float16: X.F16})
    return _TYPES


@functools.lru_cache(maxsize=1024)
def _attn_bytes(*sizes) -> int:
    return X.load().otpu_attn_call_bytes(*sizes)


@functools.lru_cache(maxsize=1024)
def _evict_bytes(*sizes) -> int:
    return X.load().otpu_kv_evict_work_bytes(*sizes)


def _check(who: str, name: str, t, dtype, shape, dev: int):
    """t is a tensor of this type and shape on device `dev`."""
    if t.dtype != dtype or t.shape != shape or t.get_device() != dev:
        raise ValueError(f"{who}: {name} is {t.dtype} {list(t.shape)} on {t.device}, needs {dtype} {list(shape)} on cuda:{dev}")


def _dense(who: str, name: str, t, dtype, shape, dev: int) -> int:
    """The address of a contiguous tensor."""
    _check(who, name, t, dtype, shape, dev)
    if not t.is_contiguous():
        raise ValueError(f"{who}: {name} must be contiguous")
    return t.data_ptr()


def _rows(who: str, name: str, t, dtype, shape, dev: int, written: bool = False) -> tuple:
    """The strides of a tensor whose columns are adjacent (written: and which is no broadcast one)."""
    _check(who, name, t, dtype, shape, dev)
    s = t.stride()
    if written and 0 in s and any(n > 1 and not x for n, x in zip(shape, s)):
        raise ValueError(f"{who}: {name} is a broadcast tensor, it cannot be written to")
    if s[-1] != 1 and t.numel() and shape[-1] > 1:
        raise ValueError(f"{who}: the columns of {name} must be adjacent")
    return s


def _count(x) -> int:
    """A whole number as the ABI's int32: more slots than any cache has, or fewer than none, stay that."""
    return max(-1, min(operator.index(x), 0x7FFFFFFF))


def _used(shape, s) -> tuple:
    """Strides, 0 for dimensions of one place: no address has them in it, so they may be anything."""
    return tuple(0 if n == 1 else x for n, x in zip(shape, s))


def shared(q, prefix_k, prefix_v, k, v, lens, *, scale: float | None = None, weights=None, out=None):
    """Attention of q [B, Lq, Hq, D] over the shared prefix [P, Hkv, D] and each sequence's own cache
    k, v [B, T, Hkv, D], of which lens [B] (int32) tokens are in use, the Lq newest the queries' own:
    query i of sequence b sees the whole prefix and own tokens 0 .. lens[b] - Lq + i.  Returns out
    [B, Lq, Hq, D] in q's type; a query that sees no key gives 0.  Scores, maxima and sums are float32; for its product
    with the values each softmax weight is rounded to q's type, about as large an error as the output's own rounding.

    Hq is a multiple of Hkv, D a multiple of 8 up to 256, B * Lq * Hq at most 2^23, P at most 2^30, B * Hkv *
    ceil(T / 32) below 2^24, tokens less than 2^22 elements apart.  scale: D ** -0.5 unless given.  prefix_k and
    prefix_v may be None, so may k, v and lens together.  weights (float32 [B, Hkv, T], contiguous): each
    own token's softmax weights, summed over the queries and the query heads of its head, are added to
    it.  out: a tensor to write to, which must overlap no input."""
    kinds = _types()
    dt, dev = q.dtype, q.get_device()
    if q.dim() != 4 or dev < 0 or kinds.get(dt, X.F32) == X.F32:
        raise ValueError(f"shared: q is {dt} {list(q.shape)} on {q.device}, needs [B, Lq, Hq, D] in bfloat16 or float16")
    B, Lq, Hq, D = q.shape
    if (prefix_k is None) != (prefix_v is None) or (k is None) != (v is None) or (k is None) != (lens is None):
        raise ValueError("shared: prefix_k and prefix_v go together, so do k, v and lens")
    if prefix_k is None and k is None:
        raise ValueError("shared: neither a prefix nor a cache")
    T = X.torch()
    P = N = pk = pv = kp = vp = lp = wp = 0
    ps = pvs = ks = vs = (0, 0, 0)
    qs = q.stride()
    if qs[3] != 1:
        _rows("shared", "q", q, dt, (B, Lq, Hq, D), dev)
    own = pre = (0, 0, 0)
    if k is not None:                                      # (tests in line: the functions say what is wrong)
        own = k.shape
        if len(own) != 4:
            raise ValueError(f"shared: k is {list(own)}, needs [B, T, Hkv, D]")
        N, Hkv = own[1], own[2]
        ks, vs = k.stride(), v.stride()
        if k.dtype != dt or own[0] != B or own[3] != D or k.get_device() != dev or ks[3] != 1:
            _rows("shared", "k", k, dt, (B, N, Hkv, D), dev)
        if v.dtype != dt or v.shape != own or v.get_device() != dev or vs[3] != 1:
            _rows("shared", "v", v, dt, own, dev)
        lp = _dense("shared", "lens", lens, T.int32, (B,), dev)
        kp, vp = k.data_ptr(), v.data_ptr()
    if prefix_k is not None:
        pre = prefix_k.shape
        if len(pre) != 3:
            raise ValueError(f"shared: prefix_k is {list(pre)}, needs [P, Hkv, D]")
        if k is None:
            Hkv = pre[1]
        P, ps, pvs = pre[0], prefix_k.stride(), prefix_v.stride()
        if prefix_k.dtype != dt or pre[1] != Hkv or pre[2] != D or prefix_k.get_device() != dev or ps[2] != 1:
            _rows("shared", "prefix_k", prefix_k, dt, (P, Hkv, D), dev)
        if prefix_v.dtype != dt or prefix_v.shape != pre or prefix_v.get_device() != dev or pvs[2] != 1:
            _rows("shared", "prefix_v", prefix_v, dt, pre, dev)
        pk, pv = prefix_k.data_ptr(), prefix_v.data_ptr()
    if weights is not None:
        wp = _dense("shared", "weights", weights, T.float32, (B, Hkv, N), dev)
    if out is None:
        out = T.empty_like(q, memory_format=T.contiguous_format)
        os = out.stride()
    else:
        os = _rows("shared", "out", out, dt, (B, Lq, Hq, D), dev, True)
    if out.numel() == 0:
        return out
    if N == 1 or P == 1 or (qs[0] | qs[1] | qs[2] | ps[0] | ps[1] | pvs[0] | pvs[1] | ks[0] | ks[1] | ks[2] | vs[0] | vs[1] | vs[2]
                            | os[0] | os[1] | os[2]) & 7:
        qs, os = _used(q.shape, qs), _used(q.shape, os)
        ks, vs, ps, pvs = _used(own, ks), _used(own, vs), _used(pre, ps), _used(pre, pvs)
    nbytes = _attn_bytes(B, Lq, Hq, Hkv, D, P, N, weights is not None)
    work = q.new_empty((nbytes // 2 + 1,))                 # (of q's type: the least work for the host)
    X.call("otpu_attn_shared", X.ATTN_ARGS.pack(
        X.ATTN_ARGS.size, q.data_ptr(), qs[0], qs[1], qs[2], pk, ps[0], ps[1], pv, pvs[0], pvs[1], kp, ks[0], ks[1], ks[2], vp,
        vs[0], vs[1], vs[2], lp, out.data_ptr(), os[0], os[1], os[2], wp, work.data_ptr(), nbytes, B, Lq, Hq, Hkv, D, P, N,
        kinds[dt], D ** -0.5 if scale is None else scale), X.stream_of("shared", dev))
    return out


def evict(k, v, weights, pos, lens, budget: int, recent: int = 0, *, out=None):
    """Frees slots of the caches k, v [B, T, H, D] in place: where lens[b] > budget, each head keeps `budget`
    slots, those of its `recent` newest positions first (of more than `budget` the lower slots), then those of the
    largest accumulated weights, the lower slot where they are equal.  Slots below budget that go are overwritten by the slots past it
    that stay (both in slot order), so slots keep no order of positions.

    weights float32 and pos int32 [B, H, T] (contiguous): each slot's accumulated weight (`shared` adds to
    it) and its token's position.  lens int32 [B].  T at most 2^30, B * H below 2^22.  Returns the
    new (weights, pos, lens); slots past the new length have weight 0 and position -1.  out: the three tensors to write them to; (weights, pos, lens)
    themselves may be given."""
    dt, dev, T = k.dtype, k.get_device(), X.torch()
    if type(budget) is not int or type(recent) is not int or (budget | recent) >> 31:
        budget, recent = _count(budget), _count(recent)
    if k.dim() != 4 or dev < 0 or dt not in _types():
        raise ValueError(f"evict: k is {dt} {list(k.shape)} on {k.device}, needs [B, T, H, D] in bfloat16, float16 or float32")
    B, N, H, D = k.shape
    e = k.element_size()
    ks, vs = _rows("evict", "k", k, dt, (B, N, H, D), dev, True), _rows("evict", "v", v, dt, (B, N, H, D), dev, True)
    if e * (ks[0] | ks[1] | ks[2] | vs[0] | vs[1] | vs[2]) & 15:
        ks, vs = _used(k.shape, ks), _used(k.shape, vs)
    slots = (B, H, N)
    if out is None:
        out = (T.empty_like(weights), T.empty_like(pos), T.empty_like(lens))
    f32, i32 = T.float32, T.int32
    address = []
    for names, (w, p, n) in ((("weights", "pos", "lens"), (weights, pos, lens)), (("out[0]", "out[1]", "out[2]"), out)):
        if not (w.dtype == f32 and p.dtype == n.dtype == i32 and w.shape == p.shape == slots and n.shape == (B,)
                and w.get_device() == p.get_device() == n.get_device() == dev
                and w.is_contiguous() and p.is_contiguous() and n.is_contiguous()):
            for name, t, d, shape in zip(names, (w, p, n), (f32, i32, i32), (slots, slots, (B,))):
                _dense("evict", name, t, d, shape, dev)
        address += (w.data_ptr(), p.data_ptr(), n.data_ptr())
    nbytes = _evict_bytes(B, N, H, budget)
    work = lens.new_empty((nbytes // 4 + 1,))
    X.call("otpu_kv_evict", X.EVICT_ARGS.pack(
        X.EVICT_ARGS.size, k.data_ptr(), e * ks[0], e * ks[1], e * ks[2], v.data_ptr(), e * vs[0], e * vs[1], e * vs[2], *address,
        work.data_ptr(), nbytes, B, N, H, e * D, budget, recent), X.stream_of("evict", dev))
    return out


__all__ = ["shared", "evict"]
