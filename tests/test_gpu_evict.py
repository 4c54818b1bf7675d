"""attention.evict against its definition on the host: kept slots, moves, weights, positions and rows, all
exactly; and its refusals."""
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def T():
    import torch
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    from opentpu_amd import _lib
    _lib.load()
    return torch


def reference(k, v, w, pos, lens, budget, recent):
    """The definition: arrays k, v [B, T, H, D], w, pos [B, H, T], lens [B]."""
    k, v, nw, npos = k.copy(), v.copy(), np.zeros_like(w), np.full_like(pos, -1)
    B, H, Tn = w.shape
    for b in range(B):
        n = min(max(int(lens[b]), 0), Tn)
        left = min(n, budget)
        for h in range(H):
            src = np.arange(left)
            if n > budget:
                old = int(pos[b, h, :n].max()) - recent
                rank = [(0, 0.0, t) if int(pos[b, h, t]) > old else
                        (1, -np.inf, t) if np.isnan(w[b, h, t]) else (2, -float(w[b, h, t]), t) for t in range(n)]
                kept = sorted(range(n), key=lambda t: rank[t])[:left]
                inside = set(t for t in kept if t < left)
                src[[t for t in range(left) if t not in inside]] = sorted(t for t in kept if t >= left)
            nw[b, h, :left], npos[b, h, :left] = w[b, h, src], pos[b, h, src]
            k[b, :left, h], v[b, :left, h] = k[b, src, h], v[b, src, h]
    return k, v, nw, npos, np.minimum(np.clip(lens, 0, Tn), budget).astype(np.int32)


def make(rng, B, Tn, H, D, budget, kind):
    k, v = (rng.integers(-30000, 30000, (B, Tn, H, D)).astype(np.int16) & ~np.int16(0x7800) for _ in range(2))
    w = np.exp(2 * rng.standard_normal((B, H, Tn))).astype(np.float32)
    if kind == "ties":
        w = np.floor(w).astype(np.float32)
    elif kind == "equal":
        w[:] = 0.5
    elif kind == "odd":                                    # values that no sum of weights should have
        at = rng.random(w.shape)
        w[at < 0.1], w[(at > 0.1) & (at < 0.2)], w[(at > 0.2) & (at < 0.3)] = np.nan, np.inf, -np.inf
        w[(at > 0.3) & (at < 0.4)], w[(at > 0.4) & (at < 0.5)], w[at > 0.9] = -0.0, 0.0, -1.5
        w[(at > 0.5) & (at < 0.6)], w[(at > 0.6) & (at < 0.65)] = 1e-42, -np.nan
    pos = np.argsort(rng.random((B, H, Tn)), -1).astype(np.int32) if kind != "ties" else \
        np.broadcast_to(np.arange(Tn, dtype=np.int32), (B, H, Tn)).copy()
    lens = rng.integers(0, Tn + 1, B).astype(np.int32)
    lens[0] = Tn
    return k, v, w, pos, lens


SIZES = [
    # B, T, H, D, budget, recent
    (1, 1, 1, 8, 1, 0), (2, 2, 1, 8, 1, 1), (1, 5, 1, 16, 0, 0), (3, 33, 2, 64, 32, 8), (4, 300, 3, 40, 17, 5),
    (2, 1024, 2, 128, 1000, 100), (2, 1025, 2, 128, 1024, 0), (3, 2051, 1, 64, 1023, 512), (2, 2048, 4, 96, 2048, 3),
    (1, 5000, 2, 128, 64, 64), (1, 40000, 1, 64, 300, 10), (1, 40000, 2, 8, 39990, 300), (2, 100, 2, 64, 400, 0),
]


@pytest.mark.parametrize("kind", ["plain", "ties", "equal", "odd"])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_against_the_definition(T, size, kind):
    from opentpu_amd import attention
    say(f"evict {kind} {size}")
    B, Tn, H, D, budget, recent = size
    rng = np.random.default_rng(sum(size))
    k, v, w, pos, lens = make(rng, B, Tn, H, D, budget, kind)
    want = reference(k, v, w, pos, lens, budget, recent)
    for inplace in (False, True):
        kd, vd = (T.from_numpy(x).cuda().view(T.bfloat16) for x in (k, v))
        wd, pd, ld = (T.from_numpy(x).cuda() for x in (w, pos, lens))
        out = attention.evict(kd, vd, wd, pd, ld, budget, recent, out=(wd, pd, ld) if inplace else None)
        got = [kd.view(T.int16), vd.view(T.int16), out[0].view(T.int32), out[1], out[2]]
        for name, g, x in zip(("k", "v", "weights", "pos", "lens"), got, want):
            x = x.view(np.int32) if name == "weights" else x
            assert np.array_equal(g.cpu().numpy(), x), name
        if not inplace:
            assert np.array_equal(wd.cpu().numpy().view(np.int32), w.view(np.int32)) and np.array_equal(ld.cpu().numpy(), lens)


def test_strides_types_and_lengths_out_of_range(T):
    """Caches with heads before tokens, k and v interleaved, float32 rows; lens below 0 and past T."""
    from opentpu_amd import attention
    rng = np.random.default_rng(3)
    B, Tn, H, D, budget = 3, 90, 2, 24, 40
    k, v, w, pos, lens = make(rng, B, Tn, H, D, budget, "plain")
    lens[:] = (200, -5, 77)
    want = reference(k, v, w, pos, lens, budget, 7)
    both = T.from_numpy(np.stack([k, v], 1).astype(np.float32)).permute(0, 3, 1, 2, 4).contiguous().cuda()  # [B, H, 2, T, D]
    kd, vd = both[:, :, 0].permute(0, 2, 1, 3), both[:, :, 1].permute(0, 2, 1, 3)
    out = attention.evict(kd, vd, *(T.from_numpy(x).cuda() for x in (w, pos, lens)), budget, 7)
    assert np.array_equal(kd.cpu().numpy(), want[0].astype(np.float32))
    assert np.array_equal(vd.cpu().numpy(), want[1].astype(np.float32))
    for g, x in zip(out, want[2:]):
        assert np.array_equal(g.cpu().numpy(), x)


def test_some_in_place(T):
    """Each of the three outputs in place or not by itself."""
    from opentpu_amd import attention
    rng = np.random.default_rng(6)
    B, Tn, H, D, budget = 2, 1500, 2, 16, 700
    k, v, w, pos, lens = make(rng, B, Tn, H, D, budget, "ties")
    want = reference(k, v, w, pos, lens, budget, 9)
    for which in range(8):
        kd, vd = (T.from_numpy(x).cuda().view(T.bfloat16) for x in (k, v))
        old = [T.from_numpy(x).cuda() for x in (w, pos, lens)]
        out = [x if which >> i & 1 else T.full_like(x, 77) for i, x in enumerate(old)]
        attention.evict(kd, vd, *old, budget, 9, out=out)
        for g, x in zip((kd.view(T.int16), vd.view(T.int16), *out), want):
            assert np.array_equal(g.cpu().numpy(), x), which


def test_no_slots(T):
    """Caches without a slot: the lengths alone, in place and not."""
    from opentpu_amd import attention
    k = T.empty((2, 0, 3, 16), dtype=T.bfloat16, device="cuda")
    w, pos = T.empty((2, 3, 0), device="cuda"), T.empty((2, 3, 0), dtype=T.int32, device="cuda")
    lens = T.tensor([4, -1], dtype=T.int32, device="cuda")
    assert attention.evict(k, k.clone(), w, pos, lens, 5)[2].tolist() == [0, 0]
    attention.evict(k, k.clone(), w, pos, lens, 5, out=(w, pos, lens))
    assert lens.tolist() == [0, 0]


def test_graph(T):
    """Captured, and replayed on caches filled anew, eager work between."""
    from opentpu_amd import attention
    rng = np.random.default_rng(4)
    B, Tn, H, D, budget = 2, 300, 2, 64, 200
    first = [T.from_numpy(x).cuda() for x in make(rng, B, Tn, H, D, budget, "plain")]
    k, v, w, pos, lens = (x.clone() for x in first)
    s = T.cuda.Stream()
    with T.cuda.stream(s):
        attention.evict(k.view(T.float16), v.view(T.float16), w, pos, lens, budget, 9)
    s.synchronize()
    g = T.cuda.CUDAGraph()
    with T.cuda.graph(g):
        out = attention.evict(k.view(T.float16), v.view(T.float16), w, pos, lens, budget, 9)
    for i in range(3):
        data = make(rng, B, Tn, H, D, budget, "ties")
        for x, y in zip((k, v, w, pos, lens), data):
            x.copy_(T.from_numpy(y))
        g.replay()
        want = reference(*data, budget, 9)
        for a, b in zip((k, v, *out), want):
            assert np.array_equal(a.cpu().numpy(), b)


def test_refusals(T):
    from opentpu_amd import _lib as X
    from opentpu_amd import attention
    rng = np.random.default_rng(5)
    k, v, w, pos, lens = (T.from_numpy(x).cuda() for x in make(rng, 2, 30, 2, 16, 9, "plain"))
    k, v = k.view(T.bfloat16), v.view(T.bfloat16)
    for bad in (lambda: attention.evict(k.view(T.int16), v, w, pos, lens, 9), lambda: attention.evict(k[0], v, w, pos, lens, 9),
                lambda: attention.evict(k, v.half(), w, pos, lens, 9), lambda: attention.evict(k, v, w.double(), pos, lens, 9),
                lambda: attention.evict(k, v, w, pos.long(), lens, 9), lambda: attention.evict(k, v, w[:, :1], pos, lens, 9),
                lambda: attention.evict(k, v, w, pos, lens[:1], 9), lambda: attention.evict(k, v[:, :20], w, pos, lens, 9),
                lambda: attention.evict(k[:1].expand_as(k), v, w, pos, lens, 9), lambda: attention.evict(k.cpu(), v, w, pos, lens, 9),
                lambda: attention.evict(k, v, w.transpose(1, 2).contiguous().transpose(1, 2), pos, lens, 9),
                lambda: attention.evict(k, v, w, pos, lens, 9, out=(w, pos, lens[:1]))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: attention.evict(k, v, w, pos, lens, -1), lambda: attention.evict(k, v, w, pos, lens, 9, -1),
                lambda: attention.evict(k[..., :4], v[..., :4], w, pos, lens, 9),
                lambda: attention.evict(k[..., 4:12], v[..., 4:12], w, pos, lens, 9)):
        with pytest.raises(X.OtpuError):
            bad()
