"""attention.shared against the softmax's definition in float64, and its refusals.

The bound of an output, from the definition.  With u the unit roundoff of the 16-bit type (2^-8 bfloat16,
2^-11 float16) and A = sum_t p_t |v_t|: rounding the output gives u |o|, rounding each weight for the
matrix product u A, and an error of e in a score's exponent (fp32 sums of D products: D 2^-24 sum |q k|
scale, twice for the sum in the denominator) 2 e A; float16 holds weights under 2^-14 of the row's largest
to 2^-25 of it.  Each term once more for what is of second order."""
import math
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


def reference(q, pk, pv, k, v, lens, scale):
    """(out, A, weights, e): the definition in float64 on the host; q [B, Lq, Hq, D] etc. numpy float64."""
    B, Lq, Hq, D = q.shape
    Hkv = pk.shape[1]
    G, Tn = Hq // Hkv, k.shape[1]
    out, A = np.zeros(q.shape), np.zeros(q.shape)
    w, e = np.zeros((B, Hkv, Tn)), np.zeros((B, Lq, Hq))
    for b in range(B):
        n = min(max(int(lens[b]), 0), Tn)
        for i in range(Lq):
            seen = max(0, min(n, n - Lq + i + 1))
            for h in range(Hq):
                g = h // G
                keys = np.concatenate([pk[:, g], k[b, :seen, g]])
                vals = np.concatenate([pv[:, g], v[b, :seen, g]])
                if not len(keys):
                    continue
                s = keys @ q[b, i, h] * scale
                e[b, i, h] = D * 2.0 ** -24 * np.max(np.abs(keys) @ np.abs(q[b, i, h])) * scale + 2.0 ** -22 * np.max(np.abs(s))
                p = np.exp(s - s.max())
                p /= p.sum()
                out[b, i, h] = p @ vals
                A[b, i, h] = p @ np.abs(vals)
                w[b, g, :seen] += p[len(pk):]
    return out, A, w, e


def make(T, rng, dt, B, Lq, Hq, Hkv, D, P, Tn, spread=1.0):
    def x(*shape):
        return T.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(dt)
    q, pk, pv, k, v = x(B, Lq, Hq, D) * spread, x(P, Hkv, D), x(P, Hkv, D), x(B, Tn, Hkv, D), x(B, Tn, Hkv, D)
    lens = T.from_numpy(rng.integers(0, Tn + 1, B).astype(np.int32))
    return q.to(dt), pk, pv, k, v, lens


def check(T, dt, args, got, w0=None, w=None, scale=None):
    q, pk, pv, k, v, lens = (t.cpu().double().numpy() if t.dtype != T.int32 else t.cpu().numpy() for t in args)
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    out, A, dw, e = reference(q, pk, pv, k, v, lens, scale)
    u = 2.0 ** -8 if dt == T.bfloat16 else 2.0 ** -11
    n = pk.shape[0] + k.shape[1]
    big = max((float(np.abs(t).max()) if t.size else 0.0) for t in (pv, v))
    bound = 1.1 * (u * np.abs(out) + u * A + 4 * e[..., None] * A) + (n * 2.0 ** -25 * big if dt == T.float16 else 0) + 1e-30
    err = np.abs(got.cpu().double().numpy() - out)
    assert (err <= bound).all(), (float((err / bound).max()), float(err.max()))
    if w is not None:
        wb = w0.cpu().double().numpy()
        err = np.abs(w.cpu().double().numpy() - wb - dw)
        lim = 1.1 * (4 * e.max() + 2.0 ** -20) * dw + 2.0 ** -23 * (np.abs(wb) + dw) + 1e-30
        assert (err <= lim).all(), float((err / lim).max())


SIZES = [
    # B, Lq, Hq, Hkv, D, P, T
    (1, 1, 1, 1, 64, 1, 1),
    (1, 1, 2, 1, 128, 0, 5),
    (3, 1, 4, 2, 128, 33, 0),
    (3, 1, 16, 8, 128, 300, 70),
    (5, 1, 8, 1, 64, 65, 129),
    (2, 3, 6, 3, 40, 129, 31),
    (2, 7, 5, 1, 96, 64, 257),
    (33, 1, 2, 2, 8, 700, 3),
    (2, 70, 2, 1, 128, 511, 90),
    (1, 150, 4, 2, 64, 100, 150),
    (2, 5, 3, 1, 256, 130, 67),
    (2, 20, 8, 2, 200, 77, 40),
    (20, 2, 16, 4, 136, 520, 19),
    (70, 1, 4, 1, 128, 1025, 9),
]


@pytest.mark.parametrize("dt", ["bfloat16", "float16"])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_against_the_definition(T, dt, size):
    from opentpu_amd import attention
    say(f"shared {dt} {size}")
    dt = getattr(T, dt)
    rng = np.random.default_rng(sum(size))
    B, Lq, Hq, Hkv, D, P, Tn = size
    args = [t.cuda() for t in make(T, rng, dt, *size)]
    q, pk, pv, k, v, lens = args
    if B > 1:
        lens[0], lens[1] = 0, Tn                          # a sequence with nothing of its own, and a full one
    w0 = T.from_numpy(rng.random((B, Hkv, Tn)).astype(np.float32)).cuda()
    w = w0.clone()
    got = attention.shared(q, pk if P else None, pv if P else None, k if Tn else None, v if Tn else None,
                           lens if Tn else None, weights=w)
    check(T, dt, args, got, w0, w)
    again = attention.shared(q, pk, pv, k, v, lens)
    assert T.equal(got, again)                            # the same bits with a prefix or cache of no token


def test_scores_of_many_sizes(T):
    """Scores from far below to far above the others, in an order that raises the maximum many times."""
    from opentpu_amd import attention
    rng = np.random.default_rng(5)
    dt = T.float16
    q, pk, pv, k, v, lens = make(T, rng, dt, 4, 2, 4, 2, 64, 400, 90, 3.0)
    pk = (pk.float() * T.linspace(0.1, 3, 400)[:, None, None]).to(dt)
    k = (k.float() * T.linspace(3, 0.01, 90)[None, :, None, None]).to(dt)
    args = [t.cuda() for t in (q, pk, pv, k, v, lens)]
    for scale in (0.03, 0.5):
        check(T, dt, args, attention.shared(*args, scale=scale), scale=scale)


def test_what_is_masked_is_not_read_into_a_result(T):
    """NaN and infinities in slots past lens, and in newer tokens than a query's own."""
    from opentpu_amd import attention
    rng = np.random.default_rng(6)
    for dt in (T.bfloat16, T.float16):
        for Lq, Hq, Hkv, D in ((1, 4, 2, 128), (6, 4, 2, 128), (40, 2, 2, 64), (9, 2, 1, 256), (130, 2, 1, 128)):
            say("masked", dt, Lq, Hq, Hkv, D)
            B, P, Tn = 3, 50, 200
            q, pk, pv, k, v, _ = make(T, rng, dt, B, Lq, Hq, Hkv, D, P, Tn)
            lens = T.tensor([Lq, 150, Tn], dtype=T.int32)
            want = attention.shared(*(t.cuda() for t in (q, pk, pv, k, v, lens)))
            bad = T.tensor([float("nan"), float("inf"), -float("inf")]).to(dt)
            for b in range(B):
                n = int(lens[b])
                k[b, n:], v[b, n:] = bad[0], bad[b]
            w = T.zeros((B, Hkv, Tn), device="cuda")
            got = attention.shared(*(t.cuda() for t in (q, pk, pv, k, v, lens)), weights=w)
            assert T.equal(got, want) and bool(T.isfinite(w).all())
            if Lq == 1:
                continue
            # the newest own token: only the last query sees it
            for b in range(B):
                n = int(lens[b]) - 1
                k[b, n, :, 0], v[b, n, :, 1] = bad[0], bad[b]
            got = attention.shared(*(t.cuda() for t in (q, pk, pv, k, v, lens)))
            assert T.equal(got[:, :-1], want[:, :-1]) and bool(T.isnan(got[:, -1]).all())
            # seen infinities and NaN among the values: what the sum gives
            k[:, :, :, 0] = 0.5
            for b in range(B):
                n = int(lens[b]) - 1
                v[b, n] = 1.0
                v[b, n, :, 2], v[b, n, :, 3], v[b, n, :, 4] = bad[1], bad[2], bad[0]
            k[:, 150:, :, 0] = 0.5
            k[1, 150:] = 0
            v[1, 150:] = 0
            k[0, Lq:], v[0, Lq:] = 0, 0
            got = attention.shared(*(t.cuda() for t in (q, pk, pv, k, v, lens))).float()
            last = got[:, -1]
            assert bool((last[..., 2] == float("inf")).all()) and bool((last[..., 3] == -float("inf")).all())
            assert bool(T.isnan(last[..., 4]).all()) and bool(T.isfinite(last[..., 5:]).all())
            assert bool(T.isfinite(got[:, :-1]).all())


def test_strides(T):
    """Operands as views of larger tensors: q, k and v of one qkv row, caches with heads before tokens."""
    from opentpu_amd import attention
    rng = np.random.default_rng(7)
    dt, B, Lq, Hq, Hkv, D, P, Tn = T.bfloat16, 3, 2, 6, 2, 64, 70, 40
    q, pk, pv, k, v, lens = (t.cuda() for t in make(T, rng, dt, B, Lq, Hq, Hkv, D, P, Tn))
    want = attention.shared(q, pk, pv, k, v, lens)
    slab = T.zeros((B, Lq, Hq + 4, D), dtype=dt, device="cuda")
    slab[:, :, 2:2 + Hq] = q
    both = T.stack([k, v], 2)                              # [B, T, 2, Hkv, D]
    heads = pk.permute(1, 0, 2).contiguous().permute(1, 0, 2)
    out = T.zeros((Lq, B, Hq + 1, D + 8), dtype=dt, device="cuda")
    view = out.permute(1, 0, 2, 3)[:, :, :Hq, :D]
    got = attention.shared(slab[:, :, 2:2 + Hq], heads, pv, both[:, :, 0], both[:, :, 1], lens, out=view)
    assert got is view and T.equal(got, want)
    assert not out[:, :, Hq].any() and not out[..., D:].any()


def test_long_prefix_past_32_bits(T):
    """A prefix whose last token lies more than 2^32 bytes after its first: tokens 2^21 elements apart."""
    from opentpu_amd import attention
    rng = np.random.default_rng(8)
    dt, P, gap = T.bfloat16, 1100, 1 << 21
    q, pk, pv, k, v, lens = (t.cuda() for t in make(T, rng, dt, 2, 1, 2, 1, 64, P, 4))
    wide = T.empty((P, gap), dtype=dt, device="cuda")
    wide[:, :64], wide[:, 64:128] = pk[:, 0], pv[:, 0]
    got = attention.shared(q, wide[:, None, :64], wide[:, None, 64:128], k, v, lens)
    assert T.equal(got, attention.shared(q, pk, pv, k, v, lens))


def test_broadcast_inputs(T):
    """One query row, one prefix and one cache for all, as expanded tensors."""
    from opentpu_amd import attention
    rng = np.random.default_rng(11)
    q, pk, pv, k, v, lens = (t.cuda() for t in make(T, rng, T.float16, 1, 1, 2, 1, 64, 30, 20))
    B = 5
    args = [q.expand(B, 3, 2, 64), pk.expand(30, 2, 64), pv.expand(30, 2, 64), k.expand(B, 20, 2, 64), v.expand(B, 20, 2, 64),
            T.arange(B, dtype=T.int32, device="cuda")]
    assert T.equal(attention.shared(*args), attention.shared(*(t.contiguous() for t in args)))


def test_stream_and_graph(T):
    """On another stream than the default one, and captured: replays with new inputs, eager work between."""
    from opentpu_amd import attention
    rng = np.random.default_rng(9)
    args = [t.cuda() for t in make(T, rng, T.bfloat16, 4, 1, 4, 2, 128, 600, 64)]
    w = T.zeros((4, 2, 64), device="cuda")
    want = attention.shared(*args)
    s = T.cuda.Stream()
    s.wait_stream(T.cuda.current_stream())
    with T.cuda.stream(s):
        got = attention.shared(*args)
    s.synchronize()
    assert T.equal(got, want)
    g = T.cuda.CUDAGraph()
    with T.cuda.graph(g):
        out = attention.shared(*args, weights=w)
    for x in range(4):
        w.zero_()
        args[0].copy_(T.randn_like(args[0]))
        args[5].fill_(16 * x)
        g.replay()
        w2 = T.zeros_like(w)
        assert T.equal(out, attention.shared(*args, weights=w2)) and T.equal(w, w2)
        T.cuda.synchronize()


def test_no_queries_and_refusals(T):
    from opentpu_amd import _lib as X
    from opentpu_amd import attention
    rng = np.random.default_rng(10)
    q, pk, pv, k, v, lens = (t.cuda() for t in make(T, rng, T.bfloat16, 2, 3, 4, 2, 64, 20, 10))
    assert attention.shared(q[:, :0], pk, pv, k, v, lens).shape == (2, 0, 4, 64)
    assert attention.shared(q[:0], pk, pv, k[:0], v[:0], lens[:0]).shape == (0, 3, 4, 64)
    for bad in (lambda: attention.shared(q.float(), pk, pv, k, v, lens), lambda: attention.shared(q[0], pk, pv, k, v, lens),
                lambda: attention.shared(q, pk.half(), pv, k, v, lens), lambda: attention.shared(q, pk, None, k, v, lens),
                lambda: attention.shared(q, pk, pv, k, v, None), lambda: attention.shared(q, None, None, None, None, None),
                lambda: attention.shared(q, pk, pv, k, v, lens.long()), lambda: attention.shared(q, pk, pv, k[:, :5], v, lens),
                lambda: attention.shared(q, pk, pv[:7], k, v, lens), lambda: attention.shared(q, pk[..., :32], pv, k, v, lens),
                lambda: attention.shared(q, pk, pv, k, v, lens, weights=T.zeros((2, 2, 9), device="cuda")),
                lambda: attention.shared(q, pk, pv, k, v, lens, weights=T.zeros((2, 10, 2), device="cuda").transpose(1, 2)),
                lambda: attention.shared(q, pk, pv, k, v, lens, out=T.empty_like(q[:1])),
                lambda: attention.shared(q, pk, pv, k, v, lens, out=T.empty_like(q[:1]).expand_as(q)),
                lambda: attention.shared(q.transpose(2, 3), pk, pv, k, v, lens),
                lambda: attention.shared(q.cpu(), pk, pv, k, v, lens), lambda: attention.shared(q, pk.cpu(), pv, k, v, lens)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: attention.shared(q, pk, pv, k, v, lens, scale=0.0),
                lambda: attention.shared(q, pk, pv, k, v, lens, scale=-1.0),
                lambda: attention.shared(q, pk, pv, k, v, lens, scale=math.nan),
                lambda: attention.shared(q[:, :, :3], pk, pv, k, v, lens),
                lambda: attention.shared(q[..., :60], pk[..., :60], pv[..., :60], k[..., :60], v[..., :60], lens),
                lambda: attention.shared(q[..., 4:60], pk[..., 4:60], pv[..., 4:60], k[..., 4:60], v[..., 4:60], lens)):
        with pytest.raises(X.OtpuError):
            bad()


@pytest.mark.parametrize("dt", ["bfloat16", "float16"])
def test_what_is_no_number_is_not_lost(T, dt):
    """A NaN in a query makes its row and the weights it adds NaN, though it raises no maximum; a key's NaN every row
    that sees it; no other row changes.  Few rows and many, a prefix and a cache alone and together."""
    from opentpu_amd import attention
    rng = np.random.default_rng(21)
    dt = getattr(T, dt)
    nan = float("nan")
    for B, Lq, Hq, Hkv, D, P, Tn in ((3, 1, 4, 2, 128, 40, 9), (3, 1, 4, 2, 64, 0, 300), (2, 3, 2, 1, 96, 700, 0),
                                     (2, 50, 6, 2, 128, 200, 60), (70, 1, 4, 1, 128, 1025, 40), (2, 9, 2, 2, 256, 90, 12)):
        say("no number", dt, B, Lq, Hq, Hkv, D, P, Tn)
        q, pk, pv, k, v, _ = (t.cuda() for t in make(T, rng, dt, B, Lq, Hq, Hkv, D, P, Tn))
        lens = T.full((B,), Tn, dtype=T.int32, device="cuda")
        w0 = T.zeros((B, Hkv, Tn), device="cuda")
        want = attention.shared(q, pk, pv, k, v, lens, weights=w0)
        q2, w = q.clone(), T.zeros_like(w0)
        q2[1, Lq - 1, 1, 5] = nan
        got = attention.shared(q2, pk, pv, k, v, lens, weights=w)
        hit = T.zeros((B, Lq, Hq), dtype=T.bool, device="cuda")
        hit[1, Lq - 1, 1] = True
        assert bool(T.isnan(got[hit]).all()) and T.equal(got[~hit], want[~hit])
        if Tn:
            head = T.zeros((B, Hkv), dtype=T.bool, device="cuda")
            head[1, 1 * Hkv // Hq] = True                 # (query head 1's)
            assert bool(T.isnan(w[head]).all()) and T.equal(w[~head], w0[~head])
        if P:
            pk2 = pk.clone()
            pk2[P - 1, 0, 3] = nan
            got = attention.shared(q, pk2, pv, k, v, lens)
            G = Hq // Hkv
            assert bool(T.isnan(got[:, :, :G]).all()) and T.equal(got[:, :, G:], want[:, :, G:])


@pytest.mark.parametrize("dt", ["bfloat16", "float16"])
def test_infinities_at_the_end_of_a_prefix(T, dt):
    """The values of a prefix's last token, which the last step's places past it repeat."""
    from opentpu_amd import attention
    rng = np.random.default_rng(22)
    dt = getattr(T, dt)
    inf = float("inf")
    for B, Lq, Hq, Hkv, D, P in ((2, 1, 2, 1, 128, 33), (2, 1, 2, 1, 64, 500), (40, 2, 2, 1, 128, 65), (40, 2, 2, 1, 72, 1000), (3, 1, 1, 1, 256, 50),
                                 (40, 2, 2, 1, 256, 50)):
        say("end of a prefix", dt, B, Lq, Hq, Hkv, D, P)
        q, pk, pv, *_ = (t.cuda() for t in make(T, rng, dt, B, Lq, Hq, Hkv, D, P, 0))
        want = attention.shared(q, pk, pv, None, None, None)
        pv[P - 1, :, 3], pv[P - 1, :, 4] = inf, -inf
        got = attention.shared(q, pk, pv, None, None, None)
        assert bool((got[..., 3] == inf).all()) and bool((got[..., 4] == -inf).all())
        got[..., 3:5] = want[..., 3:5]
        assert T.equal(got, want)


def test_many_small_weights(T):
    """One key far above 2^17 others of one score: their weights are under fp16's subnormals, their sum is not small.
    Bound: rounding a weight 2^-11 or, within 2^-32 of the largest, 2^-25 absolute against its scale of 2^7 or more; the
    output's rounding 2^-11; and fp32 sums of 2^17 terms in parts of at most 2^12 (a relative 2^-12 of what they add up)."""
    from opentpu_amd import attention
    P, D = 1 << 17, 64
    q = T.zeros((1, 1, 1, D), dtype=T.float16, device="cuda")
    q[..., 0] = 1.0
    pv = T.ones((P, 1, D), dtype=T.float16, device="cuda")
    for gap in (9.0, 13.0, 16.0, 17.0, 17.5):
        for place in (0, 70000, P - 1):
            pk = T.zeros((P, 1, D), dtype=T.float16, device="cuda")
            pk[place, 0, 0] = gap
            pv[:] = 1
            pv[place] = 0
            got = attention.shared(q, pk, pv, None, None, None, scale=1.0).double()
            mass = (P - 1) * math.exp(-gap)
            want = mass / (1 + mass)
            bound = want * (2.0 ** -11 + 2.0 ** -11 + 2.0 ** -12) + P * 2.0 ** -32 + 2.0 ** -25
            assert float((got - want).abs().max()) <= bound, (gap, place, float(got[0, 0, 0, 0]), want, bound)


@pytest.mark.parametrize("dt", ["bfloat16", "float16"])
def test_one_segment(T, dt):
    """Where a row has one share and no weights are asked, it is stored as the output at once: the same bits as with
    weights, whose call joins shares; into a view; rows that see nothing; infinities among newer tokens."""
    from opentpu_amd import attention
    rng = np.random.default_rng(23)
    dt = getattr(T, dt)
    for B, Lq, Hq, Hkv, D, P, Tn in ((3, 1, 4, 2, 128, 0, 40), (90, 1, 16, 8, 64, 0, 130), (2, 70, 8, 8, 96, 0, 200), (40, 100, 4, 4, 128, 0, 140),
                                     (5, 1, 2, 1, 40, 60, 0), (300, 3, 16, 16, 128, 300, 0), (2, 3, 2, 2, 200, 0, 9)):
        say("one segment", dt, B, Lq, Hq, Hkv, D, P, Tn)
        args = [t.cuda() for t in make(T, rng, dt, B, Lq, Hq, Hkv, D, P, Tn)]
        if Tn:
            args[5][0], args[5][1] = 0, Tn
            args[4][1, Tn - 1, :, 2] = float("inf")        # the newest token of sequence 1: seen by its last query
        slab = T.full((B, Lq, Hq + 1, D + 8), 7.0, dtype=dt, device="cuda")
        got = attention.shared(*args, out=slab[:, :, :Hq, :D])
        if Tn:
            want = attention.shared(*args, weights=T.zeros((B, Hkv, Tn), device="cuda"))
            assert T.equal(got, want) and not got[0].any()
            assert bool((got[1, -1, :, 2] == float("inf")).all()) and bool(T.isfinite(got[1, :-1]).all())
        else:
            own = [x.expand(B, *x.shape) for x in args[1:3]]   # the prefix as the caches of queries that see all of it
            full = T.full((B,), P, dtype=T.int32, device="cuda")
            for i in range(Lq):
                want = attention.shared(args[0][:, i:i + 1], None, None, *own, full)
                assert float((got[:, i:i + 1].float() - want.float()).abs().max()) <= 2 * 2.0 ** (-8 if dt == T.bfloat16 else -11) * 5
        assert bool((slab[:, :, Hq:] == 7).all()) and bool((slab[..., D:] == 7).all())


def test_prompts_of_many_row_tiles(T):
    """Prompts alone whose row tiles take each CU's first place and some of the second ones, in their own order: every
    row of every sequence and head, the heads a divisor of the CUs and not."""
    from opentpu_amd import attention
    rng = np.random.default_rng(24)
    for size in ((30, 150, 5, 5, 16, 0, 160), (18, 200, 8, 8, 16, 0, 210), (3, 290, 32, 16, 16, 0, 300)):
        say("row tiles", size)
        args = [t.cuda() for t in make(T, rng, T.bfloat16, *size)]
        q, pk, pv, k, v, lens = args
        lens[2] = size[6]
        w0 = T.zeros((size[0], size[3], size[6]), device="cuda")
        w = w0.clone()
        got = attention.shared(q, None, None, k, v, lens, weights=w)
        check(T, T.bfloat16, args, got, w0, w)
        assert T.equal(attention.shared(q, None, None, k, v, lens), got)


@pytest.mark.parametrize("dt", ["bfloat16", "float16"])
def test_prefix_and_own_keys_in_one(T, dt):
    """Queries of a tile's size and more on a short prefix: a workgroup takes the prefix and its sequence's keys.  Lengths
    of 0, below the queries' number and full; infinities at the prefix's end, NaN past lens and in newer tokens."""
    from opentpu_amd import attention
    rng = np.random.default_rng(25)
    dt = getattr(T, dt)
    nan, inf = float("nan"), float("inf")
    for size in ((13, 125, 4, 4, 16, 100, 150), (3, 128, 2, 2, 128, 64, 140), (3, 64, 4, 2, 64, 7, 200), (3, 128, 2, 1, 96, 33, 256),
                 (3, 128, 1, 1, 128, 1, 128)):
        say("both", dt, size)
        B, Lq, Hq, Hkv, D, P, Tn = size
        args = [t.cuda() for t in make(T, rng, dt, *size)]
        q, pk, pv, k, v, lens = args
        lens[0], lens[1], lens[2] = 0, Tn, Lq // 2
        w0 = T.from_numpy(rng.random((B, Hkv, Tn)).astype(np.float32)).cuda()
        w = w0.clone()
        got = attention.shared(*args, weights=w)
        check(T, dt, args, got, w0, w)
        assert T.equal(attention.shared(*args), got)
        # what a query does not see
        for b in range(B):
            k[b, int(lens[b]):], v[b, int(lens[b]):] = nan, (nan, inf, -inf)[b % 3]
        assert T.equal(attention.shared(*args), got)
        k[1, Tn - 1, :, 0], v[1, Tn - 1, :, 1] = nan, inf
        new = attention.shared(*args)
        assert T.equal(new[0], got[0]) and T.equal(new[1, :-1], got[1, :-1]) and bool(T.isnan(new[1, -1]).all())
        # what every query sees
        k[1, Tn - 1, :, 0], v[1, Tn - 1, :, 1] = 0.5, 1.0
        pv[P - 1, :, 3], pv[P - 1, :, 4] = inf, -inf
        new = attention.shared(*args)
        assert bool((new[..., 3] == inf).all()) and bool((new[..., 4] == -inf).all()) and bool(T.isfinite(new[..., 5:]).all())
        q[1, 0, 0, 0] = nan
        new2 = attention.shared(*args)
        assert bool(T.isnan(new2[1, 0, 0]).all()) and T.equal(new2[1, 1:], new[1, 1:]) and T.equal(new2[0], new[0])
