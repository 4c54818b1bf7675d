"""attention.shared on own caches past one segment and past one workgroup of weights, and prompts whose row tiles go in their
own order, against the definition in float64: outputs and the weights that eviction goes by.  Bounds as in
test_gpu_attention.py, whose definition and check these are."""

import numpy as np
import pytest

from test_gpu_attention import T, check, make, say  # noqa: F401

pytestmark = pytest.mark.gpu

LENS = (0, 1, 1023, 1024, 1025, 31, 257, 513, 2049)


def lengths(T, B, Lq, n):
    """Sequences of no token, one, the edges of a segment and of 1024 tokens, fewer than the queries, and all of them."""
    return T.tensor([n, *(min(x, n) for x in LENS), Lq, max(Lq - 1, 0)][:B], dtype=T.int32, device="cuda")


@pytest.mark.parametrize("dt", ["bfloat16", "float16"])
@pytest.mark.parametrize("size", [
    # B, Lq, Hq, Hkv, D, P, T: the scores of at most 32 rows a head kept for the weights, own keys in several segments
    (12, 1, 2, 1, 64, 0, 1030), (12, 1, 4, 1, 128, 70, 2500), (12, 5, 3, 1, 64, 33, 1030), (10, 3, 4, 2, 40, 0, 2500),
    (12, 16, 2, 1, 128, 0, 1291), (4, 2, 2, 2, 256, 9, 2500),
    # more rows: the weights from the keys again, own keys in several segments
    (4, 33, 1, 1, 64, 10, 1030), (3, 20, 4, 1, 128, 0, 1291), (3, 70, 2, 1, 96, 40, 1100),
], ids=lambda s: "x".join(map(str, s)))
def test_long_own_caches(T, dt, size):  # noqa: F811
    from opentpu_amd import attention
    say("long", dt, size)
    dt = getattr(T, dt)
    rng = np.random.default_rng(sum(size))
    B, Lq, Hq, Hkv, D, P, Tn = size
    args = [t.cuda() for t in make(T, rng, dt, *size)]
    args[5] = lengths(T, B, Lq, Tn)
    q, pk, pv, k, v, lens = args
    w0 = T.from_numpy(rng.random((B, Hkv, Tn)).astype(np.float32)).cuda()
    w = w0.clone()
    got = attention.shared(*args, weights=w)
    check(T, dt, args, got, w0, w)
    check(T, dt, args, attention.shared(*args))
    # slots that no query sees, whatever they hold
    for b, n in enumerate(lens.tolist()):
        k[b, n:], v[b, n:] = float("nan"), float("inf")
    w2 = w0.clone()
    assert T.equal(attention.shared(*args, weights=w2), got) and T.equal(w, w2)


@pytest.mark.parametrize("dt", ["bfloat16", "float16"])
@pytest.mark.parametrize("size", [(3, 6, 4, 2, 128, 20, 1500), (3, 40, 2, 1, 64, 0, 1500), (2, 9, 2, 1, 256, 0, 900), (2, 130, 1, 1, 128, 50, 1100)],
                         ids=lambda s: "x".join(map(str, s)))
def test_infinities_in_a_later_segment(T, dt, size):  # noqa: F811
    """Values that are no number in the newest own tokens, which lie in the last segment: the rows that see them get what the
    definition gives, the others what they got without them."""
    from opentpu_amd import attention
    say("later segment", dt, size)
    dt = getattr(T, dt)
    rng = np.random.default_rng(sum(size))
    B, Lq, Hq, Hkv, D, P, Tn = size
    inf, nan = float("inf"), float("nan")
    args = [t.cuda() for t in make(T, rng, dt, *size)]
    q, pk, pv, k, v, lens = args
    lens[:] = Tn
    lens[1] = Tn - 37
    want = attention.shared(*args)
    check(T, dt, args, want)
    for b, n in enumerate(lens.tolist()):
        v[b, n - 1, :, 1], v[b, n - 2, :, 2], v[b, n - 3, :, 3] = inf, -inf, nan
        v[b, n - 2, :, 4], v[b, n - 3, :, 4] = inf, -inf
    w = T.zeros((B, Hkv, Tn), device="cuda")
    for got in (attention.shared(*args), attention.shared(*args, weights=w)):
        assert T.equal(got[..., 5:], want[..., 5:]) and T.equal(got[..., 0], want[..., 0])
        for d, back, value in ((1, 1, inf), (2, 2, -inf)):
            assert bool((got[:, Lq - back:, :, d] == value).all()) and T.equal(got[:, :Lq - back, :, d], want[:, :Lq - back, :, d])
        assert bool(T.isnan(got[:, Lq - 3:, :, 3]).all()) and T.equal(got[:, :Lq - 3, :, 3], want[:, :Lq - 3, :, 3])
        assert bool((got[:, Lq - 3, :, 4] == -inf).all()) and bool(T.isnan(got[:, Lq - 2:, :, 4]).all())
        assert T.equal(got[:, :Lq - 3, :, 4], want[:, :Lq - 3, :, 4])
    assert bool(T.isfinite(w).all())


@pytest.mark.parametrize("dt", ["bfloat16", "float16"])
@pytest.mark.parametrize("size", [(11, 150, 16, 8, 128, 0, 200), (14, 130, 15, 5, 72, 0, 140), (5, 240, 32, 16, 16, 0, 250),
                                  (30, 100, 14, 7, 64, 0, 128), (11, 150, 16, 8, 200, 0, 160)], ids=lambda s: "x".join(map(str, s)))
def test_row_tiles_in_their_own_order(T, dt, size):  # noqa: F811
    """Prompts alone whose row tiles take each CU's first place and some of its second one, one segment a row: each type,
    the kernels' widths, rows a tile's part, head numbers that divide the CUs and that do not."""
    from opentpu_amd import _lib as X
    from opentpu_amd import attention
    say("tile order", dt, size)
    B, Lq, Hq, Hkv, D, P, Tn = size
    cus = T.cuda.get_device_properties(0).multi_processor_count
    tiles = B * Hkv * -(-Lq * (Hq // Hkv) // 128)
    assert Lq * (Hq // Hkv) > 64 and cus < tiles <= 2 * cus
    if D <= 128:                                           # (stored as outputs: one segment)
        assert X.load().otpu_attn_call_bytes(*size, 0) == 0
    dt = getattr(T, dt)
    rng = np.random.default_rng(sum(size))
    args = [t.cuda() for t in make(T, rng, dt, *size)]
    args[5][0], args[5][1], args[5][2] = 0, Tn, Lq // 3
    w0 = T.zeros((B, Hkv, Tn), device="cuda")
    w = w0.clone()
    got = attention.shared(args[0], None, None, *args[3:], weights=w)
    check(T, dt, args, got, w0, w)
    assert T.equal(attention.shared(args[0], None, None, *args[3:]), got)


@pytest.mark.parametrize("dt", ["bfloat16", "float16"])
@pytest.mark.parametrize("size", [(5, 1, 2, 1, 40, 60, 0), (130, 2, 40, 20, 128, 199, 0), (3, 1, 4, 2, 128, 90, 0), (40, 2, 33, 33, 64, 66, 0)],
                         ids=lambda s: "x".join(map(str, s)))
def test_a_prefix_alone_in_one_segment(T, dt, size):  # noqa: F811
    """Rows of a prefix alone that are stored as outputs, against the definition."""
    from opentpu_amd import _lib as X
    from opentpu_amd import attention
    say("prefix alone", dt, size)
    assert X.load().otpu_attn_call_bytes(*size, 0) == 0
    dt = getattr(T, dt)
    args = [t.cuda() for t in make(T, np.random.default_rng(sum(size)), dt, *size)]
    check(T, dt, args, attention.shared(*args[:3], None, None, None))
