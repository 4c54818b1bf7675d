"""Dimensions of one place: their strides are no part of any address, so whatever they are the calls between the linears take
them (a view of one row of a slab of an odd pitch, one token of caches far apart)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def T():
    import torch
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    from opentpu_amd import _lib
    _lib.load()
    return torch


def odd(T, t):
    """t with odd or huge strides where it has one place: the same memory."""
    s = [x if n > 1 else (1 << 23) + 3 for n, x in zip(t.shape, t.contiguous().stride())]
    return T.as_strided(t.contiguous(), t.shape, s)


def test_norm_quantize(T):
    from opentpu_amd import mxu
    rng = np.random.default_rng(1)
    for dt in (T.float32, T.bfloat16, T.float16):
        col = T.from_numpy(rng.standard_normal((64, 1)).astype(np.float32)).to(dt).cuda()
        gamma = T.ones(64, device="cuda")
        want, h0 = mxu.norm_quantize(col.t().contiguous().clone(memory_format=T.contiguous_format).view(1, 64), gamma, col.view(1, 64))
        for x in (col.t(), odd(T, col.view(1, 64))):       # strides (1, 1), and an odd pitch
            out = odd(T, T.zeros((1, 64), dtype=dt, device="cuda"))
            got, h = mxu.norm_quantize(x, gamma, x, h=out)
            assert h is out and T.equal(h, h0) and all(T.equal(a, b) for a, b in zip(got[:3], want[:3]))
            assert T.equal(mxu.norm_quantize(x, gamma)[0][0], mxu.norm_quantize(col.view(1, 64).clone(), gamma)[0][0])


@pytest.mark.parametrize("size", [(1, 1, 1, 1, 64, 1, 1), (3, 1, 4, 1, 64, 1, 20), (1, 5, 2, 2, 128, 30, 1), (2, 1, 2, 1, 64, 9, 1)])
def test_shared(T, size):
    from opentpu_amd import attention
    rng = np.random.default_rng(2)
    B, Lq, Hq, Hkv, D, P, n = size

    def x(*shape):
        return T.from_numpy(rng.standard_normal(shape).astype(np.float32)).bfloat16().cuda()
    args = [x(B, Lq, Hq, D), x(P, Hkv, D), x(P, Hkv, D), x(B, n, Hkv, D), x(B, n, Hkv, D)]
    lens = T.full((B,), n, dtype=T.int32, device="cuda")
    want = attention.shared(*args, lens)
    out = odd(T, T.zeros((B, Lq, Hq, D), dtype=T.bfloat16, device="cuda"))
    got = attention.shared(*(odd(T, t) for t in args), lens, out=out)
    assert got is out and T.equal(out, want)
    assert T.equal(attention.shared(odd(T, args[0]), *args[1:], lens), want)


@pytest.mark.parametrize("size", [(1, 1, 1, 8), (1, 9, 1, 24), (2, 1, 3, 16), (1, 40, 2, 64)])
def test_evict(T, size):
    from opentpu_amd import attention
    rng = np.random.default_rng(3)
    B, n, H, D = size
    k, v = (T.from_numpy(rng.standard_normal((B, n, H, D)).astype(np.float32)).cuda() for _ in range(2))
    w = T.from_numpy(rng.random((B, H, n)).astype(np.float32)).cuda()
    pos = T.arange(n, dtype=T.int32, device="cuda").expand(B, H, n).contiguous()
    lens = T.full((B,), n, dtype=T.int32, device="cuda")
    k1, v1, k2, v2 = k.clone(), v.clone(), odd(T, k.clone()), odd(T, v.clone())
    want = attention.evict(k1, v1, w, pos, lens, n // 2, 1)
    got = attention.evict(k2, v2, w, pos, lens, n // 2, 1)
    assert T.equal(k1, k2) and T.equal(v1, v2) and all(T.equal(a, b) for a, b in zip(got, want))


def test_a_prefix_or_a_cache_alone(T):
    """One token of the one without the other, and rows of an odd pitch."""
    from opentpu_amd import attention
    rng = np.random.default_rng(4)
    q, p, k = (T.from_numpy(rng.standard_normal(s).astype(np.float32)).half().cuda() for s in ((2, 1, 2, 64), (1, 2, 64), (2, 1, 2, 64)))
    lens = T.ones((2,), dtype=T.int32, device="cuda")
    for x in (q, odd(T, q)):
        assert T.equal(attention.shared(x, p, p, None, None, None), p.expand(2, 1, 2, 64))
        assert T.equal(attention.shared(x, None, None, k, k, lens), k)
        assert T.equal(attention.shared(x, odd(T, p), p, None, None, None), p.expand(2, 1, 2, 64))
