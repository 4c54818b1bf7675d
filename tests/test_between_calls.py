"""What otpu_norm_qact, otpu_attn_shared and otpu_kv_evict take and refuse, by their host checks alone (no
device here: a call that passes them fails at its launch), and the sizes of their work areas."""
import os

import pytest

from opentpu_amd import _lib as X

pytestmark = pytest.mark.skipif(not os.path.exists(X.LIB_PATH) or os.path.exists("/dev/kfd"),
                                reason="a built library and no GPU (the calls' addresses are not memory)")
P = 4096                                                  # an address that passes every alignment check


def code(name, *args):
    """The refusal's code, 0 where the checks take the call (its launch fails, or nothing is to do)."""
    rc = getattr(X.load(), name)(*args)
    return rc if rc in (-1, -2, -3) else 0


def norm(x=P, ldx=256, res=P, ldr=256, dtype=0, M=4, K=256, gamma=P, eps=1e-6, flags=0, h=P, ldh=256, r=None, q=P, ldq=256,
         S=P, d=P, ldd=8):
    return code("otpu_norm_qact", x, ldx, res, ldr, dtype, M, K, gamma, eps, flags, h, ldh, r, q, ldq, S, d, ldd, None)


def test_norm_qact():
    for dtype in (0, 1, 2):
        assert norm(dtype=dtype) == 0 and norm(dtype=dtype, flags=1, d=None) == 0 and norm(dtype=dtype, res=None, h=None) == 0
    assert norm(K=32768, ldx=32768, ldr=32768, ldh=32768, ldq=32768, ldd=1024) == 0 and norm(M=0, x=None) == 0
    for bad in (dict(K=0), dict(K=240), dict(K=32800), dict(M=-1), dict(M=1 << 22), dict(eps=-1.0), dict(eps=float("nan")), dict(flags=2),
                dict(x=None), dict(gamma=None), dict(q=None), dict(S=None), dict(d=None), dict(ldx=252), dict(ldr=252),
                dict(ldh=252), dict(ldq=252), dict(ldd=7)):
        assert norm(**bad) == -1, bad
    assert norm(dtype=3) == -3 and norm(dtype=-1) == -3
    for bad in (dict(x=P + 8), dict(res=P + 4), dict(h=P + 8), dict(gamma=P + 8), dict(ldx=258), dict(q=P + 2), dict(S=P + 2),
                dict(dtype=1, ldx=260), dict(dtype=1, q=P + 4), dict(dtype=2, ldq=260)):
        assert norm(**bad) == -2, bad


def attn(q=P, qs=(2048, 2048, 128), pk=P, pks=(1024, 128), pv=P, pvs=(1024, 128), np_=100, k=P, ks=(65536, 1024, 128), v=P,
         vs=(65536, 1024, 128), lens=P, T=64, B=2, Lq=1, Hq=16, Hkv=8, D=128, dtype=1, scale=0.1, out=P,
         os=(2048, 2048, 128), weights=None, work=P, nbytes=1 << 40):
    z = lambda x: 0 if x is None else x  # noqa: E731
    return code("otpu_attn_shared", X.ATTN_ARGS.pack(
        X.ATTN_ARGS.size, z(q), *qs, z(pk), *pks, z(pv), *pvs, z(k), *ks, z(v), *vs, z(lens), z(out), *os, z(weights), z(work), nbytes,
        B, Lq, Hq, Hkv, D, np_, T, dtype, scale), None)


def test_attn_shared():
    for dtype in (1, 2):
        for D in (8, 40, 64, 96, 128, 136, 256):
            assert attn(dtype=dtype, D=D) == 0 and attn(dtype=dtype, D=D, weights=P) == 0
    assert attn(np_=0, pk=None, pv=None) == 0 and attn(T=0, k=None, v=None, lens=None) == 0
    assert attn(B=0) == 0 and attn(Lq=0) == 0 and attn(qs=(0, 0, 0)) == 0
    for bad in (dict(Hq=15), dict(Hkv=0), dict(B=-1), dict(Lq=-1), dict(np_=-1), dict(np_=(1 << 30) + 1), dict(T=-1), dict(T=(1 << 30) + 1), dict(D=4), dict(D=264), dict(D=60),
                dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(q=None),
                dict(out=None), dict(work=None), dict(pk=None), dict(pv=None), dict(k=None), dict(v=None), dict(lens=None),
                dict(nbytes=1000), dict(pks=(1 << 22, 128)), dict(ks=(65536, -1024, 128)), dict(B=1 << 20, Lq=1 << 10), dict(B=1 << 18, T=1 << 20)):
        assert attn(**bad) == -1, bad
    assert attn(dtype=0) == -3 and attn(dtype=3) == -3
    for bad in (dict(q=P + 8), dict(out=P + 2), dict(pk=P + 8), dict(pv=P + 8), dict(k=P + 8), dict(v=P + 8), dict(lens=P + 2),
                dict(weights=P + 2), dict(work=P + 128), dict(qs=(2048, 2044, 128)), dict(pks=(1020, 128)),
                dict(vs=(65536, 1024, 124)), dict(os=(2050, 2048, 128))):
        assert attn(**bad) == -2, bad


def test_attn_work_bytes():
    f = X.load().otpu_attn_work_bytes
    for sizes in ((1, 1, 1, 1, 8, 0, 1), (64, 1, 16, 8, 128, 16384, 1024), (8, 512, 16, 8, 128, 8192, 1024), (3, 5, 6, 2, 200, 0, 0)):
        n = f(*sizes)
        B, Lq, Hq, Hkv, D, p, T = sizes
        assert n >= 0 and n % 256 == 0
        assert (n > 4 * B * Lq * Hq * D) == (p + T > 0)
        assert attn(B=B, Lq=Lq, Hq=Hq, Hkv=Hkv, D=D, np_=p, T=T, nbytes=n) == 0
        if n:
            assert attn(B=B, Lq=Lq, Hq=Hq, Hkv=Hkv, D=D, np_=p, T=T, nbytes=n - 1) == -1
    assert f(1, 1, 3, 2, 64, 1, 1) == -1 and f(1, 1, 1, 1, 63, 1, 1) == -1 and f(0, 1, 1, 1, 64, 1, 1) >= 0


def evict(k=P, ks=(65536, 1024, 128), v=P, vs=(65536, 1024, 128), row=128, w=P, pos=P, lens=P, B=2, T=64, H=8, budget=9,
          recent=2, wo=P, po=P, lo=P, work=P, nbytes=1 << 40):
    z = lambda x: 0 if x is None else x  # noqa: E731
    return code("otpu_kv_evict", X.EVICT_ARGS.pack(
        X.EVICT_ARGS.size, z(k), *ks, z(v), *vs, z(w), z(pos), z(lens), z(wo), z(po), z(lo), z(work), nbytes, B, T, H, row, budget,
        recent), None)


def test_structs_of_another_size():
    """A caller built against another header: its struct's first word differs."""
    for name, s in (("otpu_attn_shared", X.ATTN_ARGS), ("otpu_kv_evict", X.EVICT_ARGS)):
        assert code(name, None, None) == -1
        for size in (0, s.size - 8, s.size + 8):
            assert code(name, size.to_bytes(8, "little") + bytes(s.size + 8), None) == -1


def test_kv_evict():
    assert evict(B=1 << 19) == -1 and evict(B=(1 << 19) - 1) == 0
    assert evict() == 0 and evict(budget=64) == 0 and evict(budget=0) == 0 and evict(B=0, lens=None) == 0 and evict(row=16) == 0
    assert evict(T=0, k=None, v=None, w=None, pos=None, wo=None, po=None) == 0
    for bad in (dict(B=-1), dict(T=-1), dict(T=(1 << 30) + 1), dict(H=0), dict(budget=-1), dict(recent=-1), dict(row=8), dict(row=24), dict(row=1 << 21),
                dict(k=None), dict(v=None), dict(w=None), dict(pos=None), dict(lens=None), dict(wo=None), dict(po=None),
                dict(lo=None), dict(work=None), dict(nbytes=64)):
        assert evict(**bad) == -1, bad
    for bad in (dict(k=P + 8), dict(v=P + 8), dict(work=P + 16), dict(ks=(65536, 1032, 128)), dict(vs=(65528, 1024, 128))):
        assert evict(**bad) == -2, bad
    f = X.load().otpu_kv_evict_work_bytes
    for sizes in ((2, 64, 8, 9), (1, 1, 1, 1), (4, 32768, 8, 4096), (3, 100, 2, 99), (5, 0, 1, 3)):
        n = f(*sizes)
        B, T, H, budget = sizes
        assert n >= 8 * B * H * min(max(T - budget, 0), budget) + 4 * B * H
        assert evict(B=B, T=T, H=H, budget=budget, nbytes=n) == 0 and evict(B=B, T=T, H=H, budget=budget, nbytes=n - 1) == -1
    assert f(1, 1, 0, 1) == -1 and f(1, 1, 1, -1) == -1
