"""The limits that include/otpu.h states for the calls between the linears: the last size that is taken, the first that is not.
Host code alone."""
import os

import pytest

from opentpu_amd import _lib as X

pytestmark = pytest.mark.skipif(not os.path.exists(X.LIB_PATH) or os.path.exists("/dev/kfd"),
                                reason="a built library and no GPU (the calls' addresses are not memory)")
P = 4096


def attn(B, Lq, Hq, Hkv, D, n, T):
    """The checks take the sizes: the work area's functions and the call alike."""
    L = X.load()
    sizes = (B, Lq, Hq, Hkv, D, n, T)
    own = (8, 8, 8)
    rc = L.otpu_attn_shared(X.ATTN_ARGS.pack(
        X.ATTN_ARGS.size, P, 8, 8, 8, P if n else 0, 8, 8, P if n else 0, 8, 8, P if T else 0, *own, P if T else 0, *own, P if T else 0,
        P, 8, 8, 8, 0, P, 1 << 60, *sizes, X.BF16, 0.1), None) not in (-1, -2, -3)
    assert rc == (L.otpu_attn_work_bytes(*sizes) >= 0) == (L.otpu_attn_call_bytes(*sizes, 1) >= 0)
    return rc


def test_attn_shared():
    # rows
    assert attn(256, 2048, 16, 8, 64, 100, 0) and not attn(256, 2049, 16, 8, 64, 100, 0)
    assert attn(1, 1 << 18, 32, 8, 128, 0, 1) and not attn(1, (1 << 18) + 1, 32, 8, 128, 0, 1)
    # a prefix
    assert attn(1, 1, 1, 1, 64, 1 << 30, 0) and not attn(1, 1, 1, 1, 64, (1 << 30) + 1, 0)
    # caches: one, and a batch's
    assert attn(1, 1, 1, 1, 64, 0, (1 << 29) - 32) and not attn(1, 1, 1, 1, 64, 0, (1 << 29) - 31)
    assert attn(256, 1, 8, 8, 128, 0, 262112) and not attn(256, 1, 8, 8, 128, 0, 262113)


def test_norm_qact():
    def norm(M, K):
        return X.load().otpu_norm_qact(P, K, None, 0, 0, M, K, P, 1e-6, 0, None, 0, None, P, K, P, P, K // 32, None) not in (-1, -2, -3)
    assert norm((1 << 22) - 1, 32) and not norm(1 << 22, 32)
    assert norm(1, 32768) and not norm(1, 32800)


def test_kv_evict():
    def evict(B, T, H, row):
        return X.load().otpu_kv_evict(X.EVICT_ARGS.pack(X.EVICT_ARGS.size, P, 16, 16, 16, P, 16, 16, 16, P, P, P, P, P, P, P, 1 << 60, B, T,
                                                        H, row, 3, 0), None) not in (-1, -2, -3)
    assert evict((1 << 22) - 1, 8, 1, 16) and not evict(1 << 22, 8, 1, 16) and not evict(1 << 19, 8, 8, 16)
    assert evict(1, 1 << 30, 1, 16) and not evict(1, (1 << 30) + 1, 1, 16)
    assert evict(1, 8, 1, 1 << 20) and not evict(1, 8, 1, (1 << 20) + 16)
