"""The work area that a call of otpu_attn_shared uses: parts by what the call asks for, and the sizes that the call
takes.  Host code alone."""
import os

import pytest

from opentpu_amd import _lib as X

pytestmark = pytest.mark.skipif(not os.path.exists(X.LIB_PATH) or os.path.exists("/dev/kfd"),
                                reason="a built library and no GPU (the calls' addresses are not memory)")
P = 4096
# B, Lq, Hq, Hkv, D, P, T: few rows on a long cache, a draft, a prompt's rows on a prefix, a prompt by itself, odd heads
SIZES = [(64, 8, 32, 8, 64, 0, 32768), (1, 1, 1, 1, 8, 0, 1), (64, 1, 16, 8, 128, 16384, 1024), (16, 7, 16, 8, 128, 8191, 2048),
         (8, 512, 16, 8, 128, 8192, 1024), (1, 131072, 16, 16, 128, 0, 131072), (3, 40, 6, 2, 200, 77, 40), (3, 5, 6, 2, 200, 0, 0)]


def call(sizes, weights, work, nbytes):
    B, Lq, Hq, Hkv, D, n, T = sizes
    row = (Lq * Hq * D, Hq * D, D)
    own = (T * Hkv * D, Hkv * D, D)
    rc = X.load().otpu_attn_shared(X.ATTN_ARGS.pack(
        X.ATTN_ARGS.size, P, *row, P if n else 0, Hkv * D, D, P if n else 0, Hkv * D, D, P if T else 0, *own, P if T else 0, *own,
        P if T else 0, P, *row, P if weights else 0, work, nbytes, B, Lq, Hq, Hkv, D, n, T, X.BF16, 0.1), None)
    return rc if rc in (-1, -2, -3) else 0                # (0: the checks take it, the launch has no device)


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_sizes_that_a_call_takes(sizes):
    any_call = X.load().otpu_attn_work_bytes(*sizes)
    for weights in (0, 1):
        n = X.load().otpu_attn_call_bytes(*sizes, weights)
        assert 0 <= n <= any_call and n % 256 == 0
        assert call(sizes, weights, P, n) == 0 and call(sizes, weights, P, any_call) == 0 and call(sizes, weights, P, any_call + 1) == 0
        for other in (n - 1, n + 1):
            if other < any_call:
                assert call(sizes, weights, P, other) == -1
        assert call(sizes, weights, 0, n) == (-1 if n else 0)


def test_what_a_call_does_not_use_is_not_asked_for():
    """Without weights no scores; without partials, none: what is left, from the sizes of the operands."""
    f = X.load().otpu_attn_call_bytes
    B, Lq, Hq, Hkv, D, n, T = SIZES[0]
    scores = 4 * B * Hq * Lq * T                          # a score a row and own token
    assert f(*SIZES[0], 1) >= scores and f(*SIZES[0], 0) < scores / 8
    for sizes in (SIZES[4], SIZES[5]):                    # rows stored as outputs: the rows' sums for the weights alone
        rows = sizes[0] * sizes[1] * sizes[2]
        assert f(*sizes, 0) == 0 and 4 * rows <= f(*sizes, 1) <= 4 * rows + 256
    assert f(1, 1, 3, 2, 64, 1, 1, 0) == -1 and f(1, 1, 1, 1, 63, 1, 1, 0) == -1
