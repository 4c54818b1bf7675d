"""attn_shared's scale at the ends of its range: the kernels hold scale * log2(e) in fp32, where a positive scale under half of
the least subnormal number is 0, and 0 times the -inf of a key that a row does not see no number."""
import os

import numpy as np
import pytest

from opentpu_amd import _lib as X

P = 4096


@pytest.mark.skipif(not os.path.exists(X.LIB_PATH) or os.path.exists("/dev/kfd"),
                    reason="a built library and no GPU (the call's addresses are not memory)")
def test_a_scale_that_is_0_in_fp32_is_refused():
    for scale, taken in ((5e-324, False), (1e-60, False), (4.8e-46, False), (5e-46, True), (1e-40, True), (1e-3, True), (1e30, True),
                         (1.1e30, False)):
        assert bool(np.float32(scale * 1.4426950408889634) > 0) == (taken or scale > 1)
        rc = X.load().otpu_attn_shared(X.ATTN_ARGS.pack(
            X.ATTN_ARGS.size, P, 64, 64, 64, 0, 0, 0, 0, 0, 0, P, 512, 64, 64, P, 512, 64, 64, P, P, 64, 64, 64, 0, P, 1 << 40,
            2, 1, 1, 1, 64, 0, 8, X.BF16, scale), None)
        assert (rc != -1) == taken, scale


@pytest.mark.gpu
def test_the_least_scale_is_a_mean():
    import torch as T
    from opentpu_amd import attention
    g = T.Generator("cuda").manual_seed(1)
    B, n, D = 3, 45, 64
    q, k, v = (T.randn(s, generator=g, device="cuda").bfloat16() for s in ((B, 4, 2, D), (B, n, 1, D), (B, n, 1, D)))
    lens = T.tensor([4, 20, n], dtype=T.int32, device="cuda")
    got = attention.shared(q, None, None, k, v, lens, scale=5e-46)
    for b, m in enumerate(lens.tolist()):
        for i in range(4):
            want = v[b, :m - 3 + i, 0].double().mean(0)
            # weights of 1 over a whole sum: the output's rounding, and the fp32 sums of at most 45 terms
            assert bool(((got[b, i].double() - want).abs() <= 2.0 ** -8 * want.abs() + 45 * 2.0 ** -24 * 5).all())
