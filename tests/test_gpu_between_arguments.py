"""Arguments of the calls between the linears that are out of 32 bits or of another rank: taken for what they mean, or refused
with the call's own error."""
import sys

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


def test_budget_and_recent_past_32_bits(T):
    """A budget or a number of newest positions past any cache is every slot."""
    from opentpu_amd import _lib as X
    from opentpu_amd import attention
    k = T.randn((2, 9, 2, 8), device="cuda")
    w = T.rand((2, 2, 9), device="cuda")
    pos = T.arange(9, dtype=T.int32, device="cuda").expand(2, 2, 9).contiguous()
    lens = T.tensor([9, 4], dtype=T.int32, device="cuda")

    def run(budget, recent):
        a, b = k.clone(), k.clone()
        return (a, b, *attention.evict(a, b, w, pos, lens, budget, recent))

    for many in (1 << 31, 1 << 32, (1 << 32) + 5, sys.maxsize, 1 << 70):
        for args, same in (((many, 0), (9, 0)), ((5, many), (5, 9)), ((many, many), (9, 9))):
            assert all(T.equal(x, y) for x, y in zip(run(*args), run(*same))), args
    assert all(T.equal(x, y) for x, y in zip(run(np.int64(5), np.int32(2)), run(5, 2)))
    for bad in ((-1 << 40, 0), (5, -1 << 40), (-1, 0)):
        with pytest.raises(X.OtpuError):
            run(*bad)
    for bad in ((5.0, 0), (5, 1.5), ("5", 0)):
        with pytest.raises(TypeError):
            run(*bad)


def test_other_ranks(T):
    from opentpu_amd import attention
    q, p, k = T.zeros((2, 1, 4, 64), device="cuda").half(), T.zeros((5, 2, 64), device="cuda").half(), T.zeros((2, 7, 2, 64), device="cuda").half()
    lens = T.zeros((2,), dtype=T.int32, device="cuda")
    flat, one = T.zeros((64,), device="cuda").half(), T.zeros((), device="cuda").half()
    for x in (flat, one, k[0], p[0]):
        for bad in (lambda: attention.shared(q, None, None, x, x, lens), lambda: attention.shared(q, p, p, x, k, lens),
                    lambda: attention.shared(q, p, p, k, x, lens), lambda: attention.shared(q, p, p, k, k, x),
                    lambda: attention.evict(k, x, T.zeros((2, 2, 7), device="cuda"), lens, lens, 3)):
            with pytest.raises(ValueError):
                bad()
    for x in (flat, one, k, p[0]):
        for bad in (lambda: attention.shared(q, x, x, None, None, None), lambda: attention.shared(q, x, p, k, k, lens),
                    lambda: attention.shared(q, p, x, k, k, lens)):
            with pytest.raises(ValueError):
                bad()
