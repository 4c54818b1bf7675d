"""mxu.norm_quantize: bit for bit the QACT (fp32.qact) of the row sum with the row factor it gives, the
factor and the sum against float64, the operand in a dot, and refusals.

The factor's bound: K products and sums in fp32 of terms of one sign, each within 2^-24 of its value, in
chains of at most 32 (a thread's elements) + 6 + 16 additions: 60 2^-24 of the mean, halved by the root,
plus the division, root and reciprocal: 2^-18 in all."""
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


def rows(T, rng, M, K, dt):
    x = rng.standard_normal((M, K)).astype(np.float32) * np.exp(rng.standard_normal((M, 1))).astype(np.float32)
    x[:, rng.integers(0, K, 3)] *= 40
    return T.from_numpy(x).to(dt).cuda()


@pytest.mark.parametrize("dt", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("M,K", [(1, 32), (1, 1024), (3, 96), (5, 512), (7, 544), (2, 2048), (65, 1184), (300, 4096),
                                 (3, 8192), (2, 9216), (2, 32768), (1100, 128)])
def test_is_qact_of_the_normed_row(T, dt, M, K):
    from opentpu_amd import fp32, mxu
    say(f"norm {dt} {M} x {K}")
    dt = getattr(T, dt)
    rng = np.random.default_rng(M + K)
    x, res = rows(T, rng, M, K, dt), rows(T, rng, M, K, dt)
    if M > 2:
        res[1] = -x[1]                                     # a row whose sum is 0
    gamma = T.from_numpy((1 + 0.3 * rng.standard_normal(K)).astype(np.float32)).cuda()
    for residual in (res, None):
        for row_mode in (False, True):
            r = T.empty((M,), dtype=T.float32, device="cuda")
            (q, S, d, ranges), h = mxu.norm_quantize(x, gamma, residual, eps=1e-5, row_mode=row_mode, r=r)
            s = x.float() + (residual.float() if residual is not None else 0)
            assert ranges == [K] and T.equal(h, s.to(dt)) and (residual is not None or h is x)
            ref = 1 / np.sqrt(np.mean(s.double().cpu().numpy() ** 2, -1) + 1e-5)
            assert np.all(np.abs(r.double().cpu().numpy() - ref) <= 2.0 ** -18 * ref)
            q1, S1, d1 = fp32.qact(s, 32, row_mode, rscale=r, cscale=gamma)
            assert T.equal(q, q1) and T.equal(S[0], S1) and T.equal(d, d1)


def test_in_place_strides_and_dot(T):
    """h into the residual, rows of a wider tensor, and the operand in a linear."""
    from opentpu_amd import mxu
    rng = np.random.default_rng(2)
    M, K, N = 9, 1024, 256
    w = mxu.QWeight.from_float((0.02 * rng.standard_normal((N, K))).astype(np.float32), "int4")
    gamma = T.from_numpy((1 + 0.3 * rng.standard_normal(K)).astype(np.float32)).cuda()
    for dt in (T.float32, T.bfloat16):
        wide = rows(T, rng, M, 2 * K + 64, dt)
        x, res = wide[:, :K], wide[:, K + 64:]
        want, h0 = mxu.norm_quantize(x.contiguous(), gamma, res.contiguous())
        keep = wide.clone()
        got, h = mxu.norm_quantize(x, gamma, res, h=res)
        assert h is res and T.equal(res, h0) and T.equal(wide[:, :K + 64], keep[:, :K + 64])
        for a, b in zip(got[:3], want[:3]):
            assert T.equal(a, b)
        y = mxu.dot(got, w)
        s = (x.float() + keep[:, K + 64:].float()).double()
        n = s / T.sqrt((s * s).mean(-1, keepdim=True) + 1e-6) * gamma.double()
        from opentpu_amd import quant
        ref = n @ T.from_numpy(quant.dequantize_mxu(w.rows.cpu().numpy(), w.srows.cpu().numpy(), "int4", K)).cuda().T
        # 8-bit activations: half a step of the group's largest value an element, times the weights
        wv = T.from_numpy(np.abs(quant.dequantize_mxu(w.rows.cpu().numpy(), w.srows.cpu().numpy(), "int4", K))).cuda()
        step = n.view(M, K // 32, 32).abs().amax(-1) / 127
        bound = (step.repeat_interleave(32, 1) * 1.01) @ wv.T
        assert bool(((y.double() - ref).abs() <= bound + 1e-6).all())


def test_odd_rows(T):
    """Zeros, subnormal sums, NaN and infinities: what QACT makes of them; other rows are not touched."""
    from opentpu_amd import fp32, mxu
    rng = np.random.default_rng(3)
    M, K = 6, 512
    x = rows(T, rng, M, K, T.float32)
    clean, _ = mxu.norm_quantize(x, T.ones(K, device="cuda"))
    x[0] = 0
    x[1] = 1e-42
    x[2, 5] = float("nan")
    x[3, 7] = float("inf")
    x[4] *= 1e20                                           # squares past fp32's range: the factor is 0
    r = T.empty((M,), device="cuda")
    (q, S, d, _), _ = mxu.norm_quantize(x, T.ones(K, device="cuda"), r=r)
    assert bool(T.isnan(r[2])) and float(r[3]) == 0 and float(r[4]) == 0 and float(r[0]) == pytest.approx(1000.0, rel=1e-6)
    q1, S1, d1 = fp32.qact(x, 32, rscale=r, cscale=T.ones(K, device="cuda"))
    assert T.equal(q, q1) and T.equal(d, d1) and T.equal(S[0].view(T.int32), S1.view(T.int32))
    assert T.equal(q[5], clean[0][5]) and not q[:2].any() and not q[4].any()


def test_refusals(T):
    from opentpu_amd import _lib as X
    from opentpu_amd import mxu
    x = T.zeros((4, 256), device="cuda")
    g = T.ones(256, device="cuda")
    (q, S, d, _), h = mxu.norm_quantize(x[:0], g, x[:0])
    assert q.shape == (0, 256) and h.shape == (0, 256)
    for bad in (lambda: mxu.norm_quantize(x.double(), g), lambda: mxu.norm_quantize(x[0], g),
                lambda: mxu.norm_quantize(x, g[:128]), lambda: mxu.norm_quantize(x, g, x.half()),
                lambda: mxu.norm_quantize(x, g, x[:2]), lambda: mxu.norm_quantize(x, g, x, h=x[:2]),
                lambda: mxu.norm_quantize(x, g, x, h=x.half()), lambda: mxu.norm_quantize(x, g, x, h=x[:1].expand(4, 256)), lambda: mxu.norm_quantize(x, g, r=g[:3]),
                lambda: mxu.norm_quantize(x.T, g[:4]), lambda: mxu.norm_quantize(x.cpu(), g)):
        with pytest.raises(ValueError):
            bad()
    big = T.zeros((1, 32800), device="cuda")
    for bad in (lambda: mxu.norm_quantize(x[:, :240], g[:240]), lambda: mxu.norm_quantize(x[:, :16], g[:16]),
                lambda: mxu.norm_quantize(x, g, eps=-1.0), lambda: mxu.norm_quantize(x, g, eps=float("nan")),
                lambda: mxu.norm_quantize(x[:, 1:225], g[:224]), lambda: mxu.norm_quantize(big, big[0])):
        with pytest.raises(X.OtpuError):
            bad()
