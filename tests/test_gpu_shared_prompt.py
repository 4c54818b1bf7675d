"""A batch on a shared prompt (shared_prompt.Batch): the same layers with the attention's definition in
float64 over each sequence's whole history in place of attention.shared, and its caches after evictions."""
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


def plain(T, q, k, v):
    """softmax(q k / sqrt(D)) v in float64: q [B, L, Hq, D], k, v [B, n, H, D], the L newest the queries'."""
    B, L, Hq, D = q.shape
    n, H = k.shape[1], k.shape[2]
    q = q.double().view(B, L, H, Hq // H, D).permute(0, 2, 1, 3, 4).reshape(B, H, -1, D)
    k, v = (x.double().permute(0, 2, 1, 3).contiguous() for x in (k, v))
    s = (q @ k.transpose(2, 3).contiguous() * D ** -0.5).view(B, H, L, -1, n)
    seen = T.arange(n, device="cuda") <= T.arange(n - L, n, device="cuda")[:, None]
    s = s.masked_fill(~seen[:, None], -float("inf")).softmax(-1)
    o = (s.view(B, H, -1, n) @ v).view(B, H, L, -1, D)
    return o.permute(0, 2, 1, 3, 4).reshape(B, L, Hq, D)


def rows(rng, T, *shape):
    return T.from_numpy(rng.standard_normal(shape).astype(np.float32)).cuda()


@pytest.mark.parametrize("P", [0, 37])
def test_against_each_sequence_alone(T, P):
    """No eviction: each step's rows against the layers run with the plain attention over prefix and own
    tokens.  Both round the attention's output to bfloat16 (2^-9 of it in the mean square at most, twice
    with the rounded weights) and quantize what follows to 8 bits: 2 layers stay within 3%."""
    from opentpu_amd import shared_prompt as SP
    rng = np.random.default_rng(1)
    shape = SP.Shape(hidden=256, heads=4, kv_heads=2, head=64, F=512, layers=2)
    layers = SP.random_layers(shape, "int8")
    B = 3
    prompt = rows(rng, T, P, 256)
    batch = SP.Batch(layers, shape, prompt, B, 24, 20)
    ref = SP.Batch(layers, shape, prompt[:0], B, 24, 20)
    past = [None] * 2

    def attend(i, q, k, v):
        k, v = (k, v) if past[i] is None else (T.cat([past[i][0], k], 1), T.cat([past[i][1], v], 1))
        past[i] = k, v
        return plain(T, q, k, v).to(q.dtype)

    if P:
        ref._run(prompt.expand(B, P, 256), 0, attend)
    at = P
    for L in (1, 1, 5, 1, 3):
        x = rows(rng, T, B, L, 256)
        y, want = batch.step(x), ref._run(x, at, attend)
        at += L
        err = float((y - want).norm() / want.norm())
        print("step", P, L, err, flush=True)
        assert err < 0.03
    assert batch.used == 11 and int(batch.lens[0]) == 11


def test_evicts_when_full(T):
    """Past the slots each head keeps the budget's tokens, the newest among them, with the positions and
    rows that were written, and the weights that steps add to."""
    from opentpu_amd import shared_prompt as SP
    rng = np.random.default_rng(2)
    shape = SP.Shape(hidden=256, heads=4, kv_heads=2, head=64, F=512, layers=2)
    B, slots, budget, recent = 2, 12, 8, 3
    batch = SP.Batch(SP.random_layers(shape, "int4"), shape, rows(rng, T, 20, 256), B, slots, budget, recent)
    written = {}
    for t in range(30):
        batch.step(rows(rng, T, B, 1, 256))
        n = batch.used
        for i, c in enumerate(batch.caches):
            written[i, 20 + t] = c.k[:, n - 1].clone()
            pos = c.pos[:, :, :n].cpu().numpy()
            m = min(n, recent)
            assert (np.sort(pos, -1)[..., -m:] == np.arange(21 + t - m, 21 + t)).all()
            assert (c.pos[:, :, n:] == -1).all() and (c.weights[:, :, n:] == 0).all() and bool((c.weights[:, :, :n] > 0).all())
            for b in range(B):
                for h in range(2):
                    assert len(set(pos[b, h])) == n
                    for j in (0, n // 2, n - 1):
                        assert T.equal(c.k[b, j, h], written[i, int(pos[b, h, j])][b, h])
        assert int(batch.lens[0]) == n <= slots
    sys.stdout.flush()


def test_refusals(T):
    from opentpu_amd import shared_prompt as SP
    rng = np.random.default_rng(3)
    shape = SP.Shape(hidden=256, heads=4, kv_heads=2, head=64, F=512, layers=1)
    layers = SP.random_layers(shape, "int4")
    for budget, recent in ((8, 0), (4, 5), (4, -1)):
        with pytest.raises(ValueError):
            SP.Batch(layers, shape, rows(rng, T, 0, 256), 2, 8, budget, recent)
    batch = SP.Batch(layers, shape, rows(rng, T, 0, 256), 2, 8, 4)
    with pytest.raises(ValueError):
        batch.step(rows(rng, T, 2, 9, 256))
