"""shared_prompt.Batch.step: a refused call leaves the batch as it was."""
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


def state(batch):
    return [batch.used, batch.position, batch.lens.clone()] + \
        [x.clone() for c in batch.caches for x in (c.k, c.v, c.weights, c.pos)]


def test_a_refused_step_changes_nothing(T):
    from opentpu_amd import shared_prompt as SP
    rng = np.random.default_rng(4)
    shape = SP.Shape(hidden=256, heads=4, kv_heads=2, head=64, F=512, layers=2)

    def rows(*n):
        return T.from_numpy(rng.standard_normal((*n, 256)).astype(np.float32)).cuda()

    B, slots, budget = 2, 12, 5
    layers = SP.random_layers(shape, "int4")
    batch = SP.Batch(layers, shape, rows(9), B, slots, budget)
    for c in batch.caches:
        c.k.zero_(), c.v.zero_()                           # (places in no use: comparable)
    for _ in range(8):
        batch.step(rows(B, 1))
    assert batch.used == 8 > budget
    before = state(batch)
    # 8 tokens do not fit behind 8, nor behind the budget's 5; rows of another batch, width or form
    for x in (rows(B, 8), rows(B, 13), rows(1, 1), rows(B + 1, 1), rows(B, 1)[..., :128], rows(B)):
        with pytest.raises(ValueError):
            batch.step(x)
        now = state(batch)
        assert now[:2] == before[:2] and all(T.equal(a, b) for a, b in zip(now[2:], before[2:])), tuple(x.shape)
    batch.step(rows(B, 7))                                 # evicts, and fits exactly
    assert batch.used == slots
