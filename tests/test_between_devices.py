"""The calls between the linears and tensors on a device that is not the current one: refused before anything is queued
(the current stream is the current device's).  Without a device: host tensors that say where they are, and a call that is
recorded."""
import os

import pytest
import torch

from opentpu_amd import _lib as X
from opentpu_amd import attention, mxu

pytestmark = pytest.mark.skipif(not os.path.exists(X.LIB_PATH), reason="libotpu_amd.so not built")


class On(torch.Tensor):
    """A host tensor that says it is on device 1."""

    def get_device(self):
        return 1


def on(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype).as_subclass(On)


@pytest.fixture
def calls(monkeypatch):
    made = []
    monkeypatch.setattr(X, "_T", torch)
    monkeypatch.setattr(X, "call", lambda name, *args: made.append((name, args[-1].value)))
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 64 + device, raising=False)
    monkeypatch.setattr(mxu, "_operand", lambda *a: a)
    return made


def everything():
    q, pk, k = on(2, 1, 4, 64), on(5, 2, 64), on(2, 7, 2, 64)
    lens = on(2, dtype=torch.int32)
    w, pos = on(2, 2, 7, dtype=torch.float32), on(2, 2, 7, dtype=torch.int32)
    x, g = on(3, 64, dtype=torch.float32), on(64, dtype=torch.float32)
    return (lambda: attention.shared(q, pk, pk, k, k, lens), lambda: attention.evict(k, on(2, 7, 2, 64), w, pos, lens, 3),
            lambda: mxu.norm_quantize(x, g, on(3, 64, dtype=torch.float32)))


def test_another_device_is_refused(calls, monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    for call in everything():
        with pytest.raises(ValueError, match="cuda:1"):
            call()
    assert not calls


def test_the_current_devices_stream(calls, monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    for call in everything():
        call()
    assert calls == [("otpu_attn_shared", 65), ("otpu_kv_evict", 65), ("otpu_norm_qact", 65)]
