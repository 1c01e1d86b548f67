"""Copies of operands live until the kernels that read them are launched. The C entry points are replaced here; nothing is launched."""
import contextlib
import gc
import weakref

import pytest
import torch

from lampa_amd import linear_recurrence as lr


@pytest.mark.parametrize("backward", [False, True])
def test_copies_live_until_the_launch(monkeypatch, backward):
    made, alive = [], []

    def noted(function, at):
        def call(*args):
            out = function(*args)
            t = out[at] if at is not None else out
            if t is not None and t.data_ptr() not in inputs:
                made.append(weakref.ref(t))
            return out
        return call

    class Library:
        def __getattr__(self, name):
            def call(*args):
                gc.collect()
                alive.extend(r() is not None for r in made)
                return 0
            return call

    torch.manual_seed(0)
    x, r, i, z = (torch.randn(8, 2, 3).transpose(0, 1) for _ in range(4))  # [2, 8, 3], tokens apart unevenly: copied
    A, h0 = -torch.rand(3).double(), torch.randn(2, 3).half()
    dht = torch.randn(3, 2).t()
    inputs = {t.data_ptr() for t in (x, r, i, z, A, h0, dht)}
    monkeypatch.setattr(lr, "_rows", noted(lr._rows, 0))
    monkeypatch.setattr(lr, "_plain_f32", noted(lr._plain_f32, None))
    monkeypatch.setattr(lr, "_sizes", lambda *args: (2, 256))
    monkeypatch.setattr(lr._capi, "lib", Library)
    monkeypatch.setattr(lr, "stream_of", lambda t: 0)
    monkeypatch.setattr(lr, "_on_device", lambda index: contextlib.nullcontext())
    if backward:
        lr._scan_backward(x, r, A, i, z, 0, True, h0, None, torch.empty(2, 3), torch.randn(2, 8, 3), dht)
    else:
        lr._scan_launch(x, r, A, i, z, 0, True, h0, True, None, keep=True)
    assert len(made) == (7 if backward else 6) and alive == [True] * len(made)
