"""A traced call is in the graph as the operator, not as the empty tensor that its kernel would have filled. The library is replaced here;
nothing is launched."""
import contextlib
import struct

import pytest
import torch

from lampa_amd import feed_forward as ff
from lampa_amd import linear_recurrence as lr


read = []  # where the operators were told to read x


class Library:
    def __getattr__(self, name):
        def call(first, *rest):
            read.append(struct.unpack_from("=Q", first)[0] if isinstance(first, bytes) else first)
            return 0
        return call


@pytest.fixture(autouse=True)
def replaced(monkeypatch):
    for module in (ff, lr):
        monkeypatch.setattr(module, "_same_device", lambda *args: 0)
        monkeypatch.setattr(module, "_on_device", lambda index: contextlib.nullcontext())
        monkeypatch.setattr(module, "stream_of", lambda t: 0)
        monkeypatch.setattr(module._capi, "lib", Library)
    monkeypatch.setattr(lr, "_sizes", lambda *args: (2, 256))


W = [torch.randn(8, 16), torch.randn(8, 16), torch.randn(16, 8)]
A = -torch.rand(16)
CALLS = {
    "_GatedFeedForward": lambda x: ff.gated_feed_forward(x, *W),
    "_GatedRecurrence": lambda x: lr.gated_recurrence(x[None], x[None], A)[0],
    "_Step": lambda x: lr.gated_recurrence_step(x, x, A, torch.zeros(4, 16)),
}


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("grad", [False, True])
def test_the_operator_is_in_the_graph(name, grad):
    with torch.set_grad_enabled(grad):
        graph = torch.jit.trace(CALLS[name], (torch.randn(4, 16),), check_trace=False)
    (out,) = graph.graph.outputs()
    assert f"^{name}" in str(graph.graph) and "aten::empty" not in str(out.node())
    for other in (torch.randn(4, 16), torch.randn(4, 16)):  # run on other tensors, it reads those
        read.clear()
        graph(other)
        assert other.data_ptr() in read


def test_a_modules_weights_without_gradients_go_to_the_launcher(monkeypatch):
    applied = []
    monkeypatch.setattr(ff._GatedFeedForward, "apply", lambda *args: applied.append(args))
    x, weights = torch.randn(4, 16), [torch.nn.Parameter(w) for w in W]
    ff.gated_feed_forward(x, *weights)
    assert len(applied) == 1
    with torch.no_grad():
        assert ff.gated_feed_forward(x, *weights).shape == x.shape and len(applied) == 1
        torch.func.vmap(lambda t: (ff.gated_feed_forward(x, *weights), t)[1])(x)
    assert len(applied) == 2
