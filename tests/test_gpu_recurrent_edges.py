"""The gated recurrence at its edges: results that are zero by definition, boundaries out of order in short calls, steps in every
type."""
import pytest
import torch

from lampa_amd.linear_recurrence import gated_recurrence_step
from test_gpu_linear_recurrence import _bounds, _call, _close, _expected, _gpu, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("lens", [[1], [1, 1, 0, 1], 3], ids=str)
def test_decays_without_a_state_before_them_have_no_gradient(lens, dtype):
    """Sequences of one token on no state, the input as it is: h = sigmoid(i) x holds no decay, so the gradients of A and of the decay
    gate are zero, not small."""
    n = lens if isinstance(lens, int) else len(lens)
    shape = (lens, 1) if isinstance(lens, int) else (1, sum(lens))
    t = _inputs(shape, 96, dtype, 40, n, state=False)
    leaves = _gpu(t, grad=True)
    y, last = _call(leaves, "silu", False, None if isinstance(lens, int) else _bounds(lens).cuda())
    names = ["A", "r", "x", "i", "z"]
    grads = torch.autograd.grad([y, last], [leaves[k] for k in names], [torch.ones_like(y), torch.ones_like(last)])
    assert not grads[0].any() and not grads[1].any()
    assert all(g.any() for g in grads[2:])


# D, tokens (no more than a tile: 64 for D = 512, 128 for 100, 256 for 24), boundaries as given on the device, as they are taken
MOVED = [
    (512, 40, [0, 30, 20, 40], [0, 30, 30, 40]),
    (512, 64, [0, 64, 10, 64], [0, 64, 64, 64]),
    (512, 10, [0, 8, 3], [0, 8, 8]),
    (512, 64, [7, -5, 50, 10**12, 20], [0, 0, 50, 64, 64]),
    (100, 128, [0, 128, 0, 128, 127, 128], [0, 128, 128, 128, 128, 128]),
    (100, 1, [0, 0, -1, 1, 0], [0, 0, 0, 1, 1]),
    (24, 256, [0, 200, 100, 150, 256, 3], [0, 200, 200, 200, 256, 256]),
    (24, 200, [0] + [k % 7 * 30 for k in range(150)] + [199], [0] + [min(k, 6) * 30 for k in range(150)] + [199]),
]


@pytest.mark.parametrize("case", MOVED, ids=lambda c: f"{c[0]}-{c[1]}-{len(c[2]) - 1}")
def test_boundaries_out_of_order_in_calls_of_one_tile(case):
    """Boundaries on the device that decrease or lie outside the tokens: the values and gradients of the boundaries they are taken for, every
    final state and every gradient of a state written."""
    D, T, given, taken = case
    n = len(given) - 1
    t = _inputs((1, T), D, torch.float32, 41, n)
    end = taken[-1]
    lens = [b - a for a, b in zip(taken, taken[1:])]
    g = torch.Generator().manual_seed(42)
    dy, dht = torch.randn(1, T, D, generator=g), torch.randn(n, D, generator=g)
    cut = {k: v[:, :end] if k in "xriz" else v for k, v in t.items()}
    want = _expected(cut, lens, "silu", True, dy[:, :end], dht)
    names = ["x", "r", "A", "i", "z", "h0"]
    for bounds in (given, taken):
        leaves = _gpu(t, grad=True)
        y, last = _call(leaves, "silu", True, torch.tensor(bounds).cuda())
        grads = dict(zip(names, torch.autograd.grad([y, last], [leaves[k] for k in names], [dy.cuda(), dht.cuda()])))
        assert not y[:, end:].any() and not any(grads[k][:, end:].any() for k in "xriz")
        _close("y", y[:, :end], *want["y"])
        _close("last", last, *want["last"])
        for k in names:
            _close(k, grads[k][:, :end] if k in "xriz" else grads[k], *want[k])


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["fp16", "fp32"])
@pytest.mark.parametrize("D,act,normalize", [(33, "silu", True), (512, "sigmoid", False), (130, None, True)])
def test_steps_in_the_other_types(D, act, normalize, dtype):
    """The token step against the definition where the other tests run it in bf16: sliced rows, with and without gates."""
    n, T = 3, 5
    t = _inputs((n, T), D, dtype, 43, n, i=act is not None, z=act is not None, sliced=True)
    want = _expected(t, [T] * n, act, normalize)
    g = _gpu(t)
    state = g["h0"].clone()
    for k in range(T):
        at = {m: None if g[m] is None else g[m][:, k] for m in "xriz"}
        y = gated_recurrence_step(at["x"], at["r"], g["A"], state, input_gate=at["i"], gate=at["z"], gate_activation=act,
                                  normalize=normalize)
        assert y.dtype == dtype
        _close("y", y, want["y"][0].reshape(n, T, D)[:, k], want["y"][1].reshape(n, T, D)[:, k], dtype)
    _close("last", state, *want["last"])
