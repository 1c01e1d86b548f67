"""GPU parity of the norms around a block against float64, forward and gradients.

Tolerances: fp32 throughout, rounded once. A norm adds up D squares: its 1 / rms is off by (D / 16 + 8) half-steps (eight channels a lane,
then a tree; sqrt and division correctly rounded). r is off by that through the first norm, y by that again; gradients by
three such sums. `mag` is the same formula on absolute values, which bounds every sum."""
import numpy as np
import pytest
import torch

from lampa_amd import layer_ops as lo
from oracle import state_space as os_

pytestmark = pytest.mark.gpu

HALF32 = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = {None: None, "sigmoid": "sigmoid", "silu": "silu", "swish": "silu"}


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _close(name, got, want, bound):
    if got.dtype != torch.float32:
        f = torch.finfo(got.dtype)
        bound = bound + f.eps / 2 * (np.abs(want) + bound) + f.smallest_normal * f.eps
    err = np.abs(_np(got) - want)
    assert (err <= bound).all(), (name, float(err.max()), float((err / bound).max()))


def _data(shape, dtype, res, gate, post, scale, weight, seed, device):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen).to(device)  # noqa: E731
    D = shape[-1]
    return dict(x=r(*shape).to(dtype), residual=(2 * r(*shape)).to(dtype if res == "same" else torch.float32),
                weight=1 + 0.1 * r(D) if weight else None, post_weight=1 + 0.1 * r(D) if post else None,
                gate=None if gate == "none" else r(*shape).to(dtype) if gate == "token" else r(shape[0], 1, D).to(dtype),
                scale=0.5 + 0.1 * r(D) if scale else None), r(*shape).to(dtype), r(*shape)


def _call(d, act):
    return lo.residual_norm(d["x"], d["residual"], d["weight"], d["post_weight"], d["gate"], act, d["scale"])


def _mag(n, act, dy, dres):
    """Bounds of the terms' magnitudes: 1 / rms factors as they are, everything else absolute."""
    a = {k: None if v is None else np.abs(v) for k, v in n.items()}
    D = n["x"].shape[-1]
    one = np.ones(D)
    pw, w, sc = (one if a[k] is None else a[k] for k in ("post_weight", "weight", "scale"))
    i1 = 1 / np.sqrt((n["x"] ** 2).mean(-1, keepdims=True) + 1e-5) if n["post_weight"] is not None else 1.0
    v, slope = (1.0, 0.0) if n["gate"] is None else (np.abs(n["gate"]), 1.0) if act is None else (1.0, 0.25) if act == "sigmoid" else (
        np.abs(n["gate"]), 1.1)
    am = a["x"] * i1 * pw
    r = a["residual"] + sc * v * am
    true_r = os_.residual_norm(**n, act=act)[1]
    i2 = 1 / np.sqrt((true_r ** 2).mean(-1, keepdims=True) + 1e-5)
    out = {"y": r * i2 * w, "r": r}
    dyw = np.abs(dy) * w
    grow = 1 + (r ** 2).mean(-1, keepdims=True) * i2 ** 2          # how far absolute sums exceed the true ones
    dr = (np.abs(dres) + i2 * dyw * grow + r * i2 ** 3 * (dyw * r).mean(-1, keepdims=True)) * grow
    da = dr * sc * v
    lead = tuple(range(n["x"].ndim - 1))
    out["residual"] = dr
    out["weight"] = (np.abs(dy) * r * i2 * grow).sum(lead)
    out["scale"] = (dr * v * am).sum(lead)
    if n["gate"] is not None:
        dg = dr * sc * am * slope
        out["gate"] = dg if n["gate"].shape == n["x"].shape else dg.sum(1, keepdims=True)
    dn = da * pw
    out["post_weight"] = (da * a["x"] * i1).sum(lead)
    out["x"] = i1 * dn + a["x"] * i1 ** 3 * (dn * a["x"]).mean(-1, keepdims=True) if n["post_weight"] is not None else da
    return out


SHAPES = [(1, 1, 8), (2, 3, 24), (3, 70, 64), (2, 5, 128), (5, 40, 200), (2, 33, 512), (2, 9, 1000), (3, 4, 2048), (1, 3, 2056), (2, 2, 8192)]
OPTIONS = [("same", "none", None, False, False, True), ("fp32", "token", "sigmoid", True, True, True), ("same", "sequence", "silu", True, False, True),
           ("fp32", "token", None, False, True, False), ("same", "sequence", None, False, True, True), ("same", "token", "swish", True, True, False)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_gradients(device, dtype, shape):
    for k, (res, gate, act, post, scale, weight) in enumerate(OPTIONS):
        d, dy, dres = _data(shape, dtype, res, gate, post, scale, weight, sum(shape) + k, device)
        dres = dres.to(d["residual"].dtype)
        y, r = _call(d, act)
        assert y.dtype == dtype and r.dtype == d["residual"].dtype
        leaves = {k: v.detach().requires_grad_(True) for k, v in d.items() if v is not None}
        y2, r2 = _call({**d, **leaves}, act)
        assert torch.equal(y, y2) and torch.equal(r, r2)
        grads = torch.autograd.grad([y2, r2], list(leaves.values()), [dy, dres], retain_graph=True)
        for a, b in zip(grads, torch.autograd.grad([y2, r2], list(leaves.values()), [dy, dres])):
            assert torch.equal(a, b)
        n = {k: _np(v) for k, v in d.items()}
        wy, wr, wg = os_.residual_norm(**n, act=ACTS[act], dy=_np(dy), dres=_np(dres))
        mag = _mag(n, ACTS[act], _np(dy), _np(dres))
        unit = (3 * (shape[-1] / 16 + 8) + 16) * HALF32
        _close("y", y, wy, unit * mag["y"])
        _close("r", r, wr, unit * mag["r"])
        for name, a in zip(leaves, grads):
            rows = shape[0] * shape[1] if a.dim() == 1 or (name == "gate" and gate == "sequence") else 0
            assert a.shape == d[name].shape and a.dtype == d[name].dtype
            _close(name, a, wg[name], (2 * unit + rows * HALF32) * mag[name] + 1e-30)


def test_against_the_plain_norm(device):
    """Without post-norm, gate and scale it is the pre-norm residual add that ``rms_norm`` has."""
    x, r, w = torch.randn(70, 128, device=device).bfloat16(), torch.randn(70, 128, device=device).bfloat16(), torch.rand(128, device=device)
    y, out = lo.residual_norm(x, r, w)
    y2, out2 = lo.rms_norm(x, w, None, r, 1e-5, True)
    assert torch.equal(y, y2) and torch.equal(out, out2)


@pytest.mark.parametrize("dtype", DTYPES)
def test_without_a_residual(device, dtype):
    """The gated norm alone: the same bits as on a residual of zeros, and no second output."""
    d, dy, dres = _data((2, 40, 128), dtype, "same", "token", False, False, True, 7, device)
    d["residual"] = torch.zeros_like(d["residual"])
    leaves = [d[k].requires_grad_(True) for k in ("x", "gate", "weight")]
    y = lo.residual_norm(leaves[0], None, leaves[2], gate=leaves[1], gate_activation="silu")
    y2, _ = lo.residual_norm(leaves[0], d["residual"], leaves[2], gate=leaves[1], gate_activation="silu")
    assert torch.equal(y, y2)
    for a, b in zip(torch.autograd.grad(y, leaves, dy), torch.autograd.grad(y2, leaves, dy)):
        assert torch.equal(a, b)
    with torch.no_grad():
        assert torch.equal(lo.residual_norm(leaves[0], None, leaves[2], gate=leaves[1], gate_activation="silu"), y)


def test_one_gradient_and_strides(device):
    d, dy, dres = _data((2, 30, 64), torch.bfloat16, "same", "token", True, True, True, 1, device)
    leaves = {k: v.detach().requires_grad_(True) for k, v in d.items()}
    y, r = _call(leaves, "silu")
    a = torch.autograd.grad(y, leaves["x"], dy, retain_graph=True)[0]
    b = torch.autograd.grad([y, r], leaves["x"], [dy, torch.zeros_like(r)], retain_graph=True)[0]
    assert torch.equal(a, b)
    a = torch.autograd.grad(r, leaves["gate"], dres.bfloat16(), retain_graph=True)[0]
    b = torch.autograd.grad([y, r], leaves["gate"], [torch.zeros_like(y), dres.bfloat16()])[0]
    assert torch.equal(a, b)
    wide = torch.randn(30, 2, 72, device=device).bfloat16().transpose(0, 1)
    y, r = lo.residual_norm(wide[..., 4:68], wide[..., :64], d["weight"], gate=wide[..., 8:72])
    y2, r2 = lo.residual_norm(wide[..., 4:68].contiguous(), wide[..., :64].contiguous(), d["weight"], gate=wide[..., 8:72].contiguous())
    assert torch.equal(y, y2) and torch.equal(r, r2)


def test_empty_rows_and_rows_that_are_not_finite(device):
    w = torch.rand(64, device=device, requires_grad=True)
    x = torch.zeros(0, 64, device=device, requires_grad=True)
    y, r = lo.residual_norm(x, torch.zeros(0, 64, device=device), w)
    assert y.shape == (0, 64) and not torch.autograd.grad(y.sum(), w)[0].any()
    x = torch.randn(10, 64, device=device)
    res = torch.randn(10, 64, device=device)
    clean = lo.residual_norm(x, res, w.detach(), post_weight=w.detach())
    x[3, 5] = float("inf")
    res[7, 0] = float("nan")
    y, r = lo.residual_norm(x, res, w.detach(), post_weight=w.detach())
    keep = [i for i in range(10) if i not in (3, 7)]
    assert torch.equal(y[keep], clean[0][keep]) and torch.equal(r[keep], clean[1][keep])
    assert torch.isnan(y[7]).all() and not torch.isfinite(r[3]).all()


def test_captured_gradients(device):
    d, dy, dres = _data((2, 50, 512), torch.bfloat16, "fp32", "sequence", True, True, True, 2, device)
    leaves = {k: v.requires_grad_(True) for k, v in d.items()}

    def step(l):
        y, r = _call(l, "sigmoid")
        return [y, r, *torch.autograd.grad([y, r], list(l.values()), [dy, dres])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(leaves)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(leaves)
    for seed in (3, 4, 5):
        new = {k: v.requires_grad_(True) for k, v in _data((2, 50, 512), torch.bfloat16, "fp32", "sequence", True, True, True, seed, device)[0].items()}
        for k in leaves:
            leaves[k].data.copy_(new[k])
        graph.replay()
        for a, b in zip(out, step(new)):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


def test_refusals(device):
    x = torch.zeros(2, 3, 16, device=device).bfloat16()
    with pytest.raises(ValueError, match="one shape"):
        lo.residual_norm(x, x[:1])
    with pytest.raises(ValueError, match="multiple of 8"):
        lo.residual_norm(x[..., :12], x[..., :12])
    with pytest.raises(TypeError, match="residual"):
        lo.residual_norm(x, x.half())
    with pytest.raises(TypeError, match="gate"):
        lo.residual_norm(x, x, gate=x.float())
    with pytest.raises(ValueError, match="gate"):
        lo.residual_norm(x, x, gate=x[:, :2])
    with pytest.raises(ValueError, match="weight"):
        lo.residual_norm(x, x, torch.ones(8, device=device))
    with pytest.raises(ValueError, match="not supported"):
        lo.residual_norm(x, x, gate=x, gate_activation="relu")
