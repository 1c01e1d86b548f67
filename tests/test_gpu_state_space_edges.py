"""Calls of the state-space operators, the convolution and the norms at the borders of what they take: offsets beyond 2^31,
many short sequences, several streams, states changed in place, growth, values that are not finite beside large ones."""
import numpy as np
import pytest
import torch

from lampa_amd import layer_ops as lo
from lampa_amd import state_space as ss
from test_gpu_state_space import DTYPES, _bound, _call, _check, _inputs, _oracle, _to

pytestmark = pytest.mark.gpu
NAMES = ["x", "dt", "A", "B", "C", "D", "dt_bias", "h0"]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_offsets_beyond_32_bits(device, dtype, monkeypatch):
    """The last sequence of a call of 2.4e9 elements comes out as by itself (segments of one length in both calls), and so do its
    gradients."""
    monkeypatch.setattr(ss, "_segment_tokens", lambda *a: 640)
    T, H, P, N, tail = 590000, 64, 64, 8, 1500
    gen = torch.Generator(device=device).manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=gen, device=device, dtype=dtype)  # noqa: E731
    d = dict(x=r(1, T, H, P), dt=r(1, T, H), B=r(1, T, 1, N), C=r(1, T, 1, N))
    shared = dict(A=-torch.rand(H, generator=gen, device=device), D=None, dt_bias=None, h0=None)
    assert d["x"].numel() > 2 ** 31
    cu = torch.tensor([0, T - tail, T], device=device)
    dy = r(1, tail, H, P)
    out = []
    for whole in (True, False):
        e = {k: (t if whole else t[:, T - tail:].clone()).requires_grad_(True) for k, t in d.items()}
        y, ht = _call({**e, **shared}, cu=cu if whole else None)
        g = dy
        if whole:
            g = torch.zeros_like(y)
            g[:, T - tail:] = dy
        grads = torch.autograd.grad(y, list(e.values()), g)
        out.append([y[:, -tail:].detach().clone(), ht[-1:].detach().clone()] + [t[:, -tail:].clone() for t in grads])
        del y, ht, g, grads, e
    for k, a, b in zip(["y", "ht", "x", "dt", "B", "C"], *out):
        assert torch.equal(a, b), k

    # the convolution and the norm over the same rows
    x = d["x"].detach().flatten(2)
    w, bias = torch.randn(H * P, 4, device=device), torch.randn(H * P, device=device)
    out = []
    for whole in (True, False):
        e = (x if whole else x[:, T - tail:].clone()).requires_grad_(True)
        y = lo.causal_conv1d(e, w, bias, activation="silu", cu_seqlens=cu if whole else None)
        y2, last = lo.causal_conv1d(e.detach(), w, bias, activation="silu", cu_seqlens=cu if whole else None, output_final_state=True)
        g = torch.zeros_like(y)
        g[:, -tail:] = dy.flatten(2)
        dx, = torch.autograd.grad(y, e, g)
        h = lo.residual_norm(e.detach(), None, bias)
        out.append([t[:, -tail:].detach().clone() for t in (y, y2, dx, h)] + [last[-1].clone()])
        del e, y, y2, g, dx, h, last
    for a, b in zip(*out):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_short_sequences(device, dtype):
    lens = [k * 7 % 4 for k in range(1500)]
    T, H, P, N = sum(lens), 2, 16, 8
    i = _inputs((1, T), H, P, 1, N, dtype, 60, len(lens))
    gen = torch.Generator().manual_seed(61)
    dy, dht = torch.randn(1, T, H, P, generator=gen).to(dtype), torch.randn(len(lens), H, N, P, generator=gen)
    (y, last, g), (ym, lastm, gm) = _oracle(i, lens, dy=dy, dht=dht)
    d = _to(i, device, grad=True)
    got, ht = _call(d, cu=torch.tensor(np.cumsum([0] + lens), dtype=torch.int32))
    _check("y", got, y, _bound(dtype, 3, y, ym, N), dtype)
    _check("last", ht, last, _bound(dtype, 3, last, lastm, 0, False))
    grads = torch.autograd.grad([got, ht], [d[k] for k in NAMES], [dy.to(device), dht.to(device)])
    for k, a in zip(NAMES, grads):
        wide = {"x": N, "B": P * H, "C": P * H, "h0": 0, "D": T * P}.get(k, N * P + T)
        _check(k, a, g[k], _bound(dtype, 3, g[k], gm[k], wide, k in ("x", "B", "C")), d[k].dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_growing_states(device, dtype):
    """A above zero: e^(0.5) to e^(3) over the sequence."""
    i = _inputs((1, 300), 2, 32, 1, 32, dtype, 62, 1)
    i["A"], i["dt_bias"] = torch.tensor([0.05, 0.1]), None
    i["dt"] = (i["dt"].abs() * 0.1).to(dtype)
    dy = torch.randn(1, 300, 2, 32, generator=torch.Generator().manual_seed(63)).to(dtype)
    (y, last, g), (ym, lastm, gm) = _oracle(i, [300], softplus=False, dy=dy)
    d = _to(i, device, grad=True)
    got, ht = _call(d, softplus=False)
    _check("y", got, y, _bound(dtype, 300, y, ym, 32), dtype)
    _check("last", ht, last, _bound(dtype, 300, last, lastm, 0, False))
    names = [k for k in NAMES if k != "dt_bias"]
    for k, a in zip(names, torch.autograd.grad(got, [d[k] for k in names], dy.to(device))):
        wide = {"x": 32, "B": 64, "C": 64, "h0": 0, "D": 300 * 32}.get(k, 32 * 32 + 300)
        _check(k, a, g[k], _bound(dtype, 300, g[k], gm[k], wide, k in ("x", "B", "C")), d[k].dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("state_type", [torch.float32, torch.bfloat16])
def test_gradients_of_the_final_state_alone(device, dtype, state_type):
    """No gradient for y; the initial state in another type, its heads out of order."""
    i = _inputs((2, 150), 4, 16, 2, 24, dtype, 64, 2)
    i["h0"] = i["h0"].to(state_type)
    dht = torch.randn(2, 4, 24, 16, generator=torch.Generator().manual_seed(65))
    (_, last, g), (_, lastm, gm) = _oracle(i, [150, 150], dy=torch.zeros(2, 150, 4, 16), dht=dht)
    d = _to(i, device, grad=True)
    turned = d["h0"].detach().permute(1, 0, 3, 2).contiguous().permute(1, 0, 3, 2).requires_grad_(True)
    d["h0"] = turned
    _, ht = _call(d)
    _check("last", ht, last, _bound(dtype, 150, last, lastm, 0, False))
    names = ["x", "dt", "A", "B", "dt_bias", "h0"]
    for k, a in zip(names, torch.autograd.grad(ht, [d[k] for k in names], dht.to(device))):
        assert a.dtype == d[k].dtype
        wide = {"x": 24, "B": 16 * 2, "h0": 0}.get(k, 24 * 16 + 150)
        _check(k, a, g[k], _bound(dtype, 150, g[k], gm[k], wide, k in ("x", "B")), d[k].dtype)


def test_a_column_that_is_not_finite_beside_large_states(device):
    """fp16: states beyond the type's range are scaled into it; a column of infinities must not take that scale away from the
    others. (It does not change what the scale of the others is, so their bits stay.)"""
    i = _inputs((1, 128), 1, 64, 1, 32, torch.float16, 66, 1, state=False)
    i["x"] = (i["x"] * 300).half()
    i["B"] = (i["B"] * 300).half()
    i["C"] = (i["C"] * 1e-4).half()
    i["A"], i["D"] = torch.tensor([-0.01]), None
    clean, state = _call(_to(i, device))
    assert state.abs().max() > 65504
    column = state[0, 0].abs().max(0).values.argmin().item()  # not the one that sets the scale
    j = dict(i, x=i["x"].clone())
    j["x"][0, 63, 0, column] = float("inf")  # the last token of a chunk: chunks stay as they were
    bad, _ = _call(_to(j, device))
    others = [p for p in range(64) if p != column]
    assert torch.isfinite(clean).all() and torch.equal(bad[:, :63], clean[:, :63])
    assert torch.isfinite(bad[..., others]).all() and not torch.isfinite(bad[:, 63:, :, column]).any()
    (y, _, _), (ym, _, _) = _oracle(i, [128])
    for out in (clean, bad):
        _check("y", out[..., others], y.reshape(1, 128, 1, 64)[..., others], _bound(torch.float16, 128, y, ym, 32).reshape(
            1, 128, 1, 64)[..., others], torch.float16)


@pytest.mark.parametrize("dtype", DTYPES)
def test_two_streams_at_once(device, dtype):
    work = []
    for seed in (70, 71):
        d = _to(_inputs((1, 2500), 4, 64, 1, 64, dtype, seed, 1), device, grad=True)
        work.append((d, torch.randn(1, 2500, 4, 64, device=device).to(dtype)))

    def run(d, dy):
        y, ht = _call(d)
        out = [y, ht, *torch.autograd.grad(y, [d[k] for k in NAMES], dy)]
        z = lo.causal_conv1d(d["x"].flatten(2), d["A"].repeat_interleave(256).reshape(256, 4), activation="silu")
        n, r = lo.residual_norm(z, d["x"].flatten(2), gate=d["x"].flatten(2), gate_activation="silu")
        return out + [z, n, r, *torch.autograd.grad([z, n], [d["x"], d["A"]], [dy.flatten(2), dy.flatten(2)])]

    want = [run(*w) for w in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(3):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(run(*work[k]))
    torch.cuda.synchronize()
    for k in (0, 1):
        for again in got[k]:
            for a, b in zip(again, want[k]):
                assert torch.equal(a, b)


def test_states_changed_in_place_are_noticed(device):
    """A step moves on a state that a backward still needs: the backward raises instead of using the new one."""
    d = _to(_inputs((1, 700), 2, 64, 1, 64, torch.bfloat16, 72, 1), device, grad=True)
    y, ht = _call(d)
    with torch.no_grad():
        ss.state_space_step(d["x"][:, 0], d["dt"][:, 0], d["A"], d["B"][:, 0], d["C"][:, 0], ht)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), d["x"])
    x = torch.randn(2, 9, 16, device=device, requires_grad=True)
    w, cache = torch.randn(16, 4, device=device), torch.randn(2, 16, 4, device=device)
    y = lo.causal_conv1d(x, w, initial_state=cache)
    lo.causal_conv1d_step(x[:, 0].detach(), cache, w)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.inference_mode():  # tensors without a counter
        state = torch.zeros(1, 2, 64, 64, device=device)
        ss.state_space_step(d["x"][:, 0], d["dt"][:, 0], d["A"], d["B"][:, 0], d["C"][:, 0], state)
        assert state.any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,D", [(3, 8), (5, 64), (301, 200), (7, 512), (2, 640), (1, 1032)])
def test_norm_without_eps(device, dtype, rows, D):
    """eps = 0: rows that a workgroup has beside the last one are no rows of zeros."""
    gen = torch.Generator().manual_seed(D)
    t = [torch.randn(*s, generator=gen).to(dtype).to(device).requires_grad_(True) for s in ((rows, D), (rows, D), (D,), (D,), (rows, D), (D,))]
    call = lambda x, r, w, pw, g, sc: lo.residual_norm(x, r, w, pw, g, "silu", sc, eps=0.0)  # noqa: E731
    y, r = call(*t)
    grads = torch.autograd.grad([y, r], t, [torch.ones_like(y), torch.ones_like(r)])
    wide = [v.detach().double().requires_grad_(True) for v in t]
    x, res, w, pw, g, sc = wide
    m = res + sc * torch.nn.functional.silu(g) * x / (x * x).mean(-1, keepdim=True).sqrt() * pw
    n = m / (m * m).mean(-1, keepdim=True).sqrt() * w
    want = torch.autograd.grad([n, m], wide, [torch.ones_like(n), torch.ones_like(m)])
    # sums over D of fp32 terms and over the rows; the terms' magnitude is a few times the largest of them; the output's rounding
    f = torch.finfo(dtype)
    for a, b in zip([y, r, *grads], [n, m, *want]):
        top = b.abs().max().item() + 1
        assert torch.isfinite(a).all()
        assert (a.double() - b).abs().max().item() <= 64 * (D + rows) * 2.0 ** -24 * top + f.eps / 2 * top


def test_convolution_of_nothing_trains(device):
    w, b = (torch.randn(16, 4, device=device, requires_grad=True), torch.randn(16, device=device, requires_grad=True))
    for shape in ((2, 0, 16), (0, 5, 16)):
        x = torch.zeros(*shape, device=device, requires_grad=True)
        y = lo.causal_conv1d(x, w, b, activation="silu")
        dx, dw, db = torch.autograd.grad(y.sum(), [x, w, b])
        assert dx.shape == shape and not dw.any() and not db.any()
