"""GPU parity of the gated linear recurrence, forward, gradients and token step, against the float64 token loop.

Tolerances follow the roundings, with HALF32 = 2^-24 and the gates within 5 (|log a| within 2): a sigmoid is off by its exponent's
rounding (at most 5 half-steps) and 3 more, a decay by the 9 of its exponent times |log a| and 2, an input by its sigmoid and
its m and 3 products, under 24 together; every token so adds at most C = 32 half-steps of the magnitude at hand (the same
recurrence on absolute values), which the later tokens' decays carry on: err_t = a_t err_{t-1} + C HALF32 mag_t. Gradients
combine two such quantities and 64 more half-steps. What is returned in 16 bits is rounded once more, half a step of its value."""
import numpy as np
import pytest
import torch

from lampa_amd import _capi
from lampa_amd.linear_recurrence import gated_recurrence, gated_recurrence_step
from oracle import linear_recurrence as ol

pytestmark = pytest.mark.gpu

HALF32, C = 2.0 ** -24, 32


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _inputs(shape, D, dtype, seed, n_seq, i=True, z=True, state=True, sliced=False, rate=2.0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen).clamp(-5, 5)  # noqa: E731
    names = ["x", "r", "i", "z"]
    if sliced:  # columns of one wider tensor
        parts = r(*shape, 4 * D + 6).to(dtype).split([D, D, D, D, 6], dim=-1)
        t = dict(zip(names, parts))
    else:
        t = {k: r(*shape, D).to(dtype) for k in names}
    if not i:
        t["i"] = None
    if not z:
        t["z"] = None
    # from a memory of thousands of tokens to one of less than one
    t["A"] = -rate * 10.0 ** (-3.5 * torch.rand(D, generator=gen))
    t["h0"] = r(n_seq, D) if state else None
    return t


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _flat(t):
    return None if t is None else _np(t).reshape(-1, t.shape[-1])


def _expected(t, lens, act, normalize, dy=None, dht=None):
    """{name: (value, bound without the output's own rounding)}."""
    x, r, i, z, A, h0 = _flat(t["x"]), _flat(t["r"]), _flat(t["i"]), _flat(t["z"]), _np(t["A"]), _np(t["h0"])
    n = x.shape[0]
    sr, la, a, si, m = ol.pieces(x, r, A, i, normalize)
    mag = np.abs(m * si * x)
    h, last = ol.run(a, m * si * x, h0, lens)
    magh, maglast = ol.run(a, mag, None if h0 is None else np.abs(h0), lens)
    errh, errlast = ol.run(a, C * HALF32 * magh, None, lens)
    value, slope = (np.ones((n, x.shape[1])), np.zeros((n, x.shape[1]))) if z is None else ol.act(act, z)
    out = {"y": (h * value, errh * np.abs(value) + 12 * HALF32 * np.abs(h * value)), "last": (last, errlast + C * HALF32 * maglast)}
    if dy is None:
        return out
    dyn, dl = _flat(dy), _np(dht)
    G, first = ol.run_back(a, dyn * value, dl, lens)
    magG, magfirst = ol.run_back(a, np.abs(dyn * value), None if dl is None else np.abs(dl), lens)
    errG, errfirst = ol.run_back(a, C * HALF32 * magG, None, lens)
    g = ol.scan_grads(x, r, A, i, z, act, normalize, h0, lens, dyn, dl)
    prev, magprev = ol.before(h, h0, lens), ol.before(magh, None if h0 is None else np.abs(h0), lens)
    errprev = ol.before(errh, None, lens)
    through = np.abs(si * x) * a * a / m if normalize else 0.0
    magdla = magG * (a * magprev + through)
    errdla = errG * (a * magprev + through) + magG * a * errprev + 64 * HALF32 * magdla
    out["x"] = (g["x"], errG * m * si + 64 * HALF32 * magG * m * si)
    out["r"] = (g["r"], (errdla + 16 * HALF32 * magdla) * np.abs(la) * (1 - sr) + 16 * HALF32 * np.abs(la) * sr * magdla)
    # a sum of n values in fp32: at most n half-steps of their magnitudes
    out["A"] = (g["A"], ((errdla + 16 * HALF32 * magdla) * sr).sum(0) + n * HALF32 * (magdla * sr).sum(0))
    if i is not None:
        k = m * np.abs(x) * si
        out["i"] = (g["i"], (errG + 64 * HALF32 * magG) * k * (1 - si) + 16 * HALF32 * magG * k * si)
    if z is not None:
        out["z"] = (g["z"], np.abs(dyn) * (errh * np.abs(slope) + 64 * HALF32 * magh * (np.abs(slope) + np.abs(value) + 1)))
    if h0 is not None:
        out["h0"] = (first, errfirst + C * HALF32 * magfirst)
    return out


def _close(name, got, want, bound, dtype=torch.float32):
    got = _np(got).reshape(want.shape)
    tol = bound + (np.abs(want) + bound) * _half(dtype) + (2.0 ** -25 if dtype == torch.float16 else 1e-37)
    worst = np.max((np.abs(got - want) - tol), initial=-np.inf)
    assert np.isfinite(got).all() and worst <= 0, (name, worst, np.max(np.abs(got - want) / np.maximum(tol, 1e-300), initial=0))


def _cuda(t, grad=False):
    """To the GPU; slices of one tensor stay slices of one tensor."""
    if t is None:
        return None
    if t._base is not None:
        wide = t._base.cuda()
        t = wide.as_strided(t.shape, t.stride(), t.storage_offset()).detach()
    else:
        t = t.cuda()
    return t.requires_grad_(True) if grad else t


def _gpu(t, grad=False):
    return {k: _cuda(v, grad) for k, v in t.items()}


def _call(t, act, normalize, cu=None, want=True):
    return gated_recurrence(t["x"], t["r"], t["A"], input_gate=t["i"], gate=t["z"], gate_activation=act, normalize=normalize,
                            initial_state=t["h0"], output_final_state=want, cu_seqlens=cu)


def _bounds(lens):
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int64)


CASES = [
    # n or lens, T, D, dtype, input gate, gate, activation, normalize, state, sliced
    (2, 77, 97, torch.float32, True, True, "silu", True, True, False),
    (1, 1, 8, torch.bfloat16, True, True, "silu", True, False, False),
    (3, 64, 128, torch.bfloat16, True, True, "sigmoid", True, True, True),
    (1, 65, 130, torch.float16, False, True, None, True, True, False),
    (1, 2500, 128, torch.float32, True, True, "silu", True, True, False),      # more than one group of tiles
    (1, 4300, 256, torch.bfloat16, True, True, "silu", True, False, True),     # more than two, two blocks of channels
    (1, 8500, 24, torch.float32, True, False, None, True, True, False),        # tiles of 256 tokens
    (2, 300, 40, torch.float16, True, True, "silu", False, False, False),      # tiles of 128
    ([0, 1, 63, 64, 65, 0, 127, 2200, 1, 0], None, 128, torch.float32, True, True, "silu", True, True, False),
    ([5, 700, 0, 256, 1, 255, 257], None, 96, torch.bfloat16, True, True, "sigmoid", True, True, True),
    ([30, 40], None, 33, torch.float16, False, False, None, True, False, False),
    ([1] * 40, None, 64, torch.float32, True, True, None, False, True, False),
    ([0, 0, 0], None, 16, torch.float32, True, True, "silu", True, True, False),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_forward_and_gradients(case):
    n, T, D, dtype, i, z, act, normalize, state, sliced = case
    lens = n if isinstance(n, list) else [T] * n
    shape = (1, sum(lens)) if isinstance(n, list) else (n, T)
    t = _inputs(shape, D, dtype, 3, len(lens), i, z, state, sliced)
    cu = _bounds(lens).cuda() if isinstance(n, list) else None
    g = torch.Generator().manual_seed(4)
    dy = torch.randn(*shape, D, generator=g).to(dtype)
    dht = torch.randn(len(lens), D, generator=g)
    want = _expected(t, lens, act, normalize, dy, dht)
    y, last = _call(_gpu(t), act, normalize, cu)
    _close("y", y, *want["y"], dtype)
    _close("last", last, *want["last"])
    assert _call(_gpu(t), act, normalize, cu, want=False)[1] is None
    leaves = _gpu(t, grad=True)
    y2, last2 = _call(leaves, act, normalize, cu)
    assert torch.equal(y2, y) and torch.equal(last2, last)
    names = [k for k in ("x", "r", "A", "i", "z", "h0") if t[k] is not None]
    grads = torch.autograd.grad([y2, last2], [leaves[k] for k in names], [dy.cuda(), dht.cuda()])
    for k, v in zip(names, grads):
        assert v.dtype == t[k].dtype and v.shape == t[k].shape
        _close(k, v, *want[k], dtype if k in "xriz" else torch.float32)
    y3, last3 = _call(leaves, act, normalize, cu)
    again = torch.autograd.grad([y3, last3], [leaves[k] for k in names], [dy.cuda(), dht.cuda()])
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


def test_gradients_of_either_output_alone():
    t = _inputs((1, 200), 64, torch.float32, 5, 1)
    dy, dht = torch.randn(1, 200, 64), torch.randn(1, 64)
    for use_y, use_last in ((True, False), (False, True)):
        leaves = _gpu(t, grad=True)
        y, last = _call(leaves, "silu", True)
        want = _expected(t, [200], "silu", True, dy if use_y else dy * 0, dht if use_last else dht * 0)
        names = ["x", "r", "A", "i", "h0"] + (["z"] if use_y else [])
        out, d = (y, dy) if use_y else (last, dht)
        for k, v in zip(names, torch.autograd.grad(out, [leaves[k] for k in names], d.cuda(), retain_graph=True)):
            _close(k, v, *want[k])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_out_of_line(dtype):
    """Tensors one element off their alignment, tokens far apart, a transposed batch: the same bits as contiguous ones."""
    t = _gpu(_inputs((2, 150), 64, dtype, 6, 2))
    want = _call(t, "silu", True)
    moved = dict(t)
    for k in ("x", "r", "i", "z"):
        buf = torch.zeros(2 * 150 * 67 + 1, dtype=dtype, device="cuda")
        moved[k] = buf[1:].view(2, 150, 67)[..., :64]
        moved[k].copy_(t[k])
    got = _call(moved, "silu", True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    turned = dict(t, x=t["x"].transpose(0, 1).contiguous().transpose(0, 1), z=t["z"].flip(-1).flip(-1))
    got = _call(turned, "silu", True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    leaf = [moved[k].detach().requires_grad_(True) for k in ("x", "r", "i", "z")]
    flat = [t[k].detach().requires_grad_(True) for k in ("x", "r", "i", "z")]
    d = torch.randn(2, 64, 150, device="cuda").to(dtype).transpose(1, 2)
    for a, b in zip(torch.autograd.grad(_call(dict(moved, **dict(zip("xriz", leaf))), "silu", True)[0], leaf, d),
                    torch.autograd.grad(_call(dict(t, **dict(zip("xriz", flat))), "silu", True)[0], flat, d)):
        assert torch.equal(a, b)


def test_boundaries_on_the_device_are_held_inside():
    """Rows behind the last boundary come back as zero and enter nothing, whatever they hold; boundaries that decrease or lie outside
    are moved, and the call ends."""
    T, D, lens = 700, 64, [100, 0, 333]
    t = _inputs((1, T), D, torch.float32, 7, 3)
    for k in ("x", "r", "i", "z"):
        t[k][:, 433:] = float("nan")
    dy = torch.randn(1, T, D)
    dy[:, 433:] = float("nan")
    leaves = _gpu(t, grad=True)
    y, last = _call(leaves, "silu", True, _bounds(lens).cuda())
    names = ["x", "r", "A", "i", "z", "h0"]
    grads = dict(zip(names, torch.autograd.grad(y, [leaves[k] for k in names], dy.cuda())))
    cut = {k: v[:, :433] if k in "xriz" else v for k, v in t.items()}
    want = _expected(cut, lens, "silu", True, dy[:, :433], torch.zeros(3, D))
    assert not y[:, 433:].any()
    _close("y", y[:, :433], *want["y"])
    _close("last", last, *want["last"])
    for k in names:
        got = grads[k]
        if k in "xriz":
            assert not got[:, 433:].any()
            got = got[:, :433]
        _close(k, got, *want[k])
    whole = _gpu(_inputs((1, T), D, torch.float32, 8, 4, state=False))
    for given, taken in (([0, 300, 200, 900, 700], [0, 300, 300, 700, 700]), ([5, -7, 400, 10**12, 650], [0, 0, 400, 700, 700])):
        got = _call(whole, "silu", True, torch.tensor(given).cuda())
        ref = _call(whole, "silu", True, torch.tensor(taken))
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


def test_values_that_are_not_finite_stay_in_their_channel():
    T, D = 400, 40
    t = _inputs((1, T), D, torch.float32, 9, 1)
    clean = _call(_gpu(t), "silu", True)[0]
    for bad in (float("nan"), float("inf")):
        for k in ("x", "r", "i", "z"):
            hurt = {**t, k: t[k].clone()}
            hurt[k][0, 200, 7] = bad
            y = _call(_gpu(hurt), "silu", True)[0]
            other = [c for c in range(D) if c != 7]
            assert torch.equal(y[:, :200], clean[:, :200]) and torch.equal(y[..., other], clean[..., other])
            if k in "xr" and bad != bad:
                assert y[0, 200:, 7].isnan().all()


def test_extreme_gates():
    """Gates at both ends of the type: the state kept or replaced whole, no slope through m where nothing is let in."""
    D = 8
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.ones(1, 70, D, dtype=dtype)
        r = torch.zeros(1, 70, D, dtype=dtype)
        r[:, :35], r[:, 35:] = -1e4, 1e4
        t = {"x": x, "r": r, "i": torch.full_like(x, 1e4), "z": None, "A": torch.full((D,), -200.0), "h0": torch.full((1, D), 3.0)}
        leaves = _gpu(t, grad=True)
        y, last = _call(leaves, None, True)
        assert torch.equal(y[:, :35].float().cpu(), torch.full((1, 35, D), 3.0))  # nothing decays, nothing comes in
        assert torch.equal(y[:, 35:].float().cpu(), torch.ones(1, 35, D))         # nothing is kept, all comes in
        grads = torch.autograd.grad(y, [leaves[k] for k in ("x", "r", "A", "i", "h0")], torch.ones_like(y))
        assert all(g.isfinite().all() for g in grads)
        assert not grads[1].any() and torch.equal(grads[4].cpu(), torch.full((1, D), 35.0))


@pytest.mark.parametrize("D", [33, 512])
def test_steps_follow_the_scan(D):
    n, T = 3, 9
    t = _inputs((n, T), D, torch.bfloat16, 10, n, sliced=True)
    g = _gpu(t)
    state = g["h0"].clone()
    want = _expected(t, [T] * n, "silu", True)
    for k in range(T):
        at = {m: g[m][:, k] for m in ("x", "r", "i", "z")}
        new = torch.empty_like(state)
        y0 = gated_recurrence_step(at["x"], at["r"], g["A"], state, input_gate=at["i"], gate=at["z"], gate_activation="silu",
                                   new_state=new)
        version = state._version
        y = gated_recurrence_step(at["x"], at["r"], g["A"], state, input_gate=at["i"], gate=at["z"], gate_activation="silu")
        assert state._version > version and torch.equal(new, state) and torch.equal(y, y0)
        _close("y", y, want["y"][0].reshape(n, T, D)[:, k], want["y"][1].reshape(n, T, D)[:, k], torch.bfloat16)
    _close("last", state, *want["last"])
    empty = gated_recurrence_step(at["x"][:0], at["r"][:0], g["A"], state[:0])
    assert empty.shape == (0, D)


def test_a_final_state_that_was_moved_on_is_noticed():
    leaves = _gpu(_inputs((2, 20), 32, torch.float32, 11, 2), grad=True)
    y, last = _call(leaves, "silu", True)
    row = [leaves[k][:, -1].detach() for k in ("x", "r")]
    gated_recurrence_step(row[0], row[1], leaves["A"].detach(), last.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    step = gated_recurrence_step(leaves["x"][:, 0], leaves["r"][:, 0], leaves["A"], torch.zeros(2, 32, device="cuda"))
    with pytest.raises(NotImplementedError):
        step.sum().backward()


def test_captured_and_replayed():
    """Forward and token step in one graph, gradients in another, replayed with other inputs and boundaries."""
    T, D = 3000, 64
    lens = [[1000, 0, 2000], [1, 2900, 0]]
    sets = [_gpu(_inputs((1, T), D, torch.bfloat16, 20 + k, 3)) for k in range(2)]
    static = {k: v.clone() for k, v in sets[0].items()}
    cu = _bounds(lens[0]).cuda()
    dy = torch.randn(1, T, D, device="cuda").bfloat16()
    leaves = {k: static[k].detach().requires_grad_(True) for k in ("x", "r", "i", "z", "A")}

    def forward():
        y, last = _call(static, "silu", True, cu)
        new = torch.empty_like(last)
        return y, last, gated_recurrence_step(y[0, :3], y[0, :3], static["A"], last, new_state=new), new

    def train():
        y, _ = _call({**leaves, "h0": static["h0"]}, "silu", True, cu)
        return torch.autograd.grad(y, list(leaves.values()), dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        forward()
        train()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for fn in (forward, train):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(fn())
        graphs.append(graph)
    for rep in range(4):
        for k, v in sets[rep % 2].items():
            static[k].copy_(v)
        cu.copy_(_bounds(lens[rep % 2]))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for out in outs for o in out]
        for a, b in zip(got, [*forward(), *train()]):
            assert torch.equal(a, b)


def test_streams_side_by_side():
    """Calls under way at once on two streams, each with words of its own, give what they give alone."""
    sets = [_gpu(_inputs((1, 6000), 128, torch.float32, 30 + k, 1)) for k in range(2)]
    want = [_call(t, "silu", True) for t in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for rep in range(3):
        for t, s in zip(sets, streams):
            with torch.cuda.stream(s):
                got.append(_call(t, "silu", True))
    torch.cuda.synchronize()
    for k, (y, last) in enumerate(got):
        assert torch.equal(y, want[k % 2][0]) and torch.equal(last, want[k % 2][1])


def test_refusals():
    t = _gpu(_inputs((2, 10), 16, torch.float32, 12, 2))
    x, r, A, h0 = t["x"], t["r"], t["A"], t["h0"]
    bad = [
        (ValueError, dict(decay_gate=r[:, :9])), (TypeError, dict(decay_gate=r.half())), (ValueError, dict(A=A[:8])),
        (TypeError, dict(A=A.long())), (ValueError, dict(input_gate=r[..., :8])), (TypeError, dict(gate=r.half())),
        (ValueError, dict(gate_activation="relu", gate=r)), (ValueError, dict(gate_activation="silu")),
        (ValueError, dict(initial_state=h0[:1])), (TypeError, dict(initial_state=h0.long())),
        (ValueError, dict(cu_seqlens=torch.tensor([0, 10]))), (ValueError, dict(x=x[0], decay_gate=r[0])),
        (TypeError, dict(x=x.double(), decay_gate=r.double())), (ValueError, dict(x=x[:0], decay_gate=r[:0])),
        (_capi.LampaError, dict(A=A.cpu())),
    ]
    for error, change in bad:
        with pytest.raises(error):
            gated_recurrence(**{"x": x, "decay_gate": r, "A": A, **change})
    for bounds in ([0, 5], [1, 10], [0, 7, 5, 10], [0.0, 10.0]):
        with pytest.raises(ValueError):
            gated_recurrence(x[:1], r[:1], A, cu_seqlens=torch.tensor(bounds))
    step = dict(x=x[:, 0], decay_gate=r[:, 0], A=A, state=h0)
    for change in (dict(state=h0[:1]), dict(state=h0.half()), dict(state=h0.t().contiguous().t()),
                   dict(state=torch.zeros(3, 16, device="cuda")[:2], new_state=None, A=A[:3]), dict(new_state=h0.half())):
        with pytest.raises(ValueError):
            gated_recurrence_step(**{**step, **change})
    buf = torch.zeros(3, 16, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        gated_recurrence_step(**{**step, "state": buf[:2], "new_state": buf[1:]})
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(Exception):
            torch.autograd.forward_ad.unpack_dual(gated_recurrence(dual, r, A)[0])
