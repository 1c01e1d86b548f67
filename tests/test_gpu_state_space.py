"""GPU parity of the state-space operators, forward and gradients, against the float64 token loop.

Tolerances are worst-case bounds from the rounding of each step, against the same computation on absolute values (`mag`, which
bounds the sum of the magnitudes of everything that was added up):

* fp32: a token's state takes a product, a sum, and a decay whose exponential is off by a few half-steps (and by the
  exponent's own rounding, |g| half-steps of a factor e^-|g|): at most 8 half-steps a token, and N or P more for a read-out;
* 16-bit types: additionally the output's own rounding, half a step of its value, and for the pairs of tokens within a chunk
  one rounding of their weight to the input type, half a step of `mag`. States enter their products as two parts of 8 (bf16)
  bits or more, which leaves 2^-16 of `mag`."""
import numpy as np
import pytest
import torch

from lampa_amd import _capi
from lampa_amd import state_space as ss
from oracle import state_space as os_

pytestmark = pytest.mark.gpu

HALF32 = 2.0 ** -24


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _inputs(shape, H, P, G, N, dtype, seed, n_seq, state=True, sliced=False, rate=16.0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    if sliced:  # columns of one wider tensor
        wide = r(*shape, H * P + 2 * G * N + 8).to(dtype)
        x, B, C, _ = wide.split([H * P, G * N, G * N, 8], dim=-1)
        x, B, C = x.unflatten(-1, (H, P)), B.unflatten(-1, (G, N)), C.unflatten(-1, (G, N))
    else:
        x, B, C = r(*shape, H, P).to(dtype), r(*shape, G, N).to(dtype), r(*shape, G, N).to(dtype)
    step = torch.exp(torch.rand(H, generator=gen) * 4.6 - 6.9)
    return dict(x=x, dt=r(*shape, H).to(dtype), A=-(0.5 + rate * torch.rand(H, generator=gen)), B=B, C=C, D=r(H),
                dt_bias=step + torch.log(-torch.expm1(-step)), h0=r(n_seq, H, N, P) * 0.5 if state else None)


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _flat(t):
    a = _np(t)
    return a.reshape(-1, *a.shape[2:])


def _oracle(i, lens, softplus=True, dy=None, dht=None):
    """(values, magnitudes), each (y, last, grads or None)."""
    raw = _flat(i["dt"]) + (0 if i["dt_bias"] is None else _np(i["dt_bias"]))
    delta = os_.softplus(raw) if softplus else raw
    args = [_flat(i["x"]), delta, _np(i["A"]), _flat(i["B"]), _flat(i["C"]), _np(i["D"]), _np(i["h0"])]
    mags = [np.abs(args[0]), np.abs(delta), args[2]] + [None if a is None else np.abs(a) for a in args[3:]]
    out = []
    for a, up in ((args, lambda t: t), (mags, np.abs)):
        y, last = os_.scan(*a[:6], a[6], lens)
        g = None
        if dy is not None:
            g = os_.scan_grads(*a[:6], a[6], lens, up(_flat(dy)), None if dht is None else up(_np(dht)))
            s = os_.sigmoid(raw) if softplus else np.ones_like(raw)
            if up is np.abs:
                # what dg is summed up from: every later token's |read| and |written| of its sequence, and |<R, S>| at its end
                Bw, Cw = (np.repeat(t, a[0].shape[1] // t.shape[1], axis=1) for t in (a[3], a[4]))
                read = np.einsum("thp,thp->th", y - a[5][:, None] * a[0] if a[5] is not None else y, up(_flat(dy)))
                dxs = g["x"] - (0 if a[5] is None else a[5][:, None] * up(_flat(dy)))
                # written = delta x . (R^T B); written / delta is wanted where delta is tiny: bounded through its own sum
                written = np.einsum("thp,thp->th", dxs, a[0])
                reach = written / np.maximum(a[1], 1e-30)
                total, t0 = np.zeros_like(read), 0
                for k, n in enumerate(lens):
                    tail = 0.0 if dht is None else (up(_np(dht))[k] * last[k]).sum((-1, -2))
                    total[t0:t0 + n] = np.cumsum((read + written)[t0:t0 + n][::-1], 0)[::-1] + tail
                    t0 += n
                # segments start anew from <R, S>, which the same sums bound
                g["delta"] = np.abs(a[2]) * 2 * total + reach
                g["A"] = (a[1] * 2 * total).sum(0)
            g["dt"] = g.pop("delta") * s
            g["dt_bias"] = g["dt"].sum(0)
        out.append((y, last, g))
    return out


def _bound(dtype, T, value, mag, wide, pairs=True):
    """`wide`: read-out length; `pairs`: the pair weights' rounding enters."""
    b = (8 * T + wide + 32) * HALF32 * mag + 1e-30
    if dtype != torch.float32:
        b = b + 2.0 ** -16 * mag + (_half(dtype) * mag if pairs else 0.0)
    return b


def _check(name, got, want, bound, out_dtype=torch.float32):
    got = got.detach().double().cpu().numpy().reshape(want.shape)
    if out_dtype != torch.float32:
        tiny = torch.finfo(out_dtype).smallest_normal * torch.finfo(out_dtype).eps
        bound = (bound + _half(out_dtype) * np.abs(want)) * (1 + _half(out_dtype)) + tiny
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (name, int(bad.sum()), float(np.abs(got - want).max()), float((np.abs(got - want) / bound).max()))


def _to(i, device, grad=False):
    out = {}
    for k, t in i.items():
        if t is not None:
            t = t.to(device)
            t = t.detach().requires_grad_(True) if grad else t
        out[k] = t
    return out


def _call(d, softplus=True, final=True, cu=None):
    return ss.state_space_scan(d["x"], d["dt"], d["A"], d["B"], d["C"], D=d["D"], dt_bias=d["dt_bias"], dt_softplus=softplus,
                               initial_state=d["h0"], output_final_state=final, cu_seqlens=cu)


DTYPES = [torch.float32, torch.bfloat16, torch.float16]
SHAPES = [
    # lens (None: dense [B, T]), B, T, H, P, G, N
    (None, 1, 1, 2, 8, 1, 8),
    (None, 2, 63, 4, 20, 2, 24),
    (None, 1, 65, 3, 64, 3, 64),
    (None, 3, 130, 2, 33, 1, 17),
    (None, 1, 700, 2, 128, 1, 128),
    (None, 1, 300, 6, 16, 2, 100),
    ([64, 0, 1, 128, 200, 0, 7, 65], 1, 465, 4, 64, 1, 32),
    ([1], 1, 1, 1, 1, 1, 1),
    ([0, 0, 333], 1, 333, 2, 72, 2, 48),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,B,T,H,P,G,N", SHAPES)
def test_scan_and_gradients(device, dtype, lens, B, T, H, P, G, N, monkeypatch):
    n_seq = B if lens is None else len(lens)
    i = _inputs((B, T), H, P, G, N, dtype, T + H, n_seq, sliced=P % 8 == 0)
    gen = torch.Generator().manual_seed(T)
    dy, dht = torch.randn(B, T, H, P, generator=gen).to(dtype), torch.randn(n_seq, H, N, P, generator=gen) * 0.5
    cu = None if lens is None else torch.tensor(np.cumsum([0] + lens), device=device)
    (y, last, g), (ym, lastm, gm) = _oracle(i, [T] * B if lens is None else lens, dy=dy, dht=dht)
    n = max([T] if lens is None else lens)
    for seg in (None, 64):  # the rule's segments, and the shortest ones
        if seg:
            monkeypatch.setattr(ss, "_segment_tokens", lambda *a: seg)
        plain = _to(i, device)
        got, ht = _call(plain, cu=cu)
        assert got.dtype == dtype and ht.dtype == torch.float32
        _check("y", got, y, _bound(dtype, n, y, ym, N), dtype)
        _check("last", ht, last, _bound(dtype, n, last, lastm, 0, False))
        d = _to(i, device, grad=True)
        got2, ht2 = _call(d, cu=cu)
        assert torch.equal(got, got2) and torch.equal(ht, ht2)
        names = ["x", "dt", "A", "B", "C", "D", "dt_bias", "h0"]
        grads = torch.autograd.grad([got2, ht2], [d[k] for k in names], [dy.to(device), dht.to(device)], retain_graph=True)
        again = torch.autograd.grad([got2, ht2], [d[k] for k in names], [dy.to(device), dht.to(device)])
        for k, a, b in zip(names, grads, again):
            assert torch.equal(a, b), k  # the same bits every time
            assert a.shape == d[k].shape and a.dtype == d[k].dtype
            # B and C sum over columns (and heads), x over states, the scalars over both
            wide = {"x": N, "B": P * H // G, "C": P * H // G, "h0": 0, "D": T * P}.get(k, N * P + T)
            _check(k, a, g[k], _bound(dtype, n, g[k], gm[k], wide, k in ("x", "B", "C")), d[k].dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,bias,softplus,state", [(False, False, False, False), (True, False, True, False), (False, True, True, True)])
def test_optional_operands(device, dtype, D, bias, softplus, state):
    i = _inputs((2, 200), 2, 32, 1, 40, dtype, 5, 2, state=state)
    if not D:
        i["D"] = None
    if not bias:
        i["dt_bias"] = None
    if not softplus:
        i["dt"] = i["dt"].abs() * 0.1
    dy = torch.randn(2, 200, 2, 32, generator=torch.Generator().manual_seed(6)).to(dtype)
    (y, last, g), (ym, lastm, gm) = _oracle(i, [200, 200], softplus, dy=dy)
    d = _to(i, device, grad=True)
    got, none = _call(d, softplus, final=False)
    assert none is None
    names = [k for k in ("x", "dt", "A", "B", "C", "D", "dt_bias", "h0") if d[k] is not None]
    grads = torch.autograd.grad(got, [d[k] for k in names], dy.to(device))
    _check("y", got, y, _bound(dtype, 200, y, ym, 40), dtype)
    for k, a in zip(names, grads):
        wide = {"x": 40, "B": 64, "C": 64, "h0": 0, "D": 200 * 32 * 2}.get(k, 40 * 32 + 400)
        _check(k, a, g[k], _bound(dtype, 200, g[k], gm[k], wide, k in ("x", "B", "C")), d[k].dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_dt_in_fp32_beside_16_bit_tensors(device, dtype):
    i = _inputs((1, 150), 2, 64, 1, 64, dtype, 7, 1)
    i["dt"] = torch.randn(1, 150, 2, generator=torch.Generator().manual_seed(8))
    dy = torch.randn(1, 150, 2, 64, generator=torch.Generator().manual_seed(9)).to(dtype)
    (y, last, g), (ym, lastm, gm) = _oracle(i, [150], dy=dy)
    d = _to(i, device, grad=True)
    got, ht = _call(d)
    _check("y", got, y, _bound(dtype, 150, y, ym, 64), dtype)
    ddt, = torch.autograd.grad(got, [d["dt"]], dy.to(device))
    assert ddt.dtype == torch.float32
    _check("dt", ddt, g["dt"], _bound(dtype, 150, g["dt"], gm["dt"], 64 * 64 + 150, False))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strong_decays_cut_the_past_off(device, dtype):
    """Tokens whose step wipes the state, and steps of zero, beside ordinary ones."""
    i = _inputs((1, 260), 2, 32, 1, 32, dtype, 10, 1, rate=1.0)
    dt = torch.full((1, 260, 2), 0.05)
    dt[:, ::37] = 2000.0
    dt[:, 5::41] = 0.0
    i["dt"], i["dt_bias"] = dt.to(dtype), None
    i["x"][:, ::37] = 0  # their own write is not what is looked at
    (y, last, _), (ym, lastm, _) = _oracle(i, [260], softplus=False)
    got, ht = _call(_to(i, device), softplus=False)
    # exponents are clamped at -104: sums of them over a chunk, whose differences are taken, are off by 64 * 104 half-steps
    loose = 64 * 104 * HALF32 * 8
    _check("y", got, y, _bound(dtype, 260, y, ym, 32) + loose * ym, dtype)
    _check("last", ht, last, _bound(dtype, 260, last, lastm, 0, False) + loose * lastm)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_values_that_are_not_finite_reach_no_earlier_token(device, dtype, bad):
    i = _inputs((1, 200), 2, 64, 1, 32, dtype, 11, 1, sliced=False)
    clean, _ = _call(_to(i, device))
    for name, where in (("x", (0, 100, 1, 3)), ("B", (0, 70, 0, 5)), ("C", (0, 130, 0, 2)), ("dt", (0, 90, 1))):
        j = dict(i)
        j[name] = i[name].clone()
        j[name][where] = bad
        got, _ = _call(_to(j, device))
        t = where[1]
        assert torch.equal(got[:, :t], clean[:, :t]), name
        assert not torch.isfinite(got[:, t]).all()
        if name == "x":  # nor another column or head
            assert torch.isfinite(got[:, :, 0]).all() and torch.isfinite(got[:, :, 1, :3]).all()
            assert not torch.isfinite(got[:, t:, 1, 3]).any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_padding_behind_the_tokens_changes_no_gradient(device, dtype):
    """A padded batch: rubbish behind the real tokens, no gradient asked of it."""
    i = _inputs((1, 200), 2, 64, 1, 32, dtype, 12, 1)
    dy = torch.randn(1, 200, 2, 64, generator=torch.Generator().manual_seed(13)).to(dtype)
    dy[:, 150:] = 0
    j = dict(i)
    j["x"] = i["x"].clone()
    j["x"][:, 150:] = float("nan")
    out = []
    for k in (i, j):
        d = _to(k, device, grad=True)
        out.append(torch.autograd.grad(_call(d)[0], [d["x"], d["B"], d["C"]], dy.to(device)))
    for a, b in zip(*out):
        assert torch.equal(a[:, :150], b[:, :150])


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_outside_the_boundaries(device, dtype, monkeypatch):
    """Boundaries on the GPU are not read by the host: what lies behind the last one comes back as zero, and boundaries beyond
    the tokens are held inside. (Segments of one length in both calls: other segments round differently.)"""
    monkeypatch.setattr(ss, "_segment_tokens", lambda *a: 64)
    i = _inputs((1, 300), 2, 32, 1, 32, dtype, 14, 2)
    d = _to(i, device, grad=True)
    dy = torch.randn(1, 300, 2, 32, generator=torch.Generator().manual_seed(15)).to(dtype).to(device)
    y, ht = _call(d, cu=torch.tensor([0, 100, 170], device=device))
    grads = torch.autograd.grad(y, [d[k] for k in ("x", "dt", "B", "C", "A")], dy)
    assert not y[:, 170:].any() and all(not g[:, 170:].any() for g in grads[:4])
    cut = {k: t[:, :170] if k in ("x", "dt", "B", "C") else t for k, t in i.items()}
    e = _to(cut, device, grad=True)
    y2, ht2 = _call(e, cu=torch.tensor([0, 100, 170]))
    want = torch.autograd.grad(y2, [e[k] for k in ("x", "dt", "B", "C", "A")], dy[:, :170])
    assert torch.equal(y[:, :170], y2) and torch.equal(ht, ht2)
    for a, b in zip(grads, want):
        assert torch.equal(a[:, :170] if a.dim() > 1 else a, b)
    beyond, _ = _call(d, cu=torch.tensor([0, 100, 10 ** 9], device=device))
    inside, _ = _call(d, cu=torch.tensor([0, 100, 300], device=device))
    assert torch.equal(beyond, inside)


@pytest.mark.parametrize("dtype", DTYPES)
def test_where_the_operands_lie(device, dtype):
    """Slices off every alignment, tokens and batches out of order, broadcast tensors, gradients that are no tensors of their own:
    the bits of contiguous copies."""
    gen = torch.Generator().manual_seed(50)
    r = lambda *s: torch.randn(*s, generator=gen).to(dtype).to(device)  # noqa: E731
    i = _to(_inputs((3, 90), 2, 16, 1, 24, dtype, 51, 3), device)
    wide = r(3, 90, 100)
    forms = [
        {"x": wide[..., 3:35].unflatten(-1, (2, 16)), "B": wide[..., 37:61].unsqueeze(2), "C": wide[..., 75:99].unsqueeze(2), "dt": wide[..., 35:37]},
        {"x": r(90, 3, 2, 16).transpose(0, 1), "B": r(3, 1, 90, 24).transpose(1, 2), "C": r(90, 3, 1, 24).transpose(0, 1), "dt": r(90, 2, 3).permute(2, 0, 1)},
        {"x": r(3, 90, 16, 2).transpose(2, 3), "B": r(1, 1, 1, 24).expand(3, 90, 1, 24), "C": r(3, 1, 1, 24).expand(3, 90, 1, 24), "dt": r(3, 1, 2).expand(3, 90, 2)},
    ]
    dy = r(3, 2, 90, 16).transpose(1, 2)
    for form in forms:
        out = []
        for copy in (False, True):
            d = {**i, **form}
            d = {k: (t.contiguous().clone() if copy else t).detach().requires_grad_(True) for k, t in d.items()}
            y, ht = _call(d)
            out.append([y, ht, *torch.autograd.grad(y, [d[k] for k in ("x", "dt", "A", "B", "C", "D", "dt_bias", "h0")],
                                                    dy.contiguous() if copy else dy)])
        for a, b in zip(*out):
            assert torch.equal(a, b)
    y, _ = _call({**i, "x": i["x"].requires_grad_(True)})
    assert torch.equal(torch.autograd.grad(y.sum(), i["x"], retain_graph=True)[0], torch.autograd.grad(y, i["x"], torch.ones_like(y))[0])


def test_no_tokens(device):
    i = _to(_inputs((2, 0), 2, 16, 1, 8, torch.bfloat16, 16, 2), device, grad=True)
    y, ht = _call(i)
    assert y.shape == (2, 0, 2, 16) and torch.equal(ht, i["h0"])
    grads = torch.autograd.grad(ht, [i["h0"], i["A"], i["x"]], torch.ones_like(ht))
    assert torch.equal(grads[0], torch.ones_like(ht)) and not grads[1].any() and grads[2].shape == (2, 0, 2, 16)


@pytest.mark.parametrize("dtype", DTYPES)
def test_another_stream_and_a_captured_graph(device, dtype):
    """A forward with its gradients captured once and replayed on other inputs, eager work in between: the eager bits."""
    make = lambda seed: _to(_inputs((1, 1500), 2, 64, 1, 64, dtype, seed, 2), device, grad=True)  # noqa: E731
    d = make(20)
    cu = torch.tensor([0, 700, 1500], device=device)
    names = ["x", "dt", "A", "B", "C", "D", "dt_bias", "h0"]
    dy = torch.randn(1, 1500, 2, 64, device=device).to(dtype)

    def step(d):
        y, ht = _call(d, cu=cu)
        return [y, ht, *torch.autograd.grad([y, ht], [d[k] for k in names], [dy, ht.detach()])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step(d)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(on_side, step(d)):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(d)
    for seed, bounds in ((21, [0, 700, 1500]), (22, [0, 1, 1500]), (23, [0, 1499, 1500])):
        new = make(seed)
        for k in names:
            d[k].data.copy_(new[k])
        cu.copy_(torch.tensor(bounds))
        graph.replay()
        want = step(new)
        for k, a, b in zip(["y", "ht"] + names, out, want):
            assert torch.equal(a, b), (seed, k)
        torch.cuda.synchronize()


# ---------------------------------------------------------------------------------------------------------- one token
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,H,P,G,N", [(1, 8, 64, 1, 64), (3, 4, 20, 2, 24), (70, 4, 64, 1, 128), (2, 2, 33, 1, 17), (5, 1, 1, 1, 1),
                                       (2, 3, 130, 3, 300)])
def test_step(device, dtype, n, H, P, G, N):
    i = _inputs((n,), H, P, G, N, dtype, n + P, n)
    want = [os_.scan(_np(i["x"])[b:b + 1], os_.softplus(_np(i["dt"]) + _np(i["dt_bias"]))[b:b + 1], _np(i["A"]), _np(i["B"])[b:b + 1],
                     _np(i["C"])[b:b + 1], _np(i["D"]), _np(i["h0"])[b:b + 1]) for b in range(n)]
    mags = [os_.scan(abs(_np(i["x"]))[b:b + 1], os_.softplus(_np(i["dt"]) + _np(i["dt_bias"]))[b:b + 1], _np(i["A"]),
                     abs(_np(i["B"]))[b:b + 1], abs(_np(i["C"]))[b:b + 1], abs(_np(i["D"])), abs(_np(i["h0"]))[b:b + 1])
            for b in range(n)]
    d = _to(i, device)
    args = (d["x"], d["dt"], d["A"], d["B"], d["C"])
    kw = dict(D=d["D"], dt_bias=d["dt_bias"], dt_softplus=True)
    new = torch.empty_like(d["h0"])
    before = d["h0"].clone()
    y = ss.state_space_step(*args, d["h0"], new_state=new, **kw)
    assert torch.equal(d["h0"], before)
    in_place = ss.state_space_step(*args, d["h0"], **kw)
    assert torch.equal(y, in_place) and torch.equal(d["h0"], new)
    ym = np.concatenate([m[0] for m in mags])
    _check("y", y, np.concatenate([w[0] for w in want]), (8 + N + 32) * HALF32 * ym, dtype)
    _check("state", new, np.concatenate([w[1] for w in want]), 40 * HALF32 * np.concatenate([m[1] for m in mags]))


def test_step_without_options_and_strided(device):
    gen = torch.Generator().manual_seed(30)
    wide = torch.randn(4, 2 * 16 + 2 * 8 + 2, generator=gen).to(device)
    x, B, C, dt = wide.split([32, 8, 8, 2], dim=-1)
    x, B, C, dt = x.unflatten(-1, (2, 16)), B.unflatten(-1, (1, 8)), C.unflatten(-1, (1, 8)), dt.abs()
    state = torch.randn(4, 2, 8, 16, generator=gen).to(device)
    A = -torch.rand(2, generator=gen).to(device)
    copy = state.clone()
    y = ss.state_space_step(x, dt, A, B, C, state)
    y2 = ss.state_space_step(x.contiguous(), dt.contiguous(), A, B.contiguous(), C.contiguous(), copy)
    assert torch.equal(y, y2) and torch.equal(state, copy)
    scan, last = ss.state_space_scan(x[:, None], dt[:, None], A, B[:, None], C[:, None], output_final_state=True,
                                     initial_state=torch.zeros_like(state))
    assert scan.shape == (4, 1, 2, 16)


@pytest.mark.parametrize("dtype", DTYPES)
def test_steps_continue_a_scan(device, dtype):
    """A prompt by the scan, then tokens one at a time: the outputs of the whole sequence by the scan."""
    i = _inputs((2, 140), 4, 32, 2, 16, dtype, 31, 2, state=False)
    (y, last, _), (ym, lastm, _) = _oracle(i, [140, 140])
    d = _to(i, device)
    head = {k: t[:, :130] if k in ("x", "dt", "B", "C") else t for k, t in d.items()}
    _, state = _call(head)
    for t in range(130, 140):
        out = ss.state_space_step(d["x"][:, t], d["dt"][:, t], d["A"], d["B"][:, t], d["C"][:, t], state, D=d["D"],
                                  dt_bias=d["dt_bias"], dt_softplus=True)
        want = y.reshape(2, 140, 4, 32)[:, t]
        _check("y", out, want, _bound(dtype, 140, want, ym.reshape(2, 140, 4, 32)[:, t], 16), dtype)
    _check("state", state, last, _bound(dtype, 140, last, lastm, 0, False))


# ----------------------------------------------------------------------------------------------------------- refusals
def test_refusals(device):
    i = _to(_inputs((1, 10), 4, 16, 2, 8, torch.bfloat16, 40, 1), device)
    call = lambda **c: _call({**i, **c})  # noqa: E731
    with pytest.raises(ValueError, match="dt"):
        call(dt=i["dt"][:, :9])
    with pytest.raises(ValueError, match="G"):
        call(B=i["B"][:, :, :1], C=i["C"])
    with pytest.raises(ValueError, match="divisor"):
        call(B=torch.zeros(1, 10, 3, 8, device=device, dtype=torch.bfloat16), C=torch.zeros(1, 10, 3, 8, device=device, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="A must have shape"):
        call(A=i["A"][:3])
    with pytest.raises(TypeError):
        call(B=i["B"].float())
    with pytest.raises(TypeError):
        call(dt=i["dt"].half())
    with pytest.raises(ValueError, match="initial_state"):
        call(h0=i["h0"][:, :, :, :8])
    with pytest.raises(ValueError, match="at most 128"):
        big = torch.zeros(1, 10, 2, 136, device=device, dtype=torch.bfloat16)
        call(B=big, C=big, h0=None)
    with pytest.raises(_capi.LampaError):
        call(x=i["x"].cpu())
    for cu in ([0, 4, 9], [1, 10], [0, 7, 3, 10], [0]):
        with pytest.raises(ValueError, match="cu_seqlens"):
            _call({**i, "h0": None}, cu=torch.tensor(cu))
    with pytest.raises(ValueError, match="batch size"):
        two = {k: t.repeat(2, *[1] * (t.dim() - 1)) if k in ("x", "dt", "B", "C") else t for k, t in i.items()}
        _call(two, cu=torch.tensor([0, 10]))
    s = i["h0"]
    step = lambda state, **c: ss.state_space_step(i["x"][:, 0], i["dt"][:, 0], i["A"], i["B"][:, 0], i["C"][:, 0], state, **c)  # noqa: E731
    with pytest.raises(ValueError, match="float32"):
        step(s.bfloat16())
    with pytest.raises(ValueError, match="contiguous"):
        step(s.transpose(-1, -2).contiguous().transpose(-1, -2))
    with pytest.raises(ValueError, match="overlaps"):
        pool = torch.zeros(s.numel() + 4, device=device)
        step(pool[:-4].view_as(s), new_state=pool[4:].view_as(s))
    with pytest.raises(NotImplementedError):
        leaf = i["x"][:, 0].clone().requires_grad_(True)
        ss.state_space_step(leaf, i["dt"][:, 0], i["A"], i["B"][:, 0], i["C"][:, 0], s).float().sum().backward()
