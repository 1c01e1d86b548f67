"""GPU parity of the gated feed-forward block, forward and gradients, against its definition in float64.

Tolerances follow the roundings. H = 2^-24 is half a step of fp32, h half a step of the type. A product of K terms in fp32 is off by
at most (K + 1) H of the sum of its terms' magnitudes. With |G|, |U|, |dS| bounded by those sums (Gm, Um, Sm):
  eG = (D + 1) H Gm, eU and eS likewise;  act is within 1.1 |G| and its slopes within 1.1 (silu' <= 1.1, silu'' <= 0.5), and is
  off by 16 H of |G| + 1 by itself (exponential, division, |G| below 30 half-steps of exponent on a factor of at most 1/4 |G|);
  the hidden value S = act U: eS' = (1.1 eG + 16 H (Gm + 1)) Um + 1.1 Gm eU, rounded by h |S| in 16-bit types (none in fp32);
the last products add their own (K + 1) H, and what is returned is rounded by h."""
import numpy as np
import pytest
import torch

from lampa_amd import _capi
from lampa_amd.feed_forward import gated_feed_forward
from oracle import feed_forward as of
from oracle.linear_recurrence import act as oracle_act

pytestmark = pytest.mark.gpu

H = 2.0 ** -24


def _inputs(rows, D, F, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return [t.to(dtype) for t in (r(rows, D), r(F, D) / D ** 0.5, r(F, D) / D ** 0.5, r(D, F) / F ** 0.5, r(rows, D))]


def _np(t):
    return t.detach().double().cpu().numpy()


def _expected(tensors, activation, dtype):
    """[(value, bound)] of y, dx, dw_gate, dw_up, dw_down, without the outputs' own rounding."""
    x, wg, wu, wd, dy = (_np(t) for t in tensors)
    rows, D, F = x.shape[0], x.shape[1], wg.shape[0]
    h = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0  # half a step of fp16's smallest values
    G, U, dS = x @ wg.T, x @ wu.T, dy @ wd
    mag = lambda a, b: np.abs(a) @ np.abs(b)  # noqa: E731
    Gm, Um, Sm = mag(x, wg.T), mag(x, wu.T), mag(dy, wd)
    e = (D + 1) * H
    value, slope = oracle_act(activation, G)
    ev = 1.1 * e * Gm + 16 * H * (Gm + 1)      # of act and of its slope
    S = value * U
    eS = ev * np.abs(U) + (np.abs(value) + ev) * e * Um + h * np.abs(S) + 4 * H * np.abs(S) + tiny
    dG, dU = dS * U * slope, dS * value
    edG = (ev * np.abs(U) * np.abs(dS) + np.abs(slope) * (e * Um * np.abs(dS) + np.abs(U) * e * Sm) + (h + 8 * H) * np.abs(dG)) + tiny
    edU = ev * np.abs(dS) + np.abs(value) * e * Sm + (h + 8 * H) * np.abs(dU) + tiny
    second = 1.001  # products of two errors
    k = lambda n: (n + 1) * H  # noqa: E731
    return [
        (S @ wd.T, second * (eS @ np.abs(wd.T) + k(F) * mag(S, wd.T))),
        (dG @ wg + dU @ wu, second * (edG @ np.abs(wg) + edU @ np.abs(wu) + k(2 * F) * (mag(dG, wg) + mag(dU, wu)))),
        (dG.T @ x, second * (edG.T @ np.abs(x) + k(rows) * mag(dG.T, x))),
        (dU.T @ x, second * (edU.T @ np.abs(x) + k(rows) * mag(dU.T, x))),
        (dy.T @ S, second * (np.abs(dy.T) @ eS + k(rows) * mag(dy.T, S))),
    ]


def _close(name, got, want, bound, dtype):
    got = _np(got).reshape(want.shape)
    tol = bound + (np.abs(want) + bound) * torch.finfo(dtype).eps / 2 + (2.0 ** -25 if dtype == torch.float16 else 1e-37)
    worst = np.max(np.abs(got - want) / tol, initial=0)
    assert np.isfinite(got).all() and worst <= 1, (name, worst)


def _check(rows, D, F, dtype, activation, seed=1):
    tensors = _inputs(rows, D, F, dtype, seed)
    want = _expected(tensors, activation, dtype)
    *leaves, dy = (t.cuda() for t in tensors)
    y0 = gated_feed_forward(*leaves, activation=activation)
    _close("y", y0, *want[0], dtype)
    leaves = [t.requires_grad_(True) for t in leaves]
    y = gated_feed_forward(*leaves, activation=activation)
    assert torch.equal(y, y0)
    got = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    for name, g, w, leaf in zip(("dx", "dw_gate", "dw_up", "dw_down"), got, want[1:], leaves):
        assert g.shape == leaf.shape and g.dtype == dtype
        _close(name, g, *w, dtype)
    assert all(torch.equal(a, b) for a, b in zip(got, torch.autograd.grad(y, leaves, dy)))


# rows off every tile, widths below, at and above the tiles of 32, 64 and 128, and widths that leave tails of 8
SIZES = [(1, 8, 8), (1, 128, 512), (3, 96, 256), (33, 64, 40), (129, 128, 512), (300, 104, 72), (257, 136, 128), (64, 200, 264),
         (700, 32, 32), (130, 256, 136), (515, 16, 1000), (90, 520, 96), (2, 1024, 1400), (1500, 128, 136)]


@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_forward_and_gradients(size, dtype):
    _check(*size, dtype, "silu")


@pytest.mark.parametrize("activation", [None, "sigmoid", "swish"])
@pytest.mark.parametrize("size", [(65, 128, 96), (40, 168, 48)], ids=lambda s: "x".join(map(str, s)))
def test_activations(activation, size):
    for dtype in (torch.bfloat16, torch.float32):
        _check(*size, dtype, "silu" if activation == "swish" else activation)
    tensors = [t.cuda() for t in _inputs(*size, torch.bfloat16, 2)[:4]]
    assert torch.equal(gated_feed_forward(*tensors, activation="swish"), gated_feed_forward(*tensors, activation="silu"))


@pytest.mark.parametrize("D", [64, 160])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_out_of_line(D, dtype):
    """Column slices, rows off their alignment, turned weights, other shapes in front: the same bits."""
    x, wg, wu, wd, dy = (t.cuda() for t in _inputs(70, D, 96, dtype, 3))
    want = gated_feed_forward(x, wg, wu, wd)
    wide = torch.randn(70, D + 24, device="cuda").to(dtype)
    for at in (8, 3):
        part = wide[:, at:at + D]
        part.copy_(x)
        assert torch.equal(gated_feed_forward(part, wg, wu, wd), want)
    assert torch.equal(gated_feed_forward(x.t().contiguous().t(), wg.t().contiguous().t(), wu, wd), want)
    assert torch.equal(gated_feed_forward(x.view(2, 5, 7, D), wg, wu, wd), want.view(2, 5, 7, D))
    assert torch.equal(gated_feed_forward(x[4], wg, wu, wd), gated_feed_forward(x[4:5], wg, wu, wd)[0])
    buf = torch.zeros(96 * D + 1, dtype=dtype, device="cuda")
    off = buf[1:].view(96, D)
    off.copy_(wg)
    assert torch.equal(gated_feed_forward(x, off, wu, wd), want)
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
    ref = torch.autograd.grad(gated_feed_forward(*leaves), leaves, dy)
    got = torch.autograd.grad(gated_feed_forward(*leaves), leaves, dy.t().contiguous().t())
    assert all(torch.equal(a, b) for a, b in zip(ref, got))
    row = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
    one = torch.autograd.grad(gated_feed_forward(*row).sum(), row)  # a broadcast gradient
    two = torch.autograd.grad(gated_feed_forward(*row), row, torch.ones_like(x))
    assert all(torch.equal(a, b) for a, b in zip(one, two))


@pytest.mark.parametrize("D", [64, 160])
def test_gradients_of_some(D):
    x, wg, wu, wd, dy = (t.cuda() for t in _inputs(200, D, 64, torch.bfloat16, 4))
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
    whole = torch.autograd.grad(gated_feed_forward(*leaves), leaves, dy)
    for mask in range(1, 16):
        some = [t.clone().requires_grad_(bool(mask >> k & 1)) for k, t in enumerate((x, wg, wu, wd))]
        wanted = [k for k in range(4) if mask >> k & 1]
        got = torch.autograd.grad(gated_feed_forward(*some), [some[k] for k in wanted], dy)
        for k, g in zip(wanted, got):
            assert torch.equal(g, whole[k]), (mask, k)


def test_no_rows():
    leaves = [t.cuda().requires_grad_(True) for t in _inputs(0, 32, 64, torch.bfloat16, 5)[:4]]
    y = gated_feed_forward(*leaves)
    assert y.shape == (0, 32)
    assert all(not g.any() for g in torch.autograd.grad(y.sum(), leaves))


@pytest.mark.parametrize("D", [64, 160])
def test_values_that_are_not_finite_stay_in_their_rows(D):
    x, wg, wu, wd, dy = (t.cuda() for t in _inputs(200, D, 96, torch.bfloat16, 6))
    clean = gated_feed_forward(x, wg, wu, wd)
    for bad in (float("nan"), float("inf"), 1e38):
        hurt = x.clone()
        hurt[77, 5] = bad
        y = gated_feed_forward(hurt, wg, wu, wd)
        keep = [k for k in range(200) if k != 77]
        assert torch.equal(y[keep], clean[keep])
        leaf = hurt.requires_grad_(True)
        dx, = torch.autograd.grad(gated_feed_forward(leaf, wg, wu, wd), leaf, dy)
        assert dx[keep].isfinite().all()


@pytest.mark.parametrize("size", [(600, 64, 256), (100, 160, 96)], ids=lambda s: "x".join(map(str, s)))
def test_captured_and_replayed(size):
    sets = [[t.cuda() for t in _inputs(*size, torch.bfloat16, 10 + k)] for k in range(2)]
    static = [t.clone() for t in sets[0]]
    leaves = [t.detach().requires_grad_(True) for t in static[:4]]

    def step():
        y = gated_feed_forward(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, static[4]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for rep in range(4):
        for a, b in zip(static, sets[rep % 2]):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_streams_side_by_side():
    sets = [[t.cuda() for t in _inputs(3000, 128, 256, torch.bfloat16, 20 + k)[:4]] for k in range(2)]
    want = [gated_feed_forward(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for rep in range(3):
        for t, s in zip(sets, streams):
            with torch.cuda.stream(s):
                got.append(gated_feed_forward(*t))
    torch.cuda.synchronize()
    for k, y in enumerate(got):
        assert torch.equal(y, want[k % 2])


def test_refusals():
    x, wg, wu, wd, _ = (t.cuda() for t in _inputs(10, 32, 64, torch.bfloat16, 7))
    for error, args in ((ValueError, (x[:, :24], wg, wu, wd)), (ValueError, (x, wg, wu[:32], wd)), (ValueError, (x, wg, wu, wd.t())),
                        (ValueError, (x[:, :12], wg[:, :12], wu[:, :12], wd[:12])), (TypeError, (x.float(), wg, wu, wd)),
                        (TypeError, (x, wg, wu, wd.half())), (TypeError, tuple(t.double() for t in (x, wg, wu, wd))),
                        (ValueError, (x, wg[:60], wu[:60], wd[:, :60])), (_capi.LampaError, (x, wg, wu, wd.cpu()))):
        with pytest.raises(error):
            gated_feed_forward(*args)
    with pytest.raises(ValueError):
        gated_feed_forward(x, wg, wu, wd, activation="relu")
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(Exception):
            torch.autograd.forward_ad.unpack_dual(gated_feed_forward(dual, wg, wu, wd))
