"""GPU parity of the short convolution's state, token step and gradients against float64.

Tolerances: fp32 arithmetic rounded once. y is half a step of its value plus the fp32 error of W + 1 terms through SiLU (whose slope is
at most 1.1), with hardware exponential and reciprocal (each off by a step at most): 16 half-steps of the terms' magnitude.
dweight and dbias add up one term for each token, at most T half-steps of their magnitude."""
import numpy as np
import pytest
import torch

from lampa_amd import layer_ops as lo
from oracle import layer_ops as ol
from oracle import state_space as os_

pytestmark = pytest.mark.gpu

HALF32 = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _close(name, got, want, bound):
    if got.dtype != torch.float32:
        f = torch.finfo(got.dtype)
        bound = bound + f.eps / 2 * (np.abs(want) + bound) + f.smallest_normal * f.eps
    err = np.abs(_np(got) - want)
    assert (err <= bound).all(), (name, float(err.max()), float((err / bound).max()))


def _data(B, T, D, W, dtype, seed, n_seq, bias=True):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    return r(B, T, D).to(dtype), (r(D, W) * 0.5), r(D) if bias else None, r(n_seq, D, W).to(dtype), r(B, T, D).to(dtype)


def _want(x, w, b, past, act, lens):
    """(y, last, magnitude of pre) of packed sequences with what precedes them."""
    W = w.shape[1]
    rows, y, mag, last, t0 = _np(x).reshape(-1, x.shape[-1]), [], [], [], 0
    for k, n in enumerate(lens):
        head = np.zeros((W, x.shape[-1])) if past is None else _np(past[k]).T
        ext = np.concatenate([head, rows[t0:t0 + n]])
        y.append(ol.causal_conv1d(ext[None], _np(w), _np(b), None, act)[0][W:])
        mag.append(ol.causal_conv1d(np.abs(ext)[None], np.abs(_np(w)), None if b is None else np.abs(_np(b)))[0][W:])
        last.append(ext[n:].T)
        t0 += n
    return np.concatenate(y).reshape(x.shape), np.stack(last), np.concatenate(mag).reshape(x.shape)


CASES = [(None, 1, 1, 8, 4), (None, 3, 2, 16, 4), (None, 2, 37, 64, 4), (None, 1, 300, 136, 3), (None, 2, 50, 24, 8), (None, 1, 20, 8, 1),
         ([3, 0, 1, 40, 2, 0, 100, 17, 16, 8], 1, 187, 72, 4), ([0], 1, 0, 8, 2), ([0, 0, 5], 1, 5, 8, 5)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,B,T,D,W", CASES)
def test_prefill_with_state(device, dtype, lens, B, T, D, W):
    n_seq = B if lens is None else len(lens)
    each = [T] * B if lens is None else lens
    cu = None if lens is None else torch.tensor(np.cumsum([0] + lens))
    for bias, act, with_past in ((True, "silu", True), (False, None, True), (True, "silu", False)):
        x, w, b, past, _ = _data(B, T, D, W, dtype, T + D, n_seq, bias)
        past = past if with_past else None
        y, last = lo.causal_conv1d(x.to(device), w.to(device), None if b is None else b.to(device), None, act, cu,
                                   None if past is None else past.to(device), True)
        wy, wl, mag = _want(x, w, b, past, act, each)
        assert y.dtype == dtype and last.shape == (n_seq, D, W) and last.dtype == dtype
        _close("y", y, wy, 16 * HALF32 * mag + 1e-30)
        assert np.array_equal(_np(last), wl)
        only = lo.causal_conv1d(x.to(device), w.to(device), None if b is None else b.to(device), None, act, cu,
                                torch.zeros(n_seq, D, W, dtype=dtype, device=device) if past is None else past.to(device))
        assert torch.equal(only, y)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,B,T,D,W", CASES)
def test_gradients(device, dtype, lens, B, T, D, W):
    n_seq = B if lens is None else len(lens)
    each = [T] * B if lens is None else lens
    cu = None if lens is None else torch.tensor(np.cumsum([0] + lens), device=device)
    for bias, act, with_past in ((True, "silu", False), (False, None, False), (True, "silu", True)):
        x, w, b, past, dy = _data(B, T, D, W, dtype, T * D + W, n_seq, bias)
        leaves = [t.to(device).requires_grad_(True) for t in (x, w, b) if t is not None]
        res = torch.ones(B, T, D, device=device, dtype=dtype, requires_grad=True) if act is None else None
        y = lo.causal_conv1d(leaves[0], leaves[1], leaves[2] if bias else None, res, act, cu,
                             past.to(device) if with_past else None)
        got = torch.autograd.grad(y, leaves + ([] if res is None else [res]), dy.to(device), retain_graph=True)
        again = torch.autograd.grad(y, leaves, dy.to(device))
        for a, c in zip(got, again):
            assert torch.equal(a, c)
        if res is not None:
            assert torch.equal(got[-1], dy.to(device))
        rows = lambda t: _np(t).reshape(-1, D)  # noqa: E731
        want = os_.conv_grads(rows(x), _np(w), _np(b), act, rows(dy), each, _np(past) if with_past else None)
        _, _, pre = _want(x, w, b, past if with_past else None, act, each)
        # |dpre| <= 1.1 |dy|, off by its own 16 half-steps and, through sigma's slope, by the error of pre
        slack = np.abs(rows(dy)) * (1 + pre.reshape(-1, D)) * 20
        mag = os_.conv_grads(np.abs(rows(x)), np.abs(_np(w)), None, None, slack, each, None if not with_past else np.abs(_np(past)))
        for name, a, v, m, n in zip(("x", "weight", "bias"), got, want, mag, (W, T, T)):
            if name == "bias" and not bias:
                continue
            _close(name, a.reshape(v.shape), v, (2 + n) * HALF32 * m + 1e-30)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,D,W", [(1, 8, 4), (3, 20, 4), (64, 640, 4), (2, 7, 1), (2, 16, 8)])
def test_step(device, dtype, n, D, W):
    x, w, b, cache, _ = _data(1, n, D, W, dtype, n * D, n)
    x = x[0]
    wy, wl, mag = _want(x[:, None], w, b, cache, "silu", [1] * n)
    c = cache.to(device)
    new = torch.empty_like(c)
    args = (x.to(device), c, w.to(device), b.to(device), "silu")
    y = lo.causal_conv1d_step(*args, new_cache=new)
    assert torch.equal(c, cache.to(device))
    assert torch.equal(y, lo.causal_conv1d_step(*args)) and torch.equal(c, new)
    _close("y", y, wy[:, 0], 16 * HALF32 * mag[:, 0] + 1e-30)
    assert np.array_equal(_np(new), wl)


def test_steps_continue_a_prefill(device):
    x, w, b, past, _ = _data(2, 30, 16, 4, torch.bfloat16, 1, 2)
    x, w, b = x.to(device), w.to(device), b.to(device)
    whole = lo.causal_conv1d(x, w, b, activation="silu")
    y, cache = lo.causal_conv1d(x[:, :2], w, b, activation="silu", output_final_state=True)
    assert torch.equal(y, whole[:, :2])
    y, cache = lo.causal_conv1d(x[:, 2:20], w, b, activation="silu", initial_state=cache, output_final_state=True)
    assert torch.equal(y, whole[:, 2:20])
    for t in range(20, 30):
        assert torch.equal(lo.causal_conv1d_step(x[:, t], cache, w, b, "silu"), whole[:, t])


def test_strided_and_unaligned_inputs(device):
    wide = torch.randn(2, 60, 40, device=device).bfloat16()
    w, b = torch.randn(16, 4, device=device), torch.randn(16, device=device)
    for cols in (wide[..., 8:24], wide[..., 3:19], wide.flip(1)[..., :16], wide[:1, :1, :16].expand(2, 60, 16)):
        leaf = cols.detach().requires_grad_(True)
        same = cols.detach().contiguous().requires_grad_(True)
        ya, la = lo.causal_conv1d(leaf, w, b, activation="silu", output_final_state=True)
        yb, lb = lo.causal_conv1d(same, w, b, activation="silu", output_final_state=True)
        assert torch.equal(ya, yb) and torch.equal(la, lb)
        dy = wide[..., 5:21]
        assert torch.equal(torch.autograd.grad(ya, leaf, dy)[0], torch.autograd.grad(yb, same, dy)[0])
    cache = torch.zeros(60, 16, 4, device=device, dtype=torch.bfloat16)
    assert torch.equal(lo.causal_conv1d_step(wide[0, :, 3:19], cache.clone(), w, b), lo.causal_conv1d_step(
        wide[0, :, 3:19].contiguous(), cache, w, b))


def test_short_convolution_trains_and_steps(device):
    """The module on top: its gradients, and its step against the same tokens at once."""
    conv = lo.ShortConvolution(24, 4, bias=True).to(device)
    x = torch.randn(2, 19, 24, device=device, requires_grad=True)
    y, _ = conv(x)
    dy = torch.randn_like(y)
    y.backward(dy)
    want = os_.conv_grads(_np(x).reshape(-1, 24), _np(conv.weight)[:, 0], _np(conv.bias), "silu", _np(dy).reshape(-1, 24), [19, 19])
    for got, v in zip((x.grad, conv.weight.grad, conv.bias.grad), want):
        assert np.allclose(_np(got).reshape(v.shape), v, rtol=1e-4, atol=1e-4)
    with torch.no_grad():
        cache = None
        for t in range(19):
            out, cache = conv(x[:, t:t + 1], cache=cache, output_final_state=True)
            assert torch.equal(out, y[:, t:t + 1])


def test_captured_gradients(device):
    x, w, b, _, dy = _data(1, 500, 64, 4, torch.bfloat16, 3, 1)
    leaves = [t.to(device).requires_grad_(True) for t in (x, w, b)]
    dy = dy.to(device)
    step = lambda l: torch.autograd.grad(lo.causal_conv1d(*l, activation="silu"), l, dy)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(leaves)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(leaves)
    for seed in (4, 5, 6):
        new = [t.to(device).requires_grad_(True) for t in _data(1, 500, 64, 4, torch.bfloat16, seed, 1)[:3]]
        for a, c in zip(leaves, new):
            a.data.copy_(c)
        graph.replay()
        for a, c in zip(out, step(new)):
            assert torch.equal(a, c)
        torch.cuda.synchronize()


def test_refusals(device):
    x, w = torch.zeros(2, 5, 16, device=device), torch.zeros(16, 4, device=device)
    past = torch.zeros(2, 16, 4, device=device)
    with pytest.raises(ValueError, match="initial_state must have shape"):
        lo.causal_conv1d(x, w, initial_state=past[:1])
    with pytest.raises(ValueError, match="no residual"):
        lo.causal_conv1d(x, w, residual=x, initial_state=past)
    with pytest.raises(ValueError, match="detached"):
        lo.causal_conv1d(x, w, initial_state=past.clone().requires_grad_(True))
    with pytest.raises(ValueError, match="weight"):
        lo.causal_conv1d(x, w[:8], initial_state=past)
    with pytest.raises(ValueError, match="cu_seqlens"):
        lo.causal_conv1d(x[:1], w, cu_seqlens=torch.tensor([0, 4]), output_final_state=True)
    with pytest.raises(ValueError, match="cache"):
        lo.causal_conv1d_step(x[:, 0], past.half(), w)
    with pytest.raises(ValueError, match="overlaps"):
        pool = torch.zeros(past.numel() + 1, device=device)
        lo.causal_conv1d_step(x[:, 0], pool[:-1].view_as(past), w, new_cache=pool[1:].view_as(past))
    with pytest.raises(ValueError, match="not supported"):
        lo.causal_conv1d_step(x[:, 0], past, w, activation="relu")
    with pytest.raises(NotImplementedError):
        leaf = w.clone().requires_grad_(True)
        lo.causal_conv1d_step(x[:, 0], past, leaf).sum().backward()
