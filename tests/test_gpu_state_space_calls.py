"""Calls of the state-space operators, the convolution and the norms that a program may make beside the ordinary ones: rubbish behind
the last sequence, gradients through a single token, forward-mode gradients, slices of long tensors, parameters without gradients."""
import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from lampa_amd import block
from lampa_amd import layer_ops as lo
from lampa_amd import state_space as ss
from oracle import state_space as os_
from test_gpu_conv_state import HALF32, _close, _np, _want
from test_gpu_state_space import _bound, _call, _check, _half, _inputs, _oracle, _to

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("W", [1, 4, 8])
@pytest.mark.parametrize("activation", [None, "silu"])
@pytest.mark.parametrize("rubbish", [float("nan"), float("inf")])
def test_convolution_gradients_leave_out_what_lies_behind_the_sequences(device, dtype, W, activation, rubbish):
    """A buffer of fixed size whose last rows belong to no sequence: the gradients of the call without them, to the bit where
    the sums run over the same workgroups, and zero for the rows themselves."""
    gen = torch.Generator().manual_seed(W)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    T, D, used = 200, 24, 137
    x, dy = r(1, T, D).to(dtype), r(1, T, D).to(dtype)
    w, b, past = r(D, W), r(D), r(3, D, W).to(dtype)
    x[:, used:] = rubbish
    cu = torch.tensor([0, 100, 100, used], device=device)
    out = []
    for rows in (T, used):
        leaves = [t.to(device).requires_grad_(True) for t in (x[:, :rows], w, b)]
        y = lo.causal_conv1d(*leaves, activation=activation, cu_seqlens=cu, initial_state=past.to(device))
        out.append((y, *torch.autograd.grad(y, leaves, dy[:, :rows].to(device))))
    (y, dx, dw, db), (y2, dx2, dw2, db2) = out
    assert torch.equal(y[:, :used], y2) and not y[:, used:].any()
    assert torch.equal(dx[:, :used], dx2) and not dx[:, used:].any()
    # sums of 137 terms over the same rows, in an order that depends on the rows in all
    bound = 2 * used * 2.0 ** -24 * (dy[:, :used].abs().float().sum(1) * 1.1).max().item() * max(1.0, x[:, :used].abs().max().item())
    assert (dw - dw2).abs().max().item() <= bound and (db - db2).abs().max().item() <= bound


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("packed", [False, True])
def test_short_convolution_trains_through_a_single_token(device, dtype, packed):
    """One token with a cache, or with the cache asked for, has the gradients that more tokens have; the cache moves on as without
    gradients, and moving it on again does not disturb the backward. Tolerances as in test_gpu_conv_state.test_gradients."""
    D, W, n = 24, 4, 3
    gen = torch.Generator().manual_seed(7)
    r = lambda *s: torch.randn(*s, generator=gen).to(dtype).to(device)  # noqa: E731
    conv = lo.ShortConvolution(D, W, bias=True).to(device)
    shape, cu = ((1, n, D), torch.arange(n + 1, device=device)) if packed else ((n, 1, D), None)
    for given in (True, False):
        x, dy, cache = r(*shape), r(*shape), r(n, D, W) if given else None
        start = torch.zeros(n, D, W, device=device, dtype=dtype) if cache is None else cache.clone()
        with torch.no_grad():
            want_y, want_cache = conv(x, cache=start.clone(), cu_seqlens=cu)
        leaf = x.clone().requires_grad_(True)
        y, cache = conv(leaf, cache=cache, output_final_state=True, cu_seqlens=cu)
        assert torch.equal(y, want_y) and torch.equal(cache, want_cache)
        with torch.no_grad():
            conv(x, cache=cache, cu_seqlens=cu)
        got = torch.autograd.grad(y, [leaf, conv.weight, conv.bias], dy)
        rows = lambda t: _np(t).reshape(-1, D)  # noqa: E731
        w, b = _np(conv.weight).reshape(D, W), _np(conv.bias)
        want = os_.conv_grads(rows(x), w, b, "silu", rows(dy), [1] * n, _np(start))
        _, _, pre = _want(x.reshape(1, n, D), conv.weight.reshape(D, W), conv.bias, start, "silu", [1] * n)
        slack = abs(rows(dy)) * (1 + pre.reshape(-1, D)) * 20
        mag = os_.conv_grads(abs(rows(x)), abs(w), None, None, slack, [1] * n, abs(_np(start)))
        for name, a, v, m, terms in zip(("x", "weight", "bias"), got, want, mag, (W, n, n)):
            _close(name, a.reshape(v.shape), v, (2 + terms) * HALF32 * m + 1e-30)


@pytest.mark.parametrize("x_type,cache_type", [(torch.bfloat16, torch.float32), (torch.float16, torch.float32), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("grad", [False, True])
def test_a_cache_of_another_type_sets_the_type_of_the_step(device, x_type, cache_type, grad):
    """The step's window, sums and output are of the cache's type, as the convolution of that window is; what it holds is kept to
    the bit, also where the cache is no contiguous tensor."""
    D, W, n = 16, 4, 3
    gen = torch.Generator().manual_seed(8)
    conv = lo.ShortConvolution(D, W, bias=True).to(device).requires_grad_(grad)
    start = torch.randn(n, D, W, generator=gen).to(cache_type).to(device)
    cache = start.transpose(0, 1).contiguous().transpose(0, 1)
    assert not cache.is_contiguous()
    window = start
    for _ in range(W + 1):
        x = torch.randn(n, 1, D, generator=gen).to(x_type).to(device)
        y, back = conv(x, cache=cache)
        assert back is cache
        window = torch.cat([window[..., 1:], x.transpose(1, 2).to(cache_type)], -1)
        want = lo.causal_conv1d(window.transpose(1, 2), conv.weight.reshape(D, W), conv.bias, activation="silu")[:, -1:]
        assert y.dtype == cache_type and torch.equal(y, want) and torch.equal(cache, window)


NAMES = ["x", "dt", "A", "B", "C", "D", "dt_bias", "h0"]


def _scan_against_float64(device, i, dy, dht, dtype, T, P, N, H, G):
    """Outputs and gradients of one sequence within the bounds of test_gpu_state_space."""
    (y, last, g), (ym, lastm, gm) = _oracle(i, [T], dy=dy, dht=dht)
    d = _to(i, device, grad=True)
    got, ht = _call(d)
    _check("y", got, y, _bound(dtype, T, y, ym, N), dtype)
    _check("last", ht, last, _bound(dtype, T, last, lastm, 0, False))
    grads = torch.autograd.grad([got, ht], [d[k] for k in NAMES], [dy.to(device), dht.to(device)])
    for k, a in zip(NAMES, grads):
        wide = {"x": N, "B": P * H // G, "C": P * H // G, "h0": 0, "D": T * P}.get(k, N * P + T)
        _check(k, a, g[k], _bound(dtype, T, g[k], gm[k], wide, k in ("x", "B", "C")), d[k].dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size", [1e-2, 1e-3, 1e-4, 1e-5])
@pytest.mark.parametrize("seg", [None, 64])
def test_small_values_keep_the_bits_of_states_and_adjoints(device, dtype, size, seg, monkeypatch):
    """x or C, which the states and adjoints are made of beside dy, small all over or in every other column: two operands of 11
    bits hold a state as they do where x is about one."""
    if seg:
        monkeypatch.setattr(ss, "_segment_tokens", lambda *a: seg)
    T, H, P, G, N = 200, 2, 32, 1, 40
    gen = torch.Generator().manual_seed(3)
    for small, alternate in (("x", False), ("dy", False), ("C", False), ("x", True), ("C", True)):
        i = _inputs((1, T), H, P, G, N, dtype, 80, 1)
        dy, dht = torch.randn(1, T, H, P, generator=gen).to(dtype), torch.randn(1, H, N, P, generator=gen)
        step = 2 if alternate else 1
        if small == "dy":
            dy, dht = dy * size, dht * size
        else:
            i[small] = i[small].clone()
            i[small][..., ::step] = (i[small].float() * size).to(dtype)[..., ::step]
            if small == "x":
                i["h0"][..., ::step] *= size
            else:
                dht[..., ::step, :] *= size
        _scan_against_float64(device, i, dy, dht, dtype, T, P, N, H, G)


def test_forward_mode_gradients_are_refused(device):
    """No operator has forward-mode gradients: a tangent on any input raises instead of coming back without one, with gradients
    enabled or not; in the same context inputs without tangents are taken as ever."""
    gen = torch.Generator().manual_seed(9)
    r = lambda *s: torch.randn(*s, generator=gen).to(device)  # noqa: E731
    conv = dict(x=r(2, 5, 16), weight=r(16, 4), bias=r(16))
    step = dict(x=r(2, 16), cache=r(2, 16, 4), weight=r(16, 4), bias=r(16))
    norm = dict(x=r(2, 5, 16), residual=r(2, 5, 16), weight=r(16), post_weight=r(16), gate=r(2, 5, 16), residual_scale=r(16))
    scan = dict(x=r(2, 5, 2, 8), dt=r(2, 5, 2), A=-r(2).abs(), B=r(2, 5, 1, 8), C=r(2, 5, 1, 8), D=r(2), dt_bias=r(2),
                initial_state=r(2, 2, 8, 8))
    token = {k: t[:, 0] if k in ("x", "dt", "B", "C") else t for k, t in scan.items() if k != "initial_state"}
    short = lo.ShortConvolution(16, 4, bias=True).to(device).requires_grad_(False)
    calls = [
        (lo.causal_conv1d, conv), (lo.causal_conv1d, dict(conv, residual=r(2, 5, 16))),
        (lambda **k: lo.causal_conv1d(**k, output_final_state=True), dict(conv, initial_state=r(2, 16, 4))),
        (lambda **k: lo.causal_conv1d_step(**k, new_cache=torch.empty(2, 16, 4, device=device)), step),
        (lo.residual_norm, norm), (lambda **k: ss.state_space_scan(**k, output_final_state=True), scan),
        (lambda **k: ss.state_space_step(**k, new_state=torch.empty(2, 2, 8, 8, device=device)), dict(token, state=r(2, 2, 8, 8))),
        (lambda x: short(x, cache=torch.zeros(2, 16, 4, device=device)), dict(x=r(2, 1, 16))),
    ]
    for call, inputs in calls:
        want = call(**inputs)
        for enabled in (True, False):
            with forward_ad.dual_level(), torch.set_grad_enabled(enabled):
                got = call(**inputs)
                for a, b in zip(*((t if isinstance(t, tuple) else (t,)) for t in (got, want))):
                    assert torch.equal(a, b)
                for name in inputs:
                    dual = forward_ad.make_dual(inputs[name], torch.ones_like(inputs[name]))
                    with pytest.raises(RuntimeError, match="jvp"):  # (NotImplementedError is one)
                        call(**dict(inputs, **{name: dual}))


def test_a_cache_with_a_gradient_is_refused_in_the_backward(device):
    """The token steps have no gradients, of what they are handed in their caches neither."""
    cache = torch.randn(2, 16, 4, device=device, requires_grad=True)
    y = lo.causal_conv1d_step(torch.randn(2, 16, device=device), cache * 1.0, torch.randn(16, 4, device=device))
    with pytest.raises(NotImplementedError):
        y.sum().backward()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 2])
def test_tokens_out_of_long_sequences(device, dtype, T):
    """The next token of each of several sequences, sliced out of tensors whose sequences lie more than 2^24 elements apart: the
    bits of a contiguous copy, gradients too."""
    long = dict(x=torch.zeros(3, 17000, 2, 512, device=device, dtype=dtype), B=torch.zeros(3, 17000, 16, 64, device=device, dtype=dtype),
                C=torch.zeros(3, 17000, 16, 64, device=device, dtype=dtype), dt=torch.zeros(3, 17000, 1000, device=device, dtype=dtype))
    gen = torch.Generator().manual_seed(10)
    sizes = dict(x=(3, T, 2, 512), B=(3, T, 1, 64), C=(3, T, 1, 64), dt=(3, T, 2))
    ends = dict(x=slice(None), B=slice(5, 6), C=slice(0, 1), dt=slice(7, 9))
    parts = {}
    for k, t in long.items():
        assert t.stride(0) > 2 ** 24
        parts[k] = t[:, 9000:9000 + T, ends[k]]
        parts[k].copy_(torch.randn(*sizes[k], generator=gen))
    shared = dict(A=-torch.rand(2, generator=gen).to(device), D=None, dt_bias=None, h0=torch.randn(3, 2, 64, 512, generator=gen).to(device))
    dy = torch.randn(3, T, 2, 512, generator=gen).to(dtype).to(device)
    out = []
    for copy in (False, True):
        d = {k: (t.contiguous().clone() if copy else t).detach().requires_grad_(True) for k, t in parts.items()}
        y, ht = _call({**d, **shared})
        with torch.no_grad():
            plain = _call({**d, **shared})
        assert torch.equal(y, plain[0]) and torch.equal(ht, plain[1])
        out.append([y, ht, *torch.autograd.grad([y, ht], list(d.values()), [dy, ht.detach()])])
    for a, b in zip(*out):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_parameters_without_gradients_are_launched_as_plain_tensors(device, dtype, monkeypatch):
    """Under no_grad a layer's parameters make no training call: the segments and the bits of the call on plain tensors, and
    nothing kept of it."""
    asked = []
    rule = ss._segment_tokens
    monkeypatch.setattr(ss, "_segment_tokens", lambda *a: asked.append(a[-1]) or rule(*a))
    T, H, P, N = 40000, 8, 64, 64
    d = _to(_inputs((1, T), H, P, 1, N, dtype, 90, 1), device)
    held = {k: torch.nn.Parameter(t) if k in ("A", "D", "dt_bias", "h0") else t for k, t in d.items()}
    assert rule(T, T, H, N, torch.bfloat16, True) != rule(T, T, H, N, torch.bfloat16, False)
    with torch.no_grad():
        want = _call(d)
        before = torch.cuda.memory_allocated()
        got = _call(held)
        kept = torch.cuda.memory_allocated() - before - sum(t.numel() * t.element_size() for t in got)
    assert asked == [False, False] and all(torch.equal(a, b) for a, b in zip(got, want))
    assert kept < 2 ** 16  # the outputs alone, as the allocator rounds them up
    _call(held)
    assert asked[2:] == [True]


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_final_state_is_not_kept_for_the_gradients(device, dtype):
    """Between forward and backward a call holds its segments' states and no final state, asked for or not, unless the caller does;
    the gradients are the same bits either way."""
    n, T, H, P, N = 40, 500, 2, 64, 128
    d = _to(_inputs((n, T), H, P, 1, N, dtype, 91, n), device, grad=True)
    dy = torch.randn(n, T, H, P, device=device).to(dtype)
    size = n * H * N * P * 4
    assert ss._segment_tokens(T, n * T, H, N, dtype, True) < T  # more than one segment a sequence
    held, grads = [], []
    for final in (False, True):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y, ht = _call(d, final=final)
        assert (ht is None) == (not final)
        del ht
        held.append(torch.cuda.memory_allocated() - before - y.numel() * y.element_size())
        grads.append(torch.autograd.grad(y, [d[k] for k in NAMES], dy))
        del y
    seg = ss._segment_tokens(T, n * T, H, N, dtype, True)
    slots = n * -(-T // seg)
    for h in held:
        assert h < slots * H * N * P * 4 + size / 2, (h, size)
    for a, b in zip(*grads):
        assert torch.equal(a, b)


def test_a_final_state_moved_on_in_place_is_noticed(device):
    """With another state for the step the scan's gradients are there; with the state moved on itself its backward raises."""
    d = _to(_inputs((1, 700), 2, 64, 1, 64, torch.bfloat16, 92, 1), device, grad=True)
    token = lambda state, **k: ss.state_space_step(  # noqa: E731
        *(d[k][:, 0].detach() if k in ("x", "dt", "B", "C") else d[k].detach() for k in ("x", "dt", "A", "B", "C")), state.detach(), **k)
    y, ht = _call(d)
    want = torch.autograd.grad([y, ht], d["x"], [torch.ones_like(y), torch.ones_like(ht)], retain_graph=True)[0]
    token(ht, new_state=torch.empty_like(ht))
    again = torch.autograd.grad([y, ht], d["x"], [torch.ones_like(y), torch.ones_like(ht)], retain_graph=True)[0]
    assert torch.equal(want, again)
    token(ht)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad([y, ht], d["x"], [torch.ones_like(y), torch.ones_like(ht)])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("every", [37, 3])
@pytest.mark.parametrize("seg", [None, 64])
def test_strong_decays_to_the_last_bits(device, dtype, every, seg, monkeypatch):
    """Tokens whose step wipes the state, one in 37 or one in 3, beside steps of zero and ordinary ones, outputs and gradients. fp32
    and the states that are handed on take no difference of long sums: the bounds of any other call. In the 16-bit outputs a pair's
    weight is 2^(gamma_t - gamma_s) of two sums over the chunk's tokens, each rounded to fp32 once: half a step of the largest."""
    if seg:
        monkeypatch.setattr(ss, "_segment_tokens", lambda *a: seg)
    T, H, P, N = 260, 2, 32, 32
    i = _inputs((1, T), H, P, 1, N, dtype, 93, 1, rate=1.0)
    dt = torch.full((1, T, H), 0.05)
    dt[:, ::every] = 2000.0
    dt[:, 5::41] = 0.0
    i["dt"], i["dt_bias"] = dt.to(dtype), None
    i["x"] = i["x"].clone()
    i["x"][:, dt[0, :, 0] == 2000] = 0  # their own write is not what is looked at
    gen = torch.Generator().manual_seed(94)
    dy, dht = torch.randn(1, T, H, P, generator=gen).to(dtype), torch.randn(1, H, N, P, generator=gen)
    (y, last, g), (ym, lastm, gm) = _oracle(i, [T], softplus=False, dy=dy, dht=dht)
    g2 = np.maximum(_np(i["dt"])[0] * _np(i["A"]), -104.0) * np.log2(np.e)
    deepest = max(abs(g2[t:t + 64].sum(0)).max() for t in range(0, T, 64))
    weights = 0.0 if dtype == torch.float32 else 2 * np.spacing(np.float32(deepest)) / 2 * np.log(2)
    d = _to(i, device, grad=True)
    got, ht = _call(d, softplus=False)
    _check("y", got, y, _bound(dtype, T, y, ym, N) + weights * ym, dtype)
    _check("last", ht, last, _bound(dtype, T, last, lastm, 0, False))
    names = [k for k in NAMES if k != "dt_bias"]
    for k, a in zip(names, torch.autograd.grad([got, ht], [d[k] for k in names], [dy.to(device), dht.to(device)])):
        wide = {"x": N, "B": P * H, "C": P * H, "h0": 0, "D": T * P}.get(k, N * P + T)
        extra = weights * gm[k] if k in ("x", "B", "C") else 0.0
        if k == "dt" and dtype != torch.float32:
            # What passes a token is a prefix sum, over 16 tokens, of the pairs that begin minus those that end there. Behind a token that
            # wipes the state nothing passes, but the sum of up to 16 terms each way is off by 32 half-steps of the pairs before it, and
            # the terms by as many of their own; gm of the chunk's first tokens bounds all pairs that end later.
            top = np.concatenate([np.repeat(gm[k][t:t + 64].max(0, keepdims=True), len(gm[k][t:t + 64]), 0) for t in range(0, T, 64)])
            extra = 64 * HALF32 * top
        bound = _bound(dtype, T, g[k], gm[k], wide, k in ("x", "B", "C")) + extra
        # a step of 2000 leaves gradients beyond fp16's range: infinite with their sign, or the largest value, and nothing else
        a, most = a.detach().double().cpu().numpy().reshape(g[k].shape), torch.finfo(d[k].dtype).max
        slack = (bound + _half(d[k].dtype) * abs(g[k])) * 2
        beyond = abs(g[k]) + slack > most
        assert (a[beyond] * np.sign(g[k][beyond]) >= np.minimum(most, abs(g[k]) - slack)[beyond]).all(), k
        _check(k, torch.from_numpy(np.where(beyond, g[k], a)), g[k], bound, d[k].dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_decay_gradients_of_a_training_step(device, dtype, monkeypatch):
    """A_log and dt_bias of every layer of a block in a training step, against float64 on what the layer's scan was given: sums of both
    signs over all tokens, within the bounds of the scan's own tests and the rounding to the parameters' type."""
    lens = [70, 0, 1, 30]
    torch.manual_seed(95)
    model = block.StateSpaceBlock(64, 3, residual_scale=0.7, d_state=16, head_dim=16, expand=2, n_groups=2).to(dtype).to(device)
    calls, upstream = [], {}
    scan = block.state_space_scan

    def recorded(x, dt, A, B, C, **k):
        y, state = scan(x, dt, A, B, C, **k)
        n = len(calls)
        calls.append(dict(x=x, dt=dt, A=A, B=B, C=C, D=k["D"], dt_bias=k["dt_bias"], h0=None))
        y.register_hook(lambda grad: upstream.update({n: grad.clone()}))
        return y, state

    monkeypatch.setattr(block, "state_space_scan", recorded)
    x = torch.randn(1, sum(lens), 64, device=device).to(dtype)
    out, _ = model(x, torch.tensor([0, 70, 70, 71, 101], device=device))
    out.backward(torch.randn_like(out))
    assert len(calls) == len(upstream) == 3
    for n, layer in enumerate(model.layers):
        i = {k: None if t is None else t.detach().cpu() for k, t in calls[n].items()}
        (_, _, g), (_, _, gm) = _oracle(i, lens, dy=upstream[n].cpu())
        N, P = i["B"].shape[-1], i["x"].shape[-1]
        bound = lambda k: _bound(dtype, max(lens), g[k], gm[k], N * P + sum(lens), False)  # noqa: E731
        A = _np(i["A"])
        _check("A_log", layer.A_log.grad, g["A"] * A, (bound("A") + 4 * HALF32 * gm["A"]) * abs(A), dtype)
        _check("dt_bias", layer.dt_bias.grad, g["dt_bias"], bound("dt_bias"), dtype)


def _decay_gradient(device, x, delta, A, B, C, dy):
    """What the decay's gradient is made of, in float64, token by token: dg_t = <R_t, a_t S_{t-1}> and x_t . (R_t^T B_t), both [T, H]."""
    xs, ds, Bs, Cs, ys = (t[0].double() for t in (x, delta, B, C, dy))
    T, H, P = xs.shape
    N = Bs.shape[-1]
    decay = torch.exp(ds * A.double())
    states = torch.zeros(T + 1, H, N, P, dtype=torch.float64, device=device)
    for t in range(T):
        states[t + 1] = decay[t, :, None, None] * states[t] + (ds[t, :, None] * Bs[t])[:, :, None] * xs[t][:, None, :]
    R = torch.zeros(H, N, P, dtype=torch.float64, device=device)
    dg, reach = (torch.empty(T, H, dtype=torch.float64, device=device) for _ in range(2))
    for t in range(T - 1, -1, -1):
        R += Cs[t, 0][None, :, None] * ys[t][:, None, :]
        reach[t] = (R * Bs[t, 0][None, :, None] * xs[t][:, None, :]).sum((-1, -2))
        R *= decay[t, :, None, None]
        dg[t] = (R * states[t]).sum((-1, -2))
    return dg, reach


def _decaying(device, dtype, rates, step, T, P, N):
    H = len(rates)
    gen = torch.Generator(device=device).manual_seed(96)
    r = lambda *s: torch.randn(*s, generator=gen, device=device)  # noqa: E731
    silu = torch.nn.functional.silu
    x, B, C, dy = silu(r(1, T, H, P)).to(dtype), silu(r(1, T, 1, N)).to(dtype), silu(r(1, T, 1, N)).to(dtype), r(1, T, H, P).to(dtype)
    A, delta = -torch.tensor(rates, device=device), torch.nn.functional.softplus(r(1, T, H) * 0.7 + float(np.log(np.expm1(step))))
    leaves = [A.clone().requires_grad_(True), delta.clone().requires_grad_(True)]
    y, _ = ss.state_space_scan(x, leaves[1], leaves[0], B, C)
    return (A, delta[0], *torch.autograd.grad(y, leaves, dy), *_decay_gradient(device, x, delta, A, B, C, dy))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_the_decay_gradient_has_no_bias(device, dtype):
    """dA is a sum over all tokens of delta_t dg_t. Errors of a token's dg that are as likely above as below add up like a random walk,
    ones that lean to one side like the number of tokens. A dg is four sums in fp32, off by two half-steps (2^-23) of dg's usual size,
    the same for the 64 tokens of a chunk at worst and independent between chunks: 4 sigma of their sum is
    4 * 2^-23 * sqrt(64 T) * rms(delta dg). (A lean of one half-step would come to T / (8 sqrt(64 T)) = 2.2 times that.)"""
    T = 19200
    A, delta, dA, _, dg, _ = _decaying(device, dtype, (1.0, 2.0, 4.0, 8.0), 0.013, T, 32, 32)
    terms = delta.double() * dg
    bound = 4 * 2.0 ** -23 * (64 * T) ** 0.5 * terms.pow(2).mean(0).sqrt()
    off = (dA.double() - terms.sum(0)).abs()
    assert (off <= bound + 2.0 ** -24 * dA.abs()).all(), (off / bound).tolist()


@pytest.mark.parametrize("rates,step", [((1.0, 2.0, 4.0, 8.0), 0.013), ((6.0, 10.0, 15.0, 30.0), 0.1)])
@pytest.mark.parametrize("P,N", [(32, 32), (8, 64), (64, 64), (80, 100)])
def test_the_exact_decay_gradient_where_little_passes_a_token(device, rates, step, P, N):
    """fp32: dg is summed up from the end of 16 tokens, each of which adds what ends there and takes away what begins there: two sums off
    by two half-steps each, of dg's usual size if a token's own output, which is e^|delta A| as large, is in neither. So the k-th dg
    from the end is off by 2 sqrt(2 k) half-steps (8.2 rms over the 16), and ddt = A dg + reach by that times A and by four half-steps
    of reach; 1.25 times their sum in squares is allowed. In dA = sum delta_t dg_t the error of a token's sums comes with the deltas
    of all tokens before it in the 16; 4 sigma."""
    T, hs = 4800, 2.0 ** -24
    A, delta, dA, ddt, dg, reach = _decaying(device, torch.float32, rates, step, T, P, N)
    A, delta = A.double(), delta.double()
    rms = lambda t: t.pow(2).mean(0).sqrt()  # noqa: E731
    off = rms(ddt[0].double() - (A * dg + reach))
    bound = 1.25 * hs * ((8.2 * A * rms(dg)) ** 2 + (4 * rms(reach)) ** 2).sqrt()
    assert (off <= bound).all(), (off / bound).tolist()
    carried = delta.view(T // 16, 16, -1).cumsum(1).flatten(0, 1)
    bound = 4 * 2 * 2 ** 0.5 * hs * rms(dg) * carried.pow(2).sum(0).sqrt() + hs * dA.abs()
    off = (dA.double() - (delta * dg).sum(0)).abs()
    assert (off <= bound).all(), (off / bound).tolist()


def test_a_residual_or_bias_of_another_size_is_refused(device):
    """The kernels read a row of the residual for each of x and a value of the bias for each channel: nothing is broadcast."""
    x, w = torch.zeros(2, 5, 16, device=device), torch.zeros(16, 4, device=device)
    for leaf in (x, x.clone().requires_grad_(True)):
        for shape in ((1, 5, 16), (2, 1, 16), (2, 5, 8)):
            with pytest.raises(ValueError, match="residual"):
                lo.causal_conv1d(leaf, w, residual=torch.zeros(*shape, device=device))
        for size in (1, 8, 32):
            with pytest.raises(ValueError, match="bias"):
                lo.causal_conv1d(leaf, w, torch.zeros(size, device=device))


def test_taps_and_bias_of_other_shapes_train(device):
    """Without a state the taps may come in any shape of D x W values and the bias in any of D, with gradients as without."""
    gen = torch.Generator().manual_seed(11)
    x, w, b = (torch.randn(*s, generator=gen).to(device) for s in ((2, 9, 16), (16, 4), (16,)))
    with torch.no_grad():
        want = lo.causal_conv1d(x, w, b, activation="silu")
    flat = [t.clone().requires_grad_(True) for t in (w, b)]
    grads = torch.autograd.grad(lo.causal_conv1d(x, *flat, activation="silu").sum(), flat)
    for shape, bias_shape in (((16, 1, 4), (1, 16)), ((64,), (16, 1)), ((1, 16, 4), (1, 1, 16))):
        leaves = [w.reshape(shape).clone().requires_grad_(True), b.reshape(bias_shape).clone().requires_grad_(True)]
        with torch.no_grad():
            assert torch.equal(lo.causal_conv1d(x, *leaves, activation="silu"), want)
        y = lo.causal_conv1d(x, *leaves, activation="silu")
        assert torch.equal(y, want)
        for a, c, leaf in zip(torch.autograd.grad(y.sum(), leaves), grads, leaves):
            assert a.shape == leaf.shape and torch.equal(a.reshape(c.shape), c)


@pytest.mark.parametrize("whole", [False, True])
def test_boundaries_on_the_host_for_a_layer_and_a_block(device, whole):
    """With and without caches, trained or not: the bits of boundaries on the GPU, and a check of what they hold."""
    torch.manual_seed(12)
    args = dict(d_state=16, head_dim=16, expand=2, n_groups=2)
    model = (block.StateSpaceBlock(64, 2, **args) if whole else block.StateSpaceLayer(64, **args)).to(device)
    x = torch.randn(1, 50, 64, device=device)
    host = torch.tensor([0, 20, 20, 50])
    for caches in (False, True):
        want = model(x, host.to(device), **{"output_caches" if whole else "output_cache": caches})[0]
        got = model(x, host, **{"output_caches" if whole else "output_cache": caches})[0]
        assert torch.equal(got, want)
        with torch.no_grad():
            assert torch.equal(model(x, host)[0], model(x, host.to(device))[0])
        for a, b in zip(torch.autograd.grad(got.sum(), list(model.parameters())), torch.autograd.grad(want.sum(), list(model.parameters()))):
            assert torch.equal(a, b)
    with pytest.raises(ValueError, match="cu_seqlens"):
        model(x, torch.tensor([0, 20, 49]))
