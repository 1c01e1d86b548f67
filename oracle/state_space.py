"""CPU oracle for the state-space operators (TEST INFRASTRUCTURE ONLY): the selective scan and its gradients token by token,
the gradients of the short convolution, and the norms around a block with their gradients, in float64 numpy.

The recurrences are the defining ones (``models/baselines/full_mamba2.py:221-430`` calls them from a package the reference does
not hold: parity unpinned, so ``tests/test_oracle_state_space.py`` pins them against closed forms and finite differences)."""
import numpy as np


def sigmoid(x):
    return 1.0 / (1.0 + np.exp(-x))


def softplus(x):
    return np.maximum(x, 0) + np.log1p(np.exp(-np.abs(x)))


def step_sizes(dt, bias=None, use_softplus=False):
    raw = np.asarray(dt, np.float64) + (0.0 if bias is None else np.asarray(bias, np.float64))
    return softplus(raw) if use_softplus else raw


def _wide(t, H):
    return np.repeat(np.asarray(t, np.float64), H // t.shape[-2], axis=-2)


def scan(x, delta, A, B, C, D=None, h0=None, lens=None):
    """x [T, H, P], delta [T, H], A [H], B, C [T, G, N], h0 [sequences, H, N, P]; sequences of `lens` tokens one after the other.
    Returns (y [T, H, P], last states [sequences, H, N, P])."""
    x, delta, A = (np.asarray(t, np.float64) for t in (x, delta, A))
    T, H, P = x.shape
    B, C = _wide(B, H), _wide(C, H)
    lens = [T] if lens is None else lens
    y = np.zeros_like(x)
    last = np.zeros((len(lens), H, B.shape[-1], P))
    t = 0
    for i, n in enumerate(lens):
        S = np.zeros((H, B.shape[-1], P)) if h0 is None else np.array(h0[i], np.float64)
        for _ in range(n):
            S = np.exp(delta[t] * A)[:, None, None] * S + delta[t][:, None, None] * B[t][:, :, None] * x[t][:, None, :]
            y[t] = np.einsum("hn,hnp->hp", C[t], S)
            t += 1
        last[i] = S
    if D is not None:
        y += np.asarray(D, np.float64)[:, None] * x
    return y, last


def scan_grads(x, delta, A, B, C, D, h0, lens, dy, dht=None):
    """Gradients of sum(y dy) + sum(last dht): a dict over x, delta, A, B, C, D, h0 (B and C summed over a group's heads)."""
    x, delta, A, dy = (np.asarray(t, np.float64) for t in (x, delta, A, dy))
    T, H, P = x.shape
    G, N = np.shape(B)[-2:]
    Bw, Cw = _wide(B, H), _wide(C, H)
    lens = [T] if lens is None else lens
    g = {"x": np.zeros_like(x), "delta": np.zeros_like(delta), "A": np.zeros(H), "B": np.zeros((T, H, N)), "C": np.zeros((T, H, N)),
         "D": np.einsum("thp,thp->h", x, dy), "h0": np.zeros((len(lens), H, N, P))}
    t0 = 0
    for i, n in enumerate(lens):
        S = [np.zeros((H, N, P)) if h0 is None else np.array(h0[i], np.float64)]
        for t in range(t0, t0 + n):
            S.append(np.exp(delta[t] * A)[:, None, None] * S[-1] + delta[t][:, None, None] * Bw[t][:, :, None] * x[t][:, None, :])
        R = np.zeros((H, N, P)) if dht is None else np.array(dht[i], np.float64)
        for t in range(t0 + n - 1, t0 - 1, -1):
            before, after = S[t - t0], S[t - t0 + 1]
            g["C"][t] = np.einsum("hnp,hp->hn", after, dy[t])
            R = R + Cw[t][:, :, None] * dy[t][:, None, :]
            reach = np.einsum("hnp,hn->hp", R, Bw[t])
            g["x"][t] = delta[t][:, None] * reach
            g["B"][t] = delta[t][:, None] * np.einsum("hnp,hp->hn", R, x[t])
            decay = np.exp(delta[t] * A)
            dg = decay * np.einsum("hnp,hnp->h", R, before)
            g["delta"][t] = A * dg + np.einsum("hp,hp->h", reach, x[t])
            g["A"] += delta[t] * dg
            R = decay[:, None, None] * R
        g["h0"][i] = R
        t0 += n
    if D is not None:
        g["x"] += np.asarray(D, np.float64)[:, None] * dy
    g["B"], g["C"] = (g[k].reshape(T, G, H // G, N).sum(2) for k in "BC")
    return g


def conv_grads(x, weight, bias, activation, dy, lens, past=None):
    """Gradients (dx, dweight, dbias) of the causal short convolution: x [T, D], weight [D, W], sequences of `lens` tokens,
    past [sequences, D, W] the inputs before each."""
    x, weight, dy = (np.asarray(t, np.float64) for t in (x, weight, dy))
    D, W = weight.shape
    dx, dw, db = np.zeros_like(x), np.zeros_like(weight), np.zeros(D)
    t0 = 0
    for i, n in enumerate(lens):
        ext = np.concatenate([np.zeros((W, D)) if past is None else np.asarray(past[i], np.float64).T, x[t0:t0 + n]])
        dext = np.zeros_like(ext)
        for t in range(n):
            window = ext[t + 1:t + 1 + W]
            pre = (window * weight.T).sum(0) + (0.0 if bias is None else np.asarray(bias, np.float64))
            s = sigmoid(pre)
            d = dy[t0 + t] * (s * (1 + pre * (1 - s)) if activation else 1.0)
            dw += (d * window).T
            db += d
            dext[t + 1:t + 1 + W] += d * weight.T
        dx[t0:t0 + n] = dext[W:]
        t0 += n
    return dx, dw, db


def residual_norm(x, residual, weight=None, post_weight=None, gate=None, act=None, scale=None, eps=1e-5, dy=None, dres=None):
    """(y, r) of r = residual + scale act(gate) a, y = rmsnorm(r) weight with a = x or rmsnorm(x) post_weight; with dy and dres
    also a dict of gradients. x [..., D]; the gate broadcasts against x and its gradient is summed accordingly."""
    f = lambda t: None if t is None else np.asarray(t, np.float64)  # noqa: E731
    x, residual, weight, post_weight, gate, scale = map(f, (x, residual, weight, post_weight, gate, scale))
    D = x.shape[-1]
    one = np.ones(D)
    i1 = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    a = x if post_weight is None else x * i1 * post_weight
    if gate is None:
        v, slope = 1.0, 0.0
    else:
        s = sigmoid(gate)
        v, slope = {None: (gate, np.ones_like(gate)), "sigmoid": (s, s * (1 - s)), "silu": (gate * s, s * (1 + gate * (1 - s)))}[act]
    sc = one if scale is None else scale
    w = one if weight is None else weight
    r = residual + sc * v * a
    i2 = 1.0 / np.sqrt((r * r).mean(-1, keepdims=True) + eps)
    y = r * i2 * w
    if dy is None:
        return y, r
    dy, dres = f(dy), f(dres)
    lead = tuple(range(x.ndim - 1))
    dr = dres + i2 * dy * w - r * i2 ** 3 * (dy * w * r).mean(-1, keepdims=True)
    da = dr * sc * v
    g = {"residual": dr, "weight": (dy * r * i2).sum(lead), "scale": (dr * v * a).sum(lead)}
    if gate is not None:
        dg = dr * sc * a * slope
        g["gate"] = dg if dg.shape == gate.shape else dg.sum(tuple(i for i in lead if gate.shape[i] == 1), keepdims=True)
    if post_weight is None:
        g["x"] = da
    else:
        dn = da * post_weight
        g["post_weight"] = (da * x * i1).sum(lead)
        g["x"] = i1 * dn - x * i1 ** 3 * (dn * x).mean(-1, keepdims=True)
    return y, r, g
