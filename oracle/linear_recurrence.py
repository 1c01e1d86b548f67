"""CPU oracle for the gated linear recurrence (TEST INFRASTRUCTURE ONLY): the recurrence and its gradients token by token in float64
numpy, from their definitions (parity unpinned: the reference's mixers import their recurrences from packages it does not hold;
``tests/test_oracle_linear_recurrence.py`` pins this one against closed forms and differences)."""
import numpy as np


def sigmoid(x):
    return 0.5 * (1.0 + np.tanh(0.5 * np.asarray(x, np.float64)))


def act(name, z):
    """(value, slope) of the output gate; name None: the gate itself."""
    s = sigmoid(z)
    return {None: (z, np.ones_like(z)), "sigmoid": (s, s * (1 - s)), "silu": (z * s, s * (1 + z * (1 - s)))}[name]


def pieces(x, r, A, i=None, normalize=True):
    """(sigmoid(r), log a, a, sigmoid(i), m) of every token."""
    sr = sigmoid(r)
    la = np.asarray(A, np.float64) * sr
    si = np.ones_like(sr) if i is None else sigmoid(i)
    m = np.sqrt(-np.expm1(2 * la)) if normalize else np.ones_like(sr)
    return sr, la, np.exp(la), si, m


def run(a, u, h0, lens):
    """h_t = a_t h_{t-1} + u_t for sequences of `lens` tokens: (all h [T, D], the last of each sequence)."""
    h, last, t = np.zeros_like(u), np.zeros((len(lens), u.shape[1])), 0
    for k, n in enumerate(lens):
        cur = np.zeros(u.shape[1]) if h0 is None else np.array(h0[k], np.float64)
        for _ in range(n):
            cur = a[t] * cur + u[t]
            h[t] = cur
            t += 1
        last[k] = cur
    return h, last


def run_back(a, d, dlast, lens):
    """G_t = d_t + a_{t+1} G_{t+1}, the last token's with dlast: (all G, the gradients of the states before the sequences)."""
    G, first, t0 = np.zeros_like(d), np.zeros((len(lens), d.shape[1])), 0
    for k, n in enumerate(lens):
        c = np.zeros(d.shape[1]) if dlast is None else np.array(dlast[k], np.float64)
        for t in range(t0 + n - 1, t0 - 1, -1):
            G[t] = d[t] + c
            c = a[t] * G[t]
        first[k] = c
        t0 += n
    return G, first


def before(h, h0, lens):
    """h_{t-1} of every token."""
    out, t = np.zeros_like(h), 0
    for k, n in enumerate(lens):
        if n:
            out[t] = 0 if h0 is None else h0[k]
            out[t + 1:t + n] = h[t:t + n - 1]
        t += n
    return out


def scan(x, r, A, i=None, z=None, activation=None, normalize=True, h0=None, lens=None):
    """x, r, i, z [T, D], A [D], h0 [sequences, D] -> (y [T, D], last states [sequences, D])."""
    x = np.asarray(x, np.float64)
    lens = [x.shape[0]] if lens is None else lens
    _, _, a, si, m = pieces(x, r, A, i, normalize)
    h, last = run(a, m * si * x, h0, lens)
    return h if z is None else h * act(activation, np.asarray(z, np.float64))[0], last


def scan_grads(x, r, A, i, z, activation, normalize, h0, lens, dy, dlast=None):
    """Gradients of sum(y dy) + sum(last dlast): a dict over x, r, A, i, z, h0."""
    x, dy = np.asarray(x, np.float64), np.asarray(dy, np.float64)
    sr, la, a, si, m = pieces(x, r, A, i, normalize)
    h, _ = run(a, m * si * x, h0, lens)
    value, slope = (np.ones_like(x), np.zeros_like(x)) if z is None else act(activation, np.asarray(z, np.float64))
    G, first = run_back(a, dy * value, dlast, lens)
    dla = G * a * before(h, h0, lens)
    if normalize:
        dla = dla - G * si * x * a * a / m
    return {"x": G * m * si, "r": dla * la * (1 - sr), "A": (dla * sr).sum(0), "i": G * m * x * si * (1 - si), "z": dy * h * slope,
            "h0": first}
