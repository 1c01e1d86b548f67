"""The state-space oracle against closed forms and central differences of its own forward (no GPU)."""
import numpy as np
import pytest

from oracle import state_space as os_


def _inputs(T, H, P, G, N, seed, n_seq=1):
    r = np.random.default_rng(seed)
    return dict(x=r.standard_normal((T, H, P)), delta=os_.softplus(r.standard_normal((T, H)) - 1), A=-r.uniform(0.5, 2, H),
                B=r.standard_normal((T, G, N)), C=r.standard_normal((T, G, N)), D=r.standard_normal(H),
                h0=r.standard_normal((n_seq, H, N, P)))


def test_scan_without_decay_is_a_causal_linear_attention():
    i = _inputs(9, 2, 3, 1, 4, 0)
    y, last = os_.scan(i["x"], i["delta"], np.zeros(2), i["B"], i["C"])
    for h in range(2):
        weights = np.tril(i["C"][:, 0] @ i["B"][:, 0].T) * i["delta"][:, h]
        assert np.allclose(y[:, h], weights @ i["x"][:, h])
        assert np.allclose(last[0, h], (i["B"][:, 0] * i["delta"][:, h:h + 1]).T @ i["x"][:, h])


def test_scan_of_one_pulse_decays_geometrically():
    T, A = 6, -0.7
    x, B = np.zeros((T, 1, 1)), np.ones((T, 1, 1))
    x[1] = 2.0
    y, _ = os_.scan(x, np.full((T, 1), 0.5), np.array([A]), B, B)
    assert np.allclose(y[:, 0, 0], [0] + [0.5 * 2.0 * np.exp(A * 0.5 * k) for k in range(T - 1)])


@pytest.mark.parametrize("name", ["x", "delta", "A", "B", "C", "D", "h0"])
def test_scan_gradients_against_differences(name):
    lens = [4, 0, 1, 3]
    i = _inputs(8, 4, 2, 2, 3, 1, n_seq=4)
    r = np.random.default_rng(2)
    dy, dht = r.standard_normal((8, 4, 2)), r.standard_normal((4, 4, 3, 2))

    def loss(**change):
        a = {**i, **change}
        y, last = os_.scan(a["x"], a["delta"], a["A"], a["B"], a["C"], a["D"], a["h0"], lens)
        return (y * dy).sum() + (last * dht).sum()

    g = os_.scan_grads(i["x"], i["delta"], i["A"], i["B"], i["C"], i["D"], i["h0"], lens, dy, dht)[name]
    along = r.standard_normal(i[name].shape)
    h = 1e-5
    diff = (loss(**{name: i[name] + h * along}) - loss(**{name: i[name] - h * along})) / (2 * h)
    assert abs(diff - (g * along).sum()) <= 1e-8 * (1 + np.abs(g * along).sum())


@pytest.mark.parametrize("which", [0, 1, 2])
def test_conv_gradients_against_differences(which):
    from oracle import layer_ops as ol

    r = np.random.default_rng(3)
    T, D, W = 7, 3, 4
    args = [r.standard_normal((T, D)), r.standard_normal((D, W)), r.standard_normal(D)]
    dy = r.standard_normal((T, D))
    lens = [2, 0, 5]
    g = os_.conv_grads(*args, "silu", dy, lens)[which]
    along, h = r.standard_normal(args[which].shape), 1e-5

    def loss(step):
        a = list(args)
        a[which] = a[which] + step * along
        return (ol.causal_conv1d(a[0][None], a[1], a[2], None, "silu", [0, 2, 2, 7])[0] * dy).sum()

    diff = (loss(h) - loss(-h)) / (2 * h)
    assert abs(diff - (g * along).sum()) <= 1e-8 * (1 + np.abs(g * along).sum())


@pytest.mark.parametrize("name", ["x", "residual", "weight", "post_weight", "gate", "scale"])
@pytest.mark.parametrize("act,per_sequence", [(None, False), ("sigmoid", True), ("silu", False)])
def test_residual_norm_gradients_against_differences(name, act, per_sequence):
    r = np.random.default_rng(4)
    B, T, D = 2, 3, 8
    i = dict(x=r.standard_normal((B, T, D)), residual=r.standard_normal((B, T, D)), weight=r.standard_normal(D),
             post_weight=r.standard_normal(D), gate=r.standard_normal((B, 1 if per_sequence else T, D)), scale=r.standard_normal(D))
    dy, dres = r.standard_normal((B, T, D)), r.standard_normal((B, T, D))

    def loss(step):
        a = dict(i)
        a[name] = a[name] + step * along
        y, res = os_.residual_norm(**a, act=act)
        return (y * dy).sum() + (res * dres).sum()

    along, h = r.standard_normal(i[name].shape), 1e-5
    g = os_.residual_norm(**i, act=act, dy=dy, dres=dres)[2][name]
    diff = (loss(h) - loss(-h)) / (2 * h)
    assert abs(diff - (g * along).sum()) <= 1e-7 * (1 + np.abs(g * along).sum())
