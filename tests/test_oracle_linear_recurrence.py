"""The gated recurrence's oracle against closed forms and central differences of its own forward (no GPU)."""
import numpy as np
import pytest

from oracle import linear_recurrence as ol

LENS = [4, 0, 1, 5]


def _inputs(seed):
    g = np.random.default_rng(seed)
    T, D = sum(LENS), 3
    return dict(x=g.standard_normal((T, D)), r=g.standard_normal((T, D)), A=-g.uniform(0.05, 1.5, D), i=g.standard_normal((T, D)),
                z=g.standard_normal((T, D)), h0=g.standard_normal((len(LENS), D)))


def test_one_pulse_decays_geometrically():
    T, A = 6, -0.7
    x = np.zeros((T, 1))
    x[1] = 2.0
    y, last = ol.scan(x, np.zeros((T, 1)), [A], normalize=False)
    assert np.allclose(y[:, 0], [0] + [2.0 * np.exp(0.5 * A * k) for k in range(T - 1)])
    assert np.allclose(last[0], y[-1])


def test_normalised_recurrence_keeps_the_variance():
    """With independent inputs of variance 1 and a constant decay the state's variance stays 1: a^2 + m^2 = 1."""
    _, la, a, _, m = ol.pieces(np.ones((2, 4)), np.zeros((2, 4)), [-1e-3, -0.1, -1.0, -30.0])
    assert np.allclose(a * a + m * m, 1.0) and np.allclose(la[0], [-5e-4, -0.05, -0.5, -15.0])


def test_empty_and_single_sequences_hand_the_state_on():
    i = _inputs(0)
    _, last = ol.scan(**i, lens=LENS)
    assert np.array_equal(last[1], i["h0"][1])
    alone = {k: v[4:5] if k in "xriz" else v for k, v in i.items()}
    assert np.allclose(ol.scan(**{**alone, "h0": i["h0"][2:3]})[1][0], last[2])


@pytest.mark.parametrize("activation", [None, "silu", "sigmoid"])
@pytest.mark.parametrize("normalize", [True, False])
def test_gradients_against_differences(activation, normalize):
    i = _inputs(1)
    g = np.random.default_rng(2)
    dy, dlast = g.standard_normal(i["x"].shape), g.standard_normal(i["h0"].shape)

    def loss(**change):
        y, last = ol.scan(**{**i, **change}, activation=activation, normalize=normalize, lens=LENS)
        return (y * dy).sum() + (last * dlast).sum()

    grads = ol.scan_grads(i["x"], i["r"], i["A"], i["i"], i["z"], activation, normalize, i["h0"], LENS, dy, dlast)
    for name, value in i.items():
        step = 1e-6
        num = np.zeros_like(value)
        for at in np.ndindex(value.shape):
            up, down = value.copy(), value.copy()
            up[at] += step
            down[at] -= step
            num[at] = (loss(**{name: up}) - loss(**{name: down})) / (2 * step)
        assert np.allclose(grads[name], num, rtol=1e-6, atol=1e-7), name
