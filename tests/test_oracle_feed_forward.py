"""The feed-forward oracle against a literal loop and central differences (no GPU)."""
import numpy as np
import pytest

from oracle import feed_forward as of


def _inputs():
    g = np.random.default_rng(0)
    return [g.standard_normal(s) for s in ((5, 4), (6, 4), (6, 4), (4, 6), (5, 4))]


def test_against_a_loop():
    x, wg, wu, wd, _ = _inputs()
    want = np.zeros_like(x)
    for t in range(5):
        for f in range(6):
            g = sum(x[t, d] * wg[f, d] for d in range(4))
            u = sum(x[t, d] * wu[f, d] for d in range(4))
            for d in range(4):
                want[t, d] += g / (1 + np.exp(-g)) * u * wd[d, f]
    assert np.allclose(of.forward(x, wg, wu, wd), want)


@pytest.mark.parametrize("activation", [None, "silu", "sigmoid"])
def test_gradients_against_differences(activation):
    *args, dy = _inputs()
    got = of.grads(*args, dy, activation)
    for k in range(4):
        num = np.zeros_like(args[k])
        for at in np.ndindex(num.shape):
            ends = []
            for step in (1e-6, -1e-6):
                moved = [a.copy() for a in args]
                moved[k][at] += step
                ends.append((of.forward(*moved, activation) * dy).sum())
            num[at] = (ends[0] - ends[1]) / 2e-6
        assert np.allclose(got[k], num, rtol=1e-6, atol=1e-7), k
