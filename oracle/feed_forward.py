"""CPU oracle for the gated feed-forward block (TEST INFRASTRUCTURE ONLY): ``GatedMLP`` of the reference
(``models/hattention/modeling_gated_deltaproduct.py:310-324``) and its gradients by the product rule, in float64 numpy."""
import numpy as np

from .linear_recurrence import act


def forward(x, wg, wu, wd, activation="silu"):
    x, wg, wu, wd = (np.asarray(t, np.float64) for t in (x, wg, wu, wd))
    return (act(activation, x @ wg.T)[0] * (x @ wu.T)) @ wd.T


def grads(x, wg, wu, wd, dy, activation="silu"):
    """Gradients of sum(y dy): (x, w_gate, w_up, w_down)."""
    x, wg, wu, wd, dy = (np.asarray(t, np.float64) for t in (x, wg, wu, wd, dy))
    value, slope = act(activation, x @ wg.T)
    up, ds = x @ wu.T, dy @ wd
    dg, du = ds * up * slope, ds * value
    return dg @ wg + du @ wu, dg.T @ x, du.T @ x, dy.T @ (value * up)
