"""Calls of the state-space operators, the convolution and the norms that a program may make beside the ordinary ones: rubbish behind
the last sequence, gradients through a single token, forward-mode gradients, slices of long tensors, parameters without gradients."""
import pytest
import torch

from lampa_amd import layer_ops as lo

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
