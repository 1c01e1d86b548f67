"""Weights' gradients of gated_feed_forward over few rows: the rounding of hidden values does not show in them."""
import pytest
import torch

from lampa_amd.feed_forward import gated_feed_forward

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("rows,D,F", [(1, 80, 432), (1, 128, 512), (21, 8, 40), (33, 96, 136)])
def test_weight_gradients_of_few_rows(rows, D, F, dtype):
    torch.manual_seed(rows + D)
    x, wg, wu, wd, dy = (torch.randn(s).to(dtype) for s in ((rows, D), (F, D), (F, D), (D, F), (rows, D)))
    wg, wu, wd = wg * D ** -0.5, wu * D ** -0.5, wd * F ** -0.5
    leaves = [t.cuda().requires_grad_() for t in (wg, wu, wd)]
    got = torch.autograd.grad(gated_feed_forward(x.cuda(), *leaves, activation=None), leaves, dy.cuda())
    X, G_, U_, W, Y = (t.double() for t in (x, wg, wu, wd, dy))
    G, U, S = X @ G_.t(), X @ U_.t(), Y @ W
    Ga, Ua, Sa = X.abs() @ G_.abs().t(), X.abs() @ U_.abs().t(), Y.abs() @ W.abs()
    exact = ((S * U).t() @ X, (S * G).t() @ X, Y.t() @ (G * U))
    terms = ((Sa * Ua).t() @ X.abs(), (Sa * Ga).t() @ X.abs(), Y.abs().t() @ (Ga * Ua))
    plain = (X.abs().sum(0).expand(F, D), X.abs().sum(0).expand(F, D), Y.abs().sum(0)[:, None].expand(D, F))
    half = torch.finfo(dtype).eps / 2
    # The output's rounding, half a step. Before it, of the terms' absolute sum: a hidden value's low part is off by half a step of half a
    # step; sums of D products in float32, twice in each value, and 2 x rows products (two parts), each off by 2^-24 at most, twice that for
    # a sum in the matrix cores' own order and rounding. fp16: a low part under its normal range is off by 2^-25, an output by as much.
    for g, e, t, p in zip(got, exact, terms, plain):
        inner = t * (half * half + (2 * D + 2 * rows + 8) * 2.0 ** -23) + (p * 2.0 ** -25 if dtype == torch.float16 else 0.0)
        limit = e.abs() * half + inner * (1 + half) + (2.0 ** -25 if dtype == torch.float16 else 0.0)
        assert bool(((g.double().cpu() - e).abs() <= limit).all()), float(((g.double().cpu() - e).abs() / limit).max())
