"""gated_feed_forward over few rows of blocks wider than 128, 16-bit types: the rounding of hidden values does not show in what it returns."""
import pytest
import torch

from lampa_amd.feed_forward import gated_feed_forward

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("rows,D,F", [(1, 136, 432), (1, 136, 32), (4, 264, 40), (2, 1024, 1400), (21, 1032, 72), (33, 520, 1096),
                                      (64, 200, 264)])
def test_few_rows(rows, D, F, dtype):
    torch.manual_seed(rows + D + F)
    x, wg, wu, wd, dy = (torch.randn(s).to(dtype) for s in ((rows, D), (F, D), (F, D), (D, F), (rows, D)))
    wg, wu, wd = wg * D ** -0.5, wu * D ** -0.5, wd * F ** -0.5
    leaves = [t.cuda().requires_grad_() for t in (x, wg, wu, wd)]
    y = gated_feed_forward(*leaves, activation=None)
    got = [y.detach(), *torch.autograd.grad(y, leaves, dy.cuda())]
    X, G_, U_, W, Y = (t.double() for t in (x, wg, wu, wd, dy))

    def products(X, G_, U_, W, Y):
        G, U, S = X @ G_.t(), X @ U_.t(), Y @ W
        return (G * U) @ W.t(), (S * U) @ G_ + (S * G) @ U_, (S * U).t() @ X, (S * G).t() @ X, Y.t() @ (G * U)

    exact = products(X, G_, U_, W, Y)
    terms = products(*(t.abs() for t in (X, G_, U_, W, Y)))
    # what one unit in every hidden value (or in every one of their gradients) comes to
    plain = (W.abs().sum(1).expand(rows, D), (G_.abs().sum(0) + U_.abs().sum(0)).expand(rows, D), X.abs().sum(0).expand(F, D),
             X.abs().sum(0).expand(F, D), Y.abs().sum(0)[:, None].expand(D, F))
    half = torch.finfo(dtype).eps / 2
    # The output's rounding, half a step. Before it, of the terms' absolute sum: a hidden value's low part is off by half a step of half a
    # step; sums of D products in float32, twice in each value, and 2 K products (two parts; K = F for y, 2 F for dx, the rows for the
    # weights), each off by 2^-24 at most, twice that for a sum in the matrix cores' own order and rounding. fp16: a low part under its
    # normal range is off by 2^-25, an output by as much.
    for name, g, e, t, p, K in zip(("y", "dx", "dw_gate", "dw_up", "dw_down"), got, exact, terms, plain, (F, 2 * F, rows, rows, rows)):
        inner = t * (half * half + (2 * D + 2 * K + 8) * 2.0 ** -23) + (p * 2.0 ** -25 if dtype == torch.float16 else 0.0)
        limit = e.abs() * half + inner * (1 + half) + (2.0 ** -25 if dtype == torch.float16 else 0.0)
        worst = float(((g.double().cpu() - e).abs() / limit).max())
        assert worst <= 1, (name, worst)
