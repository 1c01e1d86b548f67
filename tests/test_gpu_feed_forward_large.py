"""The kernels of the feed-forward block that many rows and wide blocks run: 8 waves a workgroup (D <= 128, more than 32 768 rows), hidden
values as one operand in the weights' gradients (more than 4 096 rows), tiles of 128 rows and placement by columns (D > 128, fp32).

In whole numbers every step is exact: no activation, x and dy of -1, 0, 1, four of -1, 1 in each row of w_gate and w_up and each column of
w_down, so G, U and dS are within 4, hidden values and their gradients within 16 and sums of up to 60 000 of them within 2^24. What
comes out is the exact sum, rounded once: a row, a column or a hidden value lost, doubled or misplaced shows in its bits."""
import pytest
import torch

from lampa_amd.feed_forward import gated_feed_forward
from test_gpu_feed_forward import _check

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _sparse(rows, cols, gen):
    """[rows, cols] with up to four of -1, 1 in a row."""
    w = torch.zeros(rows, cols, dtype=torch.float64, device="cuda")
    at = torch.randint(0, cols, (rows, 4), device="cuda", generator=gen)
    return w.scatter_(1, at, (torch.randint(0, 2, (rows, 4), device="cuda", generator=gen) * 2 - 1).double())


SIZES = [  # rows, D, F, types
    (32801, 128, 136, (BF16, FP16)),   # 8 waves, tails of rows and hidden columns
    (33000, 40, 520, (BF16,)),
    (51237, 96, 72, (FP16,)),
    (60000, 64, 264, (BF16,)),
    (32768, 128, 40, (BF16,)),         # the last rows of 4 waves
    (4096, 96, 264, (BF16,)),          # the last rows as two parts
    (4097, 96, 264, (BF16, FP16)),
    (4129, 16, 1000, (BF16,)),
    (4100, 264, 1032, (BF16, FP16, FP32)),  # tiles of 128 rows: hidden, gradients
    (8201, 136, 520, (BF16, FP32)),
    (8201, 1032, 72, (BF16, FP32)),    # and the last products
    (1300, 520, 1096, (BF16, FP16)),   # by columns, tiles of 64 rows
    (2100, 520, 1096, (BF16, FP32)),   # by columns, 128
    (40000, 16, 72, (FP32,)),
]


@pytest.mark.parametrize("rows,D,F,dtype", [(*s[:3], t) for s in SIZES for t in s[3]], ids=lambda v: str(v).replace("torch.", ""))
def test_whole_numbers_are_exact(rows, D, F, dtype):
    gen = torch.Generator(device="cuda").manual_seed(rows + D)
    digits = lambda: torch.randint(-1, 2, (rows, D), device="cuda", generator=gen).double()  # noqa: E731
    x, dy = digits(), digits()
    wg, wu, wd = _sparse(F, D, gen), _sparse(F, D, gen), _sparse(F, D, gen).t().contiguous()
    G, U, dS = x @ wg.t(), x @ wu.t(), dy @ wd
    dG, dU = dS * U, dS * G
    want = [(G * U) @ wd.t(), dG @ wg + dU @ wu, dG.t() @ x, dU.t() @ x, dy.t() @ (G * U)]
    leaves = [t.to(dtype).requires_grad_(True) for t in (x, wg, wu, wd)]
    y = gated_feed_forward(*leaves, activation=None)
    got = [y.detach(), *torch.autograd.grad(y, leaves, dy.to(dtype))]
    for name, g, w in zip(("y", "dx", "dw_gate", "dw_up", "dw_down"), got, want):
        assert torch.equal(g, w.to(dtype)), name


@pytest.mark.parametrize("size,dtype", [((32801, 128, 136), BF16), ((4129, 96, 264), FP16), ((4100, 264, 1032), BF16),
                                        ((4100, 264, 1032), FP32)], ids=lambda v: str(v).replace("torch.", ""))
def test_forward_and_gradients(size, dtype):
    _check(*size, dtype, "silu")
