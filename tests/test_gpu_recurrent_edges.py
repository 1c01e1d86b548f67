"""The gated recurrence at its edges: results that are zero by definition."""
import pytest
import torch

from test_gpu_linear_recurrence import _bounds, _call, _gpu, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("lens", [[1], [1, 1, 0, 1], 3], ids=str)
def test_decays_without_a_state_before_them_have_no_gradient(lens, dtype):
    """Sequences of one token on no state, the input as it is: h = sigmoid(i) x holds no decay, so the gradients of A and of the decay
    gate are zero, not small."""
    n = lens if isinstance(lens, int) else len(lens)
    shape = (lens, 1) if isinstance(lens, int) else (1, sum(lens))
    t = _inputs(shape, 96, dtype, 40, n, state=False)
    leaves = _gpu(t, grad=True)
    y, last = _call(leaves, "silu", False, None if isinstance(lens, int) else _bounds(lens).cuda())
    names = ["A", "r", "x", "i", "z"]
    grads = torch.autograd.grad([y, last], [leaves[k] for k in names], [torch.ones_like(y), torch.ones_like(last)])
    assert not grads[0].any() and not grads[1].any()
    assert all(g.any() for g in grads[2:])
