"""More workgroups than one dimension of a launch takes (2^32 threads): very many short sequences, states past 2^32 elements."""
import pytest
import torch

from lampa_amd.linear_recurrence import gated_recurrence, gated_recurrence_step

pytestmark = pytest.mark.gpu


def test_very_many_sequences():
    """2^24 sequences of a token and a few more, 256 threads each forward and 512 back: every one as in a small call."""
    n, D = (1 << 24) + 5, 8
    g = torch.Generator(device="cuda").manual_seed(1)
    x, r, dy = (torch.randn(n, 1, D, device="cuda", generator=g).bfloat16() for _ in range(3))
    A = -torch.rand(D, device="cuda", generator=g)
    h0 = torch.randn(n, D, device="cuda", generator=g)

    def call(part):
        leaves = [t[part].detach().requires_grad_(True) for t in (x, r, h0)]
        y, last = gated_recurrence(leaves[0], leaves[1], A, initial_state=leaves[2], output_final_state=True)
        return (y.detach(), last.detach(), *torch.autograd.grad([y, last], leaves, [dy[part], h0[part]]))

    whole = call(slice(None))
    for at in (0, (1 << 22) - 50, (1 << 23) - 50, n - 100):
        part = slice(at, at + 100)
        for a, b in zip(whole, call(part)):
            assert torch.equal(a[part], b)
    # all of them: h = a h0 + m x. Half a step of bf16 for y; 32 half-steps of fp32 of what is added up
    a = torch.exp(A * torch.sigmoid(r[:, 0].float()))
    m = torch.sqrt(-torch.expm1(2 * A * torch.sigmoid(r[:, 0].float())))
    h, mag = a * h0 + m * x[:, 0].float(), a * h0.abs() + m * x[:, 0].float().abs()
    assert bool(((whole[1] - h).abs() <= 64 * 2.0 ** -24 * mag).all())
    assert bool(((whole[0][:, 0].float() - h).abs() <= 2.0 ** -8 * h.abs() + 80 * 2.0 ** -24 * mag).all())


def test_steps_of_very_large_states():
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GB")
    n, D = (1 << 22) + 3, 1024
    x, r = (torch.empty(n, D, device="cuda", dtype=torch.bfloat16).normal_() for _ in range(2))
    state = torch.empty(n, D, device="cuda").normal_()
    A = -torch.rand(D, device="cuda")
    parts = [slice(at, at + 40) for at in (0, (1 << 21) - 20, n - 40)]
    small = []
    for part in parts:
        own = state[part].clone()
        small.append((gated_recurrence_step(x[part], r[part], A, own), own))
    y = gated_recurrence_step(x, r, A, state)
    for part, (yp, sp) in zip(parts, small):
        assert torch.equal(y[part], yp) and torch.equal(state[part], sp)
