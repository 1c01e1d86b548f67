"""Calls of the gated recurrence and the feed-forward block that their documentation allows and no other test makes: growth, no tokens,
shared and broadcast operands, tensors past 2^31 elements, operands changed between the passes, rounds of waits under load."""
import numpy as np
import pytest
import torch

from lampa_amd.feed_forward import gated_feed_forward
from lampa_amd.linear_recurrence import gated_recurrence, gated_recurrence_step
from oracle import linear_recurrence as ol

pytestmark = pytest.mark.gpu


def test_growth_without_the_normalising_factor():
    """A above 0: the recurrence grows as it is written. Per token a decay is off by its exponent's roundings (10 half-steps of |log a|
    below 1) and 4 more: 14 half-steps of 2^-24 of all that is positive here, over at most 100 tokens; exp(sum) in place of the
    product adds the sum's own 100 half-steps of its size, 30."""
    T, D = 100, 12
    g = torch.Generator().manual_seed(1)
    x, r, A = torch.rand(1, T, D, generator=g), torch.randn(1, T, D, generator=g), 0.6 * torch.rand(D, generator=g)
    want, last = ol.scan(x[0].numpy(), r[0].numpy(), A.numpy(), normalize=False)
    y, ht = gated_recurrence(x.cuda(), r.cuda(), A.cuda(), normalize=False, output_final_state=True)
    for got, ref in ((y[0], want), (ht, last)):
        assert np.max(np.abs(got.double().cpu().numpy() - ref) / ref) <= (14 * T + 100 * 30) * 2.0 ** -24
    assert gated_recurrence(x.cuda(), r.cuda(), A.cuda())[0].isnan().all()  # sqrt(1 - a^2) of a above 1


@pytest.mark.parametrize("shape", [(2, 0), (3, 1)])
def test_no_tokens_and_one(shape):
    D = 48
    x = torch.randn(*shape, D, device="cuda", requires_grad=True)
    A = torch.full((D,), -0.1, device="cuda", requires_grad=True)
    h0 = torch.randn(shape[0], D, device="cuda", requires_grad=True)
    y, last = gated_recurrence(x, x, A, initial_state=h0, output_final_state=True)
    d = torch.randn_like(last)
    dx, dA, dh0 = torch.autograd.grad([y, last], [x, A, h0], [torch.ones_like(y), d])
    assert dx.shape == x.shape and dA.isfinite().all()
    if shape[1] == 0:
        assert torch.equal(last, h0) and torch.equal(dh0, d) and not dA.any()
    else:
        a = torch.exp(A * torch.sigmoid(x[:, 0].detach()))
        assert torch.allclose(dh0, a * (1 + d), rtol=1e-5, atol=1e-6)


def test_shared_and_broadcast_operands():
    """One tensor as x, both gates and the output gate; A and the state spread from one value: gradients are summed over the uses."""
    T, D = 90, 32
    base = torch.randn(1, T, D, generator=torch.Generator().manual_seed(2)).double()

    def run(dtype, device):
        x = base.to(device=device, dtype=dtype).requires_grad_(True)
        a = torch.tensor(-0.3, device=device, dtype=dtype, requires_grad=True)
        h = torch.tensor(0.7, device=device, dtype=dtype, requires_grad=True)
        if device == "cuda":
            y, _ = gated_recurrence(x, x, a.expand(D), input_gate=x, gate=x, gate_activation="silu", initial_state=h.expand(1, D))
        else:
            la = a * torch.sigmoid(x[0])
            m, state, ys = torch.sqrt(-torch.expm1(2 * la)), h.expand(D), []
            for t in range(T):
                state = torch.exp(la[t]) * state + m[t] * torch.sigmoid(x[0, t]) * x[0, t]
                ys.append(state * torch.nn.functional.silu(x[0, t]))
            y = torch.stack(ys)[None]
        return torch.autograd.grad(y.sum(), [x, a, h])

    for got, want in zip(run(torch.float32, "cuda"), run(torch.float64, "cpu")):
        # a few hundred half-steps of 2^-24 of sums of up to 2 880 terms of both signs
        assert (got.double().cpu() - want).norm() <= 2e-5 * want.norm() + 2e-4


def test_operands_changed_between_the_passes_are_noticed():
    x = torch.randn(1, 20, 16, device="cuda", requires_grad=True)
    r = torch.randn(1, 20, 16, device="cuda")
    A = torch.full((16,), -0.1, device="cuda")
    y, _ = gated_recurrence(x, r, A)
    r.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    state = torch.zeros(20, 16, device="cuda")
    w = [torch.randn(32, 16, device="cuda", requires_grad=True), torch.randn(32, 16, device="cuda", requires_grad=True),
         torch.randn(16, 32, device="cuda", requires_grad=True)]
    y = gated_feed_forward(state, *w)
    gated_recurrence_step(r[0], r[0], A, state)  # writes what the block has kept
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_tensors_past_32_bits():
    """More than 2^31 elements: the last tokens, from a state that the ones before them leave nothing of, as in a call of their own."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    T, D, tail = (1 << 21) + 200, 1024, 1000
    x = torch.empty(1, T, D, device="cuda", dtype=torch.bfloat16).normal_()
    r = torch.empty(1, T, D, device="cuda", dtype=torch.bfloat16).normal_()
    A = torch.full((D,), -20.0, device="cuda")
    y, last = gated_recurrence(x, r, A, output_final_state=True)
    part, last2 = gated_recurrence(x[:, -tail:], r[:, -tail:], A, output_final_state=True)
    # behind 200 tokens of decays of exp(-20 sigmoid) nothing is left of an earlier state; both are rounded once
    assert torch.allclose(y[:, -tail + 200:].float(), part[:, 200:].float(), rtol=2.0 ** -7, atol=1e-6)
    assert torch.allclose(last, last2, rtol=1e-5, atol=1e-6)
    del x, r, y, part
    rows, D, F = (1 << 22) + 77, 136, 520
    x = torch.empty(rows, D, device="cuda", dtype=torch.bfloat16).normal_()
    w = [torch.randn(s, device="cuda").bfloat16() / 12 for s in ((F, D), (F, D), (D, F))]
    y = gated_feed_forward(x, *w)
    ref = gated_feed_forward(x[-500:].clone(), *w)
    assert torch.allclose(y[-500:].float(), ref.float(), rtol=2.0 ** -6, atol=2e-2)
    assert (y[-500:] == ref).float().mean() > 0.9


def test_long_sequences_beside_short_ones():
    """Sequences of very different lengths handed out together, and another call under way on a second stream."""
    D, lens = 256, [9000, 1, 0, 4097, 64, 20000, 3, 2048]
    T = sum(lens)
    g = torch.Generator(device="cuda").manual_seed(3)
    x, r = (torch.randn(1, T, D, device="cuda", generator=g) for _ in range(2))
    A = -0.5 * torch.rand(D, device="cuda", generator=g)
    cu = torch.tensor([0] + list(np.cumsum(lens)), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    y, last = gated_recurrence(x, r, A, output_final_state=True, cu_seqlens=cu)
    with torch.cuda.stream(side):
        y2, last2 = gated_recurrence(x, r, A, output_final_state=True, cu_seqlens=cu)
    torch.cuda.synchronize()
    assert torch.equal(y, y2) and torch.equal(last, last2)
    at = 0
    for k, n in enumerate(lens):
        if n:
            alone, end = gated_recurrence(x[:, at:at + n], r[:, at:at + n], A, output_final_state=True)
            assert torch.equal(alone, y[:, at:at + n]) and torch.equal(end[0], last[k])
        at += n
