"""Sequences of more than 256 tiles, where a tile starts from the state that a block of 256 tiles left, forward and gradients."""
import numpy as np
import pytest
import torch

from lampa_amd.linear_recurrence import gated_recurrence
from test_gpu_linear_recurrence import _bounds, _call, _close, _expected, _gpu, _inputs

pytestmark = pytest.mark.gpu

# sequences' tokens, D: tiles of 64 tokens for D = 128 and 256, of 256 for 24; blocks from 16 384 (65 536) tokens on
SIZES = [([40000], 256), ([777, 0, 50001, 1, 70, 17000], 128), ([140007], 24)]


@pytest.mark.parametrize("lens,D", SIZES, ids=lambda v: str(v))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_sums_of_whole_numbers_are_exact(lens, D, dtype):
    """Decays of 1 (A = 0) on whole numbers: the states are their sums and the gradients those from behind, exact in fp32 (within
    2^24) and rounded once in what is returned."""
    T, n = sum(lens), len(lens)
    g = torch.Generator().manual_seed(50)
    whole = lambda *s: torch.randint(-2, 3, s, generator=g).double()  # noqa: E731
    x, dy, h0, dht = whole(1, T, D), whole(1, T, D), whole(n, D), whole(n, D)
    r = torch.full((1, T, D), 200.0)  # sigmoid 1
    ends = np.cumsum(lens)
    h, G, last, first = [], [], [], []
    for k, (e, length) in enumerate(zip(ends, lens)):
        h.append(h0[k] + x[0, e - length:e].cumsum(0))
        G.append(dht[k] + dy[0, e - length:e].flip(0).cumsum(0).flip(0))
        last.append(h[k][-1] if length else h0[k])
        first.append(G[k][0] if length else dht[k])
    h, G = torch.cat(h), torch.cat(G)
    leaves = [t.to(dtype).cuda().requires_grad_(True) for t in (x, r)] + [torch.zeros(D, device="cuda", requires_grad=True),
                                                                           h0.float().cuda().requires_grad_(True)]
    y, ht = gated_recurrence(leaves[0], leaves[1], leaves[2], normalize=False, initial_state=leaves[3], output_final_state=True,
                             cu_seqlens=_bounds(lens).cuda())
    assert torch.equal(y[0].cpu(), h.to(dtype)) and torch.equal(ht.cpu().double(), torch.stack(last))
    dx, dr, dA, dh0 = torch.autograd.grad([y, ht], leaves, [dy.to(dtype).cuda(), dht.float().cuda()])
    assert torch.equal(dx[0].cpu(), G.to(dtype)) and torch.equal(dh0.cpu().double(), torch.stack(first)) and not dr.any()
    # the sum of h_{t-1} G_t, each product and each of at most T additions off by half a step of what is added up
    prev = torch.cat([torch.cat([h0[k][None], h[e - m:e - 1]]) for k, (e, m) in enumerate(zip(ends, lens)) if m])
    terms = prev * G
    assert bool(((dA.cpu().double() - terms.sum(0)).abs() <= (T + 1) * 2.0 ** -24 * terms.abs().sum(0)).all())


@pytest.mark.parametrize("lens,D", SIZES[1:], ids=lambda v: str(v))
def test_long_memories(lens, D):
    """Decays that keep a state over tens of thousands of tokens, everything positive, so that nothing cancels: a token's 32 half-steps
    over such a memory are a few percent of a state at most, and a state that comes in wrong is a large part of it."""
    t = _inputs((1, sum(lens)), D, torch.float32, 51, len(lens), z=False)
    t["x"], t["h0"] = t["x"].abs(), 50 * t["h0"].abs()
    t["A"] = -10.0 ** (-5 + torch.rand(D, generator=torch.Generator().manual_seed(52)))
    g = torch.Generator().manual_seed(53)
    dy, dht = torch.rand(1, sum(lens), D, generator=g), 50 * torch.rand(len(lens), D, generator=g)
    want = _expected(t, lens, None, True, dy, dht)
    for k in ("y", "last", "x", "h0"):
        assert np.max(want[k][1] / np.maximum(np.abs(want[k][0]), 1e-30)) < 0.25, k  # the bounds say something
    leaves = _gpu(t, grad=True)
    y, last = _call(leaves, None, True, _bounds(lens).cuda())
    _close("y", y, *want["y"])
    _close("last", last, *want["last"])
    names = ["x", "r", "A", "i", "h0"]
    for k, v in zip(names, torch.autograd.grad([y, last], [leaves[k] for k in names], [dy.cuda(), dht.cuda()])):
        _close(k, v, *want[k])
