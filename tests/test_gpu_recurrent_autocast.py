"""The gated recurrent block with float32 parameters under autocast.

Tolerance as of the block in 16 bits: to the dozen roundings of 2^-9 rms between a layer's input and output come those of the weights, one
for each of its six products; 0.05 of the norm bounds two pairs of layers (18 x 2 x 2^-9 = 0.07 if all pointed one way, 0.012
as they fall)."""
import pytest
import torch

from lampa_amd.block import GatedFeedForward
from lampa_amd.feed_forward import gated_feed_forward
from test_gpu_recurrent_block import _block, _plain, _rel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_feed_forward_in_autocasts_type(dtype):
    torch.manual_seed(0)
    layer = GatedFeedForward(64, intermediate_size=160).cuda()
    for given in (torch.float32, dtype):
        x = torch.randn(3, 7, 64, device="cuda").to(given).requires_grad_(True)
        with torch.autocast("cuda", dtype=dtype):
            y = layer(x)
        weights = [w.detach().to(dtype).requires_grad_(True) for w in layer.parameters()]
        cast = x.detach().to(dtype).requires_grad_(True)
        want = gated_feed_forward(cast, *weights)
        assert y.dtype == dtype and torch.equal(y, want)
        got = torch.autograd.grad(y.float().sum(), [x, *layer.parameters()])
        ref = torch.autograd.grad(want.float().sum(), [cast, *weights])
        for g, r, leaf in zip(got, ref, [x, *layer.parameters()]):
            assert g.dtype == leaf.dtype and torch.equal(g, r.to(leaf.dtype))
    with torch.autocast("cuda", enabled=False), pytest.raises(TypeError):
        layer(torch.randn(3, 64, device="cuda", dtype=dtype))
    with torch.autocast("cuda", dtype=dtype), pytest.raises(TypeError):
        layer(torch.randn(3, 64, device="cuda", dtype=torch.float64))


def test_block_trains_prefills_and_steps():
    lens = [70, 0, 1, 30]
    block = _block()
    x = torch.randn(1, sum(lens), 64, generator=torch.Generator().manual_seed(1))
    dy = torch.randn(1, sum(lens), 64, generator=torch.Generator().manual_seed(2))
    want, p, wx = _plain(block, x, lens)
    grads = torch.autograd.grad((want * dy.double()).sum(), [wx, *p.values()])
    block = block.cuda()
    leaf = x.cuda().requires_grad_(True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got, _ = block(leaf, torch.tensor([0, 70, 70, 71, 101]).cuda())
        loss = (got.float() * dy.cuda()).sum()
    assert _rel(got, want.detach()) <= 0.05
    loss.backward()
    assert _rel(leaf.grad, grads[0]) <= 0.05
    for (name, v), g in zip(block.named_parameters(), grads[1:]):
        if "A_log" not in name:  # a sum of both signs over all tokens
            assert v.grad.dtype == torch.float32 and _rel(v.grad, g) <= 0.05, name
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        first, caches = block(leaf[:, :60], output_caches=True)
        parts = [first]
        for t in range(60, 70):
            parts.append(block.step(leaf[:, t], caches).unsqueeze(1))
    assert _rel(torch.cat(parts, 1), want[:, :70].detach()) <= 0.05
