"""The gated recurrence and the gated feed-forward block together, as a layer and a block use them: training on packed sequences
against a float64 block of elementary torch operations, prompts continued by further prompts and by single tokens, captured calls.

Tolerances as in the state-space block's tests. fp32: the layers' products go through library GEMMs and the operators' own
(about K half-steps of fp32 in K-long sums, K <= 160): 2e-4 of a tensor's norm is more than a thousand half-steps for each of the
four mixers and feed-forward blocks. bf16: a dozen roundings of 2^-9 rms each lie between input and output of a layer, 0.05 of
the norm bounds two pairs of layers."""
import pytest
import torch
import torch.nn.functional as F

from lampa_amd.block import GatedFeedForward, GatedRecurrentBlock, GatedRecurrentLayer

pytestmark = pytest.mark.gpu


def _block(dtype=torch.float32, seed=0, **kw):
    torch.manual_seed(seed)
    return GatedRecurrentBlock(64, 2, intermediate_size=160, expand=1, **kw).to(dtype)


def _norm(v, w):
    return v * torch.rsqrt(v.pow(2).mean(-1, keepdim=True) + 1e-5) * w


def _plain(block, x, lens):
    """The block in float64 on the CPU, token by token, from elementary operations (differentiable)."""
    p = {k: v.detach().double().cpu().requires_grad_(True) for k, v in block.named_parameters()}
    x = x.detach().double().cpu().requires_grad_(True)
    outs, t0 = [], 0
    for n in lens:
        residual = x[0, t0:t0 + n]
        h = _norm(residual, p["norm_weights.0"])
        for i, layer in enumerate(block.layers):
            q = lambda name: p[f"layers.{i}.{name}"]  # noqa: E731
            u, z = F.linear(h, q("in_proj.weight")).split([layer.inner, layer.inner], -1)
            W = layer.conv_size
            ext = torch.cat([torch.zeros(W - 1, layer.inner, dtype=torch.float64), u])
            u = F.silu(sum(ext[j:j + n] * q("conv_weight")[:, j] for j in range(W)) + q("conv_bias"))
            r, g = F.linear(u, q("gate_proj.weight"), q("gate_proj.bias")).split([layer.inner, layer.inner], -1)
            la = -torch.exp(q("A_log")) * torch.sigmoid(r)
            a, m = torch.exp(la), torch.sqrt(-torch.expm1(2 * la))
            state, hs = torch.zeros(layer.inner, dtype=torch.float64), []
            for t in range(n):
                state = a[t] * state + m[t] * torch.sigmoid(g[t]) * u[t]
                hs.append(state)
            y = (torch.stack(hs) if n else u) * F.silu(z)
            residual = residual + F.linear(y, q("out_proj.weight"))
            h = _norm(residual, p[f"norm_weights.{2 * i + 1}"])
            f = lambda name: p[f"feed_forward.{i}.{name}.weight"]  # noqa: E731
            residual = residual + F.linear(F.silu(F.linear(h, f("gate_proj"))) * F.linear(h, f("up_proj")), f("down_proj"))
            h = _norm(residual, p[f"norm_weights.{2 * i + 2}"])
        outs.append(h)
        t0 += n
    return torch.cat(outs)[None], p, x


def _rel(a, b):
    return float((a.detach().double().cpu() - b).norm() / b.norm().clamp_min(1e-30))


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-4), (torch.bfloat16, 0.05)])
def test_training_step_against_float64(dtype, tol):
    lens = [70, 0, 1, 30]
    block = _block(dtype)
    x = torch.randn(1, sum(lens), 64, generator=torch.Generator().manual_seed(1)).to(dtype)
    dy = torch.randn(1, sum(lens), 64, generator=torch.Generator().manual_seed(2)).to(dtype)
    want, p, wx = _plain(block, x, lens)
    grads = torch.autograd.grad((want * dy.double()).sum(), [wx, *p.values()])
    block = block.cuda()
    leaf = x.cuda().requires_grad_(True)
    got, none = block(leaf, torch.tensor([0, 70, 70, 71, 101]).cuda())
    assert none is None and _rel(got, want.detach()) <= tol
    got.backward(dy.cuda())
    assert _rel(leaf.grad, grads[0]) <= tol
    for (name, v), g in zip(block.named_parameters(), grads[1:]):
        # decays' gradients are sums of both signs over all tokens: in 16-bit layers looked at in fp32 alone
        if dtype == torch.float32 or "A_log" not in name:
            assert v.grad.dtype == dtype and _rel(v.grad, g) <= tol, name


def test_prompts_and_tokens_continue_each_other():
    block = _block().cuda()
    x = torch.randn(3, 40, 64, generator=torch.Generator().manual_seed(3)).cuda()
    with torch.no_grad():
        whole, _ = block(x)
        first, caches = block(x[:, :17], output_caches=True)
        second, caches = block(x[:, 17:31], caches=caches, output_caches=True)
        parts = [first, second]
        for t in range(31, 40):
            parts.append(block.step(x[:, t], caches).unsqueeze(1))
    assert _rel(torch.cat(parts, 1), whole.double().cpu()) <= 2e-4
    packed = x[:2].reshape(1, 80, 64)
    with torch.no_grad():
        got, _ = block(packed, torch.tensor([0, 40, 80]))
    assert _rel(got.view(2, 40, 64), whole[:2].double().cpu()) <= 2e-4


def test_captured_training_step_and_token_loop():
    block = _block(torch.bfloat16).cuda()
    params = [v.detach().requires_grad_(True) for v in block.parameters()]
    names = [n for n, _ in block.named_parameters()]
    x = torch.randn(2, 50, 64, device="cuda").bfloat16()
    dy = torch.randn_like(x)

    def train():
        y, _ = torch.func.functional_call(block, dict(zip(names, params)), (x,))
        return (y.detach(), *torch.autograd.grad(y, params, dy))

    token = torch.randn(2, 64, device="cuda").bfloat16()
    with torch.no_grad():
        _, caches = block(x, output_caches=True)
    start = [[t.clone() for t in c] for c in caches]
    step = lambda: block.step(token, caches)  # noqa: E731

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train()
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for fn in (train, step):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(fn())
        graphs.append(graph)
    for rep in range(3):
        x.normal_()
        token.normal_()
        graphs[0].replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs[0]]
        assert all(torch.equal(a, b) for a, b in zip(got, train()))
        for c, s in zip(caches, start):
            for t, v in zip(c, s):
                t.copy_(v)
        graphs[1].replay()
        torch.cuda.synchronize()
        got = outs[1].clone()
        for c, s in zip(caches, start):
            for t, v in zip(c, s):
                t.copy_(v)
        assert torch.equal(got, step())


def test_sizes_of_the_layers():
    assert GatedFeedForward(128).intermediate_size == 512 and GatedFeedForward(96).intermediate_size == 256
    layer = GatedRecurrentLayer(64).cuda()
    out, cache = layer(torch.randn(2, 5, 64, device="cuda"), output_cache=True)
    assert out.shape == (2, 5, 64) and cache[0].shape == (2, 128, 4) and cache[1].shape == (2, 128)
    with pytest.raises(ValueError):
        layer(torch.randn(2, 5, 64, device="cuda"), torch.tensor([0, 10]))
