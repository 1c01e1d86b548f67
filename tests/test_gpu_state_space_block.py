"""The state-space operators together, as a layer and a block use them: training on packed sequences against a float64 block of
elementary torch operations, prompts continued by further prompts and by single tokens, a captured token loop.

Tolerances. fp32: the layers' products go through library GEMMs (about K half-steps of fp32 in K-long sums, K <= 160) and the
operators' bounds; three layers' norms carry relative errors on: 2e-4 of a tensor's norm is more than a thousand half-steps
for each. Two ways through the same fp32 operators (one call against pieces) agree to the same. bf16: a dozen roundings of
2^-9 rms each lie between input and output of a layer, 0.05 of the norm bounds three layers."""
import pytest
import torch
import torch.nn.functional as F

from lampa_amd.block import StateSpaceBlock, StateSpaceLayer

pytestmark = pytest.mark.gpu


def _block(dtype=torch.float32, seed=0, **kw):
    torch.manual_seed(seed)
    return StateSpaceBlock(64, 3, residual_scale=0.7, d_state=16, head_dim=16, expand=2, n_groups=2, **kw).to(dtype)


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
            z, xbc, dt = F.linear(h, q("in_proj.weight")).split([layer.inner, layer.conv_dim, layer.num_heads], -1)
            W = layer.conv_size
            ext = torch.cat([torch.zeros(W - 1, layer.conv_dim, dtype=torch.float64), xbc])
            xbc = F.silu(sum(ext[j:j + n] * q("conv_weight")[:, j] for j in range(W)) + q("conv_bias"))
            gn = layer.n_groups * layer.d_state
            xs, B, C = xbc.split([layer.inner, gn, gn], -1)
            H, G = layer.num_heads, layer.n_groups
            xs = xs.view(n, H, layer.head_dim)
            B, C = (t.view(n, G, layer.d_state).repeat_interleave(H // G, 1) for t in (B, C))
            delta = F.softplus(dt + q("dt_bias"))
            S, ys = torch.zeros(H, layer.d_state, layer.head_dim, dtype=torch.float64), []
            for t in range(n):
                S = torch.exp(-delta[t] * torch.exp(q("A_log")))[:, None, None] * S + (
                    delta[t][:, None] * B[t])[:, :, None] * xs[t][:, None, :]
                ys.append((C[t][:, :, None] * S).sum(1) + q("D")[:, None] * xs[t])
            y = torch.stack(ys).reshape(n, layer.inner) if n else xs.reshape(0, layer.inner)
            out = F.linear(_norm(y * F.silu(z), q("norm_weight")), q("out_proj.weight"))
            residual = residual + p[f"scales.{i}"] * out
            h = _norm(residual, p[f"norm_weights.{i + 1}"])
        outs.append(h)
        t0 += n
    return torch.cat(outs)[None], p, x


def _rel(a, b):
    return float((a.detach().double().cpu() - b).norm() / b.norm().clamp_min(1e-30))


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-4), (torch.bfloat16, 0.05)])
def test_training_step_against_float64(device, dtype, tol):
    lens = [70, 0, 1, 30]
    block = _block(dtype)
    x = torch.randn(1, sum(lens), 64, generator=torch.Generator().manual_seed(1)).to(dtype)
    dy = torch.randn(1, sum(lens), 64, generator=torch.Generator().manual_seed(2)).to(dtype)
    want, p, wx = _plain(block, x, lens)
    grads = torch.autograd.grad((want * dy.double()).sum(), [wx, *p.values()])
    block = block.to(device)
    leaf = x.to(device).requires_grad_(True)
    cu = torch.tensor([0, 70, 70, 71, 101], device=device)
    got, none = block(leaf, cu)
    assert none is None and _rel(got, want.detach()) <= tol
    got.backward(dy.to(device))
    assert _rel(leaf.grad, grads[0]) <= tol
    for (name, v), g in zip(block.named_parameters(), grads[1:]):
        # A_log and dt_bias: sums of both signs over all tokens and 16-bit inputs of them; looked at together with the rest in fp32
        if dtype == torch.float32 or not name.endswith(("A_log", "dt_bias")):
            assert _rel(v.grad, g) <= tol, name


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-4), (torch.bfloat16, 0.05)])
def test_prompts_in_pieces_and_single_tokens(device, dtype, tol):
    block = _block(dtype, 3).to(device)
    x = torch.randn(2, 150, 64, generator=torch.Generator().manual_seed(4)).to(dtype).to(device)
    with torch.no_grad():
        whole, _ = block(x)
        a, caches = block(x[:, :2], output_caches=True)
        b, caches = block(x[:, 2:140], caches=caches, output_caches=True)
        parts = [a, b] + [block.step(x[:, t], caches)[:, None] for t in range(140, 150)]
    assert _rel(torch.cat(parts, 1), whole.double().cpu()) <= tol


def test_captured_token_loop(device):
    """The step captured once and replayed: the eager bits, and the caches move on in the same memory."""
    block = _block(torch.bfloat16, 5).to(device)
    x = torch.randn(3, 20, 64, device=device).bfloat16()
    with torch.no_grad():
        _, caches = block(x[:, :10], output_caches=True)
        eager = [tuple(t.clone() for t in c) for c in caches]
        static = x[:, 10].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            block.step(static, [tuple(t.clone() for t in c) for c in caches])
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = block.step(static, caches)
        for t in range(10, 20):
            static.copy_(x[:, t])
            graph.replay()
            want = block.step(x[:, t], eager)
            assert torch.equal(out, want)
            for c, e in zip(caches, eager):
                assert torch.equal(c[0], e[0]) and torch.equal(c[1], e[1])


def test_refusals():
    with pytest.raises(ValueError, match="divide"):
        StateSpaceLayer(64, head_dim=48)
    with pytest.raises(ValueError, match="divide"):
        StateSpaceLayer(64, head_dim=64, expand=2, n_groups=4)
