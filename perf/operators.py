"""The state-space mixing layer's operators as timed cases: the selective scan with its gradients and its single-token
step, the causal short convolution in front of it with its state and its gradients, and the norms around the block.

A case is a dict of plain values; ``op`` names the operator:

* ``scan``  ``state_space.state_space_scan``: y_t = C_t S_t + D x_t over S_t = exp(delta_t A) S_{t-1} + delta_t B_t x_t,
  for a dense batch or packed sequences; with ``train`` the gradients of every input come back too;
* ``step``  ``state_space.state_space_step``: one token for each sequence on top of its state;
* ``conv``  ``layer_ops.causal_conv1d`` with the inputs before the first token and the last inputs handed on, forward or
  with its gradients, and ``layer_ops.causal_conv1d_step`` for one token (``mode``);
* ``norm``  ``layer_ops.residual_norm``: norm of a block's output, its gate, the scaled residual add and the next
  block's norm, forward or with gradients.
"""
import math
import random

import torch

own = False  # True: the calls of this package; False: the same operators from elementary torch operations

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CHUNK = 64  # tokens whose pairwise weights the plain scan forms at once
EPS = 1e-5


def listed():
    return [
        # one layer's scan on a full event (60 thousand hits, 8 heads of 64), x, B and C columns of one projection
        {"name": "scan_event", "op": "scan", "n": 1, "T": 60000, "packed": False, "H": 8, "P": 64, "G": 1, "N": 64,
         "dtype": "bf16", "state": False, "train": False},
        # 24 small events of very different lengths in one packed call (6 heads of 32 on a state of 16), each on top of a
        # state and returning it, as chunks of a stream are worked through
        {"name": "scan_packed", "op": "scan", "n": 24, "T": 15000, "packed": True, "H": 6, "P": 32, "G": 2, "N": 16,
         "dtype": "fp16", "state": True, "train": False},
        # a short prompt of two sequences in the exact type, sizes off every tile
        {"name": "scan_short", "op": "scan", "n": 2, "T": 77, "packed": False, "H": 4, "P": 20, "G": 1, "N": 24,
         "dtype": "fp32", "state": True, "train": False},
        # a training step's share of one layer on a full event, the wide state: the largest call
        {"name": "scan_train_event", "op": "scan", "n": 1, "T": 60000, "packed": False, "H": 8, "P": 64, "G": 1, "N": 128,
         "dtype": "bf16", "state": False, "train": True},
        # the same in the exact type on a small packed batch, with states (truncated back-propagation)
        {"name": "scan_train_exact", "op": "scan", "n": 5, "T": 6007, "packed": True, "H": 4, "P": 32, "G": 2, "N": 32,
         "dtype": "fp32", "state": True, "train": True},
        # serving: one new token of one sequence
        {"name": "step_one", "op": "step", "n": 1, "H": 8, "P": 64, "G": 1, "N": 64, "dtype": "bf16"},
        # serving: one new token for each of 250 sequences, wide states
        {"name": "step_many", "op": "step", "n": 250, "H": 8, "P": 64, "G": 1, "N": 128, "dtype": "bf16"},
        # the convolution of a token step: x | B | C columns of 64 sequences
        {"name": "conv_step", "op": "conv", "mode": "step", "n": 64, "T": 64, "packed": False, "D": 640, "W": 4,
         "dtype": "bf16"},
        # the convolution of packed events on top of the inputs before them, the last inputs handed on
        {"name": "conv_packed", "op": "conv", "mode": "prefill", "n": 24, "T": 15000, "packed": True, "D": 224, "W": 4,
         "dtype": "fp16"},
        # the convolution in a training step on a full event
        {"name": "conv_train_event", "op": "conv", "mode": "train", "n": 1, "T": 60000, "packed": False, "D": 640, "W": 4,
         "dtype": "bf16"},
        # the norms of one block border for the tokens of 64 sequences that are being answered: latency
        {"name": "norm_tokens", "op": "norm", "n": 64, "T": 1, "D": 512, "gate": "none", "act": None, "post": False,
         "scale": True, "res": "same", "dtype": "bf16", "train": False},
        # the same in a training step on a full event: post-norm, a gate for each token, a learned residual scale and a
        # residual stream in fp32
        {"name": "norm_train_event", "op": "norm", "n": 1, "T": 60000, "D": 512, "gate": "token", "act": "sigmoid",
         "post": True, "scale": True, "res": "fp32", "dtype": "bf16", "train": True},
    ]


def _spread(rng, lo, hi):
    return min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng):
    op = rng.choice(["scan", "scan", "step", "conv", "norm"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "scan":
        train = rng.random() < 0.5
        H = rng.choice([1, 2, 3, 4, 6, 8])
        P, N = rng.choice([8, 16, 20, 32, 48, 64, 64, 80, 128]), rng.choice([8, 16, 24, 32, 64, 64, 100, 128])
        most = 60000 * 8 * 64 * (64 if train else 32) // (4 if dtype == "fp32" else 1)
        tokens = _spread(rng, 16, max(16, min(60000, most // (H * P * N))))
        packed = rng.random() < 0.5
        n = min(_spread(rng, 1, 32), tokens)
        return {"op": op, "n": n, "T": tokens if packed else max(1, tokens // n), "packed": packed, "H": H, "P": P,
                "G": rng.choice([g for g in (1, 2, 3, 4) if H % g == 0]), "N": N, "dtype": dtype,
                "state": rng.random() < 0.5, "train": train}
    if op == "step":
        H = rng.choice([1, 2, 4, 6, 8, 16])
        return {"op": op, "n": _spread(rng, 1, 250), "H": H, "P": rng.choice([16, 20, 32, 64, 128]),
                "G": rng.choice([g for g in (1, 2, 4) if H % g == 0]), "N": rng.choice([16, 24, 32, 64, 128]),
                "dtype": dtype}
    if op == "conv":
        mode = rng.choice(["step", "prefill", "train"])
        W, D = rng.choice([2, 3, 4, 4, 4]), 8 * _spread(rng, 1, 96)
        packed = mode != "step" and rng.random() < 0.5
        tokens = _spread(rng, 1, 30000 * 640 // max(D, 320))
        n = min(_spread(rng, 1, 250 if mode == "step" else 32), tokens)
        return {"op": op, "mode": mode, "n": n, "T": n if mode == "step" else tokens if packed else max(1, tokens // n),
                "packed": packed, "D": D, "W": W, "dtype": dtype}
    D = rng.choice([24, 64, 96, 128, 200, 512, 768, 1024, 2048])
    rows = _spread(rng, 1, 60000 * 256 // max(D, 256))
    n = min(_spread(rng, 1, 16), rows)
    return {"op": op, "n": n, "T": max(1, rows // n), "D": D, "gate": rng.choice(["none", "token", "sequence"]),
            "act": rng.choice([None, "sigmoid", "silu"]), "post": rng.random() < 0.5, "scale": rng.random() < 0.5,
            "res": rng.choice(["same", "fp32"]), "dtype": dtype, "train": rng.random() < 0.5}


# --------------------------------------------------------------------------------------------------------- inputs
def _lengths(case, seed):
    """Ragged lengths that add up to the case's tokens: cuts at random, with an empty sequence and one of a single token
    where there are four sequences or more."""
    n, T = case["n"], case["T"]
    if not case["packed"]:
        return [T] * n
    r = random.Random(seed)
    fixed = [0, 1] if n >= 4 and T > n else []
    rest, k = T - sum(fixed), n - len(fixed)
    cuts = sorted(r.randint(0, rest) for _ in range(k - 1))
    lens = [b - a for a, b in zip([0] + cuts, cuts + [rest])] + fixed
    r.shuffle(lens)
    return lens


def _sequences(state, case, seed, dev):
    lens = _lengths(case, seed)
    state["lens"] = lens
    state["cu"] = None
    if case["packed"]:
        bounds = [0]
        for length in lens:
            bounds.append(bounds[-1] + length)
        state["cu"] = torch.tensor(bounds, dtype=torch.int64, device=dev)
    return (1, case["T"]) if case["packed"] else (case["n"], case["T"])


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    randn = lambda *s: torch.randn(*s, generator=gen, device=dev)  # noqa: E731
    rand = lambda *s: torch.rand(*s, generator=gen, device=dev)  # noqa: E731
    state = {"case": case}
    leaf = lambda t: t.requires_grad_(True) if case.get("train") or case.get("mode") == "train" else t  # noqa: E731

    if case["op"] in ("scan", "step"):
        H, P, G, N = case["H"], case["P"], case["G"], case["N"]
        shape = _sequences(state, case, seed, dev) if case["op"] == "scan" else (case["n"],)
        # x | B | C are columns of the convolution's output (behind its SiLU), dt a column block of the projection
        xbc = torch.nn.functional.silu(randn(*shape, H * P + 2 * G * N)).to(dtype)
        x, b, c = xbc.split([H * P, G * N, G * N], dim=-1)
        state["x"] = leaf(x.unflatten(-1, (H, P)).detach())
        state["B"], state["C"] = (leaf(t.unflatten(-1, (G, N)).detach()) for t in (b, c))
        state["dt"] = leaf(randn(*shape, H).mul(0.7).to(dtype))
        # the usual initial values: decay rates in 1 .. 16, steps of 0.001 .. 0.1
        state["A"] = leaf(-(1.0 + 15.0 * rand(H)))
        step = torch.exp(rand(H) * math.log(100.0) + math.log(0.001))
        state["dt_bias"] = leaf(step + torch.log(-torch.expm1(-step)))
        state["D"] = leaf(1.0 + 0.1 * randn(H))
        if case["op"] == "step":
            state["state"] = randn(case["n"], H, N, P) * 0.3
            state["new_state"] = torch.empty_like(state["state"])
        else:
            state["h0"] = leaf(randn(case["n"], H, N, P) * 0.3) if case["state"] else None
            if case["train"]:
                state["dy"] = randn(*shape, H, P).to(dtype)
                state["dht"] = randn(case["n"], H, N, P) * 0.3 if case["state"] else None
        return state

    if case["op"] == "conv":
        D, W = case["D"], case["W"]
        if case["mode"] == "step":
            state["x"] = randn(case["n"], D).to(dtype)
            state["cache"] = randn(case["n"], D, W).to(dtype)
            state["new_cache"] = torch.empty_like(state["cache"])
        else:
            shape = _sequences(state, case, seed, dev)
            state["x"] = leaf(randn(*shape, D).to(dtype))
            state["cache"] = randn(case["n"], D, W).to(dtype) if case["mode"] == "prefill" else None
        state["weight"] = leaf((rand(D, W) * 2 - 1) / math.sqrt(W))
        state["bias"] = leaf((rand(D) * 2 - 1) / math.sqrt(W))
        if case["mode"] == "train":
            state["dy"] = randn(*shape, D).to(dtype)
        return state

    n, T, D = case["n"], case["T"], case["D"]
    state["x"] = leaf(randn(n, T, D).to(dtype))
    state["residual"] = leaf((randn(n, T, D) * 2).to(torch.float32 if case["res"] == "fp32" else dtype))
    state["weight"] = leaf(1.0 + 0.1 * randn(D))
    state["post_weight"] = leaf(1.0 + 0.1 * randn(D)) if case["post"] else None
    state["scale"] = leaf(0.5 + 0.1 * randn(D)) if case["scale"] else None
    state["gate"] = {"none": lambda: None, "token": lambda: leaf(randn(n, T, D).to(dtype)),
                     "sequence": lambda: leaf(randn(n, 1, D).to(dtype))}[case["gate"]]()
    if case["train"]:
        state["dy"] = randn(n, T, D).to(dtype)
        state["dres"] = randn(n, T, D).to(state["residual"].dtype)
    return state


# ----------------------------------------------------------------------------------------------------- plain forms
def _padded(s, quantum):
    """Where the tokens of the sequences lie in a batch padded to a multiple of `quantum`: (flat index of each token, n,
    padded length)."""
    n, longest = len(s["lens"]), max(s["lens"])
    L = max(quantum, -(-longest // quantum) * quantum)
    dev = s["x"].device
    lens = torch.tensor(s["lens"], device=dev)
    seq = torch.repeat_interleave(torch.arange(n, device=dev), lens)
    start = torch.cumsum(lens, 0) - lens
    return seq * L + torch.arange(int(lens.sum()), device=dev) - start[seq], n, L


def _spread_out(t, index, n, L):
    """The tokens of t [B, T, ...] in 32 bits at `index` of a zero [n, L, ...]."""
    flat = t.float().reshape(-1, *t.shape[2:])
    return torch.zeros(n * L, *flat.shape[1:], device=t.device).index_copy(0, index, flat).view(n, L, *flat.shape[1:])


def _step_size(s):
    return torch.nn.functional.softplus(s["dt"].float() + s["dt_bias"].float())


def _plain_scan(s):
    case = s["case"]
    H, P, G, N = case["H"], case["P"], case["G"], case["N"]
    index, n, L = _padded(s, CHUNK)
    nc = L // CHUNK
    delta = _step_size(s)
    # chunks [n, H, nc, CHUNK, ...]
    chunks = lambda t: _spread_out(t, index, n, L).transpose(1, 2).unflatten(2, (nc, CHUNK))  # noqa: E731
    x, B, C = chunks(s["x"]), chunks(s["B"]), chunks(s["C"])
    B, C = (t.repeat_interleave(H // G, dim=1) for t in (B, C))
    d = chunks(delta.unsqueeze(-1)).squeeze(-1)
    # exponents are differences of long sums: 64 bits
    g = (d * s["A"].float().view(1, H, 1, 1)).double().cumsum(-1)
    causal = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=x.device).tril()
    decay = (g.unsqueeze(-1) - g.unsqueeze(-2)).masked_fill(~causal, -math.inf).exp().float()
    y = torch.matmul(torch.matmul(C, B.transpose(-1, -2).contiguous()) * decay * d.unsqueeze(-2), x)
    to_end = (g[..., -1:] - g).exp().float() * d
    local = torch.matmul((B * to_end.unsqueeze(-1)).transpose(-1, -2).contiguous(), x)        # [n, H, nc, N, P]
    total = g[..., -1].cumsum(-1)                                                              # [n, H, nc]
    h0 = torch.zeros(n, H, 1, N, P, device=x.device) if s["h0"] is None else s["h0"].float().unsqueeze(2)
    ends = torch.cat([torch.zeros_like(total[..., :1]), total], dim=-1)
    before = torch.ones(nc + 1, nc + 1, dtype=torch.bool, device=x.device).tril()
    carry = (ends.unsqueeze(-1) - ends.unsqueeze(-2)).masked_fill(~before, -math.inf).exp().float()
    states = torch.matmul(carry, torch.cat([h0, local], dim=2).flatten(3)).unflatten(-1, (N, P))
    y = y + torch.matmul(C * g.exp().float().unsqueeze(-1), states[:, :, :-1]) + s["D"].float().view(1, H, 1, 1, 1) * x
    y = y.flatten(2, 3).transpose(1, 2).reshape(n * L, H, P)[index].view(s["x"].shape).to(s["x"].dtype)
    return y, (states[:, :, -1].contiguous() if case["state"] else None)


def _plain_step(s):
    rep = s["case"]["H"] // s["case"]["G"]
    x, delta = s["x"].float(), _step_size(s)
    B, C = (s[k].float().repeat_interleave(rep, dim=1) for k in ("B", "C"))
    new = s["state"] * torch.exp(delta * s["A"])[..., None, None] + (delta[..., None] * B).unsqueeze(-1) * x.unsqueeze(-2)
    y = (C.unsqueeze(-1) * new).sum(-2) + s["D"][:, None] * x
    return y.to(s["x"].dtype), new


def _silu(t):
    return t / (1.0 + torch.exp(-t))


def _plain_conv(s):
    W, D = s["case"]["W"], s["case"]["D"]
    index, n, L = _padded(s, 1)
    x = _spread_out(s["x"], index, n, L)
    past = torch.zeros(n, W, D, device=x.device) if s["cache"] is None else s["cache"].float().transpose(1, 2)
    ext = torch.cat([past, x], dim=1)                                                           # [n, W + L, D]
    y = _silu((ext[:, 1:].unfold(1, W, 1) * s["weight"].float()).sum(-1) + s["bias"].float())   # windows [n, L, D, W]
    y = y.reshape(n * L, D)[index].view(s["x"].shape).to(s["x"].dtype)
    if s["case"]["mode"] == "train":
        return y, None
    lens = torch.tensor(s["lens"], device=x.device)
    last = lens[:, None] + torch.arange(W, device=x.device)
    return y, ext.gather(1, last.unsqueeze(-1).expand(n, W, D)).transpose(1, 2).contiguous().to(s["x"].dtype)


def _plain_conv_step(s):
    cache = torch.cat([s["cache"][..., 1:], s["x"].unsqueeze(-1)], dim=-1)
    y = _silu((cache.float() * s["weight"].float()).sum(-1) + s["bias"].float())
    return y.to(s["x"].dtype), cache


def _unit(t):
    return t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + EPS)


def _plain_norm(s):
    m = s["x"].float()
    m = m if s["post_weight"] is None else _unit(m) * s["post_weight"].float()
    if s["gate"] is not None:
        g = s["gate"].float()
        m = m * {None: lambda t: t, "sigmoid": torch.sigmoid, "silu": _silu}[s["case"]["act"]](g)
    m = m if s["scale"] is None else m * s["scale"].float()
    r = s["residual"].float() + m
    return (_unit(r) * s["weight"].float()).to(s["x"].dtype), r.to(s["residual"].dtype)


# ------------------------------------------------------------------------------------------------------------- run
def _own_scan(s):
    from lampa_amd.state_space import state_space_scan

    return state_space_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], dt_bias=s["dt_bias"], dt_softplus=True,
                            initial_state=s["h0"], output_final_state=s["case"]["state"], cu_seqlens=s["cu"])


def _own_step(s):
    from lampa_amd.state_space import state_space_step

    y = state_space_step(s["x"], s["dt"], s["A"], s["B"], s["C"], s["state"], D=s["D"], dt_bias=s["dt_bias"],
                         dt_softplus=True, new_state=s["new_state"])
    return y, s["new_state"]


def _own_conv(s):
    from lampa_amd.layer_ops import causal_conv1d

    if s["case"]["mode"] == "train":
        return causal_conv1d(s["x"], s["weight"], s["bias"], activation="silu", cu_seqlens=s["cu"]), None
    return causal_conv1d(s["x"], s["weight"], s["bias"], activation="silu", cu_seqlens=s["cu"], initial_state=s["cache"],
                         output_final_state=True)


def _own_conv_step(s):
    from lampa_amd.layer_ops import causal_conv1d_step

    y = causal_conv1d_step(s["x"], s["cache"], s["weight"], s["bias"], activation="silu", new_cache=s["new_cache"])
    return y, s["new_cache"]


def _own_norm(s):
    from lampa_amd.layer_ops import residual_norm

    return residual_norm(s["x"], s["residual"], s["weight"], post_weight=s["post_weight"], gate=s["gate"],
                         gate_activation=s["case"]["act"], residual_scale=s["scale"], eps=EPS)


LEAVES = {"scan": ("x", "dt", "A", "B", "C", "D", "dt_bias", "h0"), "conv": ("x", "weight", "bias"),
          "norm": ("x", "residual", "weight", "post_weight", "gate", "scale")}


def run(state):
    case = state["case"]
    op = case["op"] + ("_step" if case.get("mode") == "step" else "")
    if own:
        forward = {"scan": _own_scan, "step": _own_step, "conv": _own_conv, "conv_step": _own_conv_step, "norm": _own_norm}
    else:
        forward = {"scan": _plain_scan, "step": _plain_step, "conv": _plain_conv, "conv_step": _plain_conv_step,
                   "norm": _plain_norm}
    y, other = forward[op](state)
    out = {"y": y} if other is None else {"y": y, "other": other}
    if case.get("train") or case.get("mode") == "train":
        names = [k for k in LEAVES[op] if state[k] is not None]
        into = [(y, state["dy"])] + ([] if other is None else [(other, state["dht" if op == "scan" else "dres"])])
        grads = torch.autograd.grad([o for o, _ in into], [state[k] for k in names], [g for _, g in into])
        out = {k: t.detach() for k, t in out.items()}
        out.update({"d" + k: g for k, g in zip(names, grads)})
    return out


# ------------------------------------------------------------------------------------------------------------ work
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "step":
        state = case["n"] * case["H"] * case["N"] * case["P"]
        io = case["n"] * (2 * case["H"] * case["P"] + 2 * case["G"] * case["N"] + case["H"])
        return {"bytes": 2 * 4 * state + e * io, "flops": 5 * state}
    tokens = case["T"] if case.get("packed") else case["n"] * case["T"]
    if case["op"] == "scan":
        x, bc, dt = case["H"] * case["P"], 2 * case["G"] * case["N"], case["H"]
        state = case["n"] * x * case["N"] * 4 if case["state"] else 0
        # decay, update and read-out; the gradients need the state again, its adjoint, and three read-outs
        flops = (5 + (12 if case["train"] else 0)) * tokens * x * case["N"]
        return {"bytes": tokens * e * (4 * x + 2 * bc + 2 * dt if case["train"] else 2 * x + bc + dt)
                + state * (4 if case["train"] else 2), "flops": flops}
    if case["op"] == "conv":
        D, W = case["D"], case["W"]
        rows = case["n"] if case["mode"] == "step" else tokens
        cache = 0 if case["mode"] == "train" else 2 * case["n"] * D * W * e
        return {"bytes": rows * D * e * (4 if case["mode"] == "train" else 2) + cache + 4 * D * (W + 1),
                "flops": rows * D * (2 * W + 8) * (3 if case["mode"] == "train" else 1)}
    D, r = case["D"], 4 if case["res"] == "fp32" else e
    gate = {"none": 0, "token": tokens, "sequence": case["n"]}[case["gate"]] * D * e
    once = tokens * D * 2 * (e + r) + gate                  # x and the residual read, both outputs written
    return {"bytes": once * (2 if case["train"] else 1), "flops": tokens * D * (12 + (30 if case["train"] else 0))}


# ----------------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    """The operators from their definitions in 64 bits: the recurrences token by token (pieces of a sequence side by side,
    the state then handed from piece to piece), the gradients from the adjoint recurrence, convolutions and norms from
    their sums."""
    s = prepare(case, seed)
    with torch.no_grad():
        f = {k: (t.detach().double() if torch.is_tensor(t) and t.is_floating_point() else t) for k, t in s.items()}
        sig = lambda t: 1.0 / (1.0 + torch.exp(-t))  # noqa: E731

        if case["op"] == "norm":
            x, r, w, pw, sc, gate = f["x"], f["residual"], f["weight"], f["post_weight"], f["scale"], f["gate"]
            D = case["D"]
            i1 = 1.0 / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS)
            a = x if pw is None else x * i1 * pw
            one = torch.ones((), dtype=torch.float64, device=x.device)
            act, slope = {None: lambda g: (g, one), "sigmoid": lambda g: (sig(g), sig(g) * (1 - sig(g))),
                          "silu": lambda g: (g * sig(g), sig(g) * (1 + g * (1 - sig(g))))}[case["act"]](
                              one if gate is None else gate)
            act = one if gate is None else act
            scale = one if sc is None else sc
            h = r + scale * act * a
            i2 = 1.0 / torch.sqrt((h * h).sum(-1, keepdim=True) / D + EPS)
            out = {"y": h * i2 * w, "other": h}
            if case["train"]:
                dyw = f["dy"] * w
                dh = f["dres"] + i2 * dyw - h * i2 ** 3 * (dyw * h).sum(-1, keepdim=True) / D
                da = dh * scale * act
                if pw is None:
                    out["dx"] = da
                else:
                    dn = da * pw
                    out["dx"] = i1 * dn - x * i1 ** 3 * (dn * x).sum(-1, keepdim=True) / D
                out["dresidual"] = dh
                out["dweight"] = (f["dy"] * h * i2).sum((0, 1))
                if pw is not None:
                    out["dpost_weight"] = (da * x * i1).sum((0, 1))
                if gate is not None:
                    dg = dh * scale * a * slope
                    out["dgate"] = dg.sum(1, keepdim=True) if case["gate"] == "sequence" else dg
                if sc is not None:
                    out["dscale"] = (dh * act * a).sum((0, 1))
            return out

        if case["op"] == "conv" and case["mode"] == "step":
            cache = torch.roll(f["cache"], -1, -1)
            cache[..., -1] = f["x"]
            pre = torch.einsum("ndw,dw->nd", cache, f["weight"]) + f["bias"]
            return {"y": pre * sig(pre), "other": cache}

        if case["op"] == "conv":
            W, D = case["W"], case["D"]
            x = f["x"].reshape(-1, D)
            y, last, grads, at = torch.empty_like(x), [], None, 0
            if case["mode"] == "train":
                dy = f["dy"].reshape(-1, D)
                grads = [torch.zeros_like(x), torch.zeros_like(f["weight"]), torch.zeros_like(f["bias"])]
            for i, length in enumerate(s["lens"]):
                past = torch.zeros(W, D, dtype=torch.float64, device=x.device) if f["cache"] is None else f["cache"][i].T
                ext = torch.cat([past, x[at:at + length]])
                last.append(ext[length:].T)
                pre = f["bias"].expand(length, D).clone()
                for j in range(W):
                    pre += ext[j + 1:j + 1 + length] * f["weight"][:, j]
                y[at:at + length] = pre * sig(pre)
                if grads is not None:
                    dpre = dy[at:at + length] * sig(pre) * (1 + pre * (1 - sig(pre)))
                    dext = torch.zeros_like(ext)
                    for j in range(W):
                        dext[j + 1:j + 1 + length] += dpre * f["weight"][:, j]
                        grads[1][:, j] += (dpre * ext[j + 1:j + 1 + length]).sum(0)
                    grads[0][at:at + length] = dext[W:]
                    grads[2] += dpre.sum(0)
                at += length
            out = {"y": y.view(f["x"].shape)}
            if grads is None:
                return {**out, "other": torch.stack(last)}
            return {**out, "dx": grads[0].view(f["x"].shape), "dweight": grads[1], "dbias": grads[2]}

        H, P, G, N = case["H"], case["P"], case["G"], case["N"]
        raw = f["dt"] + f["dt_bias"]
        delta = torch.clamp(raw, min=0) + torch.log1p(torch.exp(-raw.abs()))
        wide = lambda t: t.repeat_interleave(H // G, dim=-2)  # noqa: E731
        if case["op"] == "step":
            new = torch.exp(delta * f["A"])[..., None, None] * f["state"] + torch.einsum(
                "bh,bhn,bhp->bhnp", delta, wide(f["B"]), f["x"])
            return {"y": torch.einsum("bhn,bhnp->bhp", wide(f["C"]), new) + f["D"][:, None] * f["x"], "other": new}

        def walk(u, v, q, a, init):
            """Per sequence: S_t = a_t S_{t-1} + u_t v_t^T from `init`, out_t = S_t^T q_t; (outs, the last S). Token by
            token in pieces of about the square root of the length, all pieces at once, then the pieces joined."""
            T = u.shape[0]
            if T == 0:
                return v.clone(), init
            L = max(1, int(math.sqrt(T)))
            m = -(-T // L)
            pad = lambda t, fill: torch.cat([t, t.new_full((m * L - T, *t.shape[1:]), fill)]).view(m, L, *t.shape[1:])  # noqa: E731
            u, v, q, a = pad(u, 0.0), pad(v, 0.0), pad(q, 0.0), pad(a, 1.0)
            S = u.new_zeros(m, H, u.shape[-1], v.shape[-1])
            alone = torch.empty_like(v)
            for t in range(L):
                S = S * a[:, t, :, None, None] + u[:, t, :, :, None] * v[:, t, :, None, :]
                alone[:, t] = (S * q[:, t, :, :, None]).sum(-2)
            reach = torch.cumprod(a, 1)
            carried, cur = [], init
            for i in range(m):
                carried.append(cur)
                cur = cur * reach[i, -1][:, None, None] + S[i]
            alone += reach.unsqueeze(-1) * torch.einsum("mlhn,mhnp->mlhp", q, torch.stack(carried))
            return alone.reshape(m * L, *v.shape[2:])[:T], cur

        flat = lambda t: t.reshape(-1, *t.shape[2:])  # noqa: E731
        x, B, C, d = flat(f["x"]), flat(wide(f["B"])), flat(wide(f["C"])), flat(delta)
        g = d * f["A"]
        a = torch.exp(g)
        y, ends, at = torch.empty_like(x), [], 0
        if case["train"]:
            dy = flat(f["dy"])
            dx, dB, dC, dd, dA = f["D"][:, None] * dy, torch.empty_like(B), torch.empty_like(C), torch.empty_like(d), 0.0
            dh0 = []
        for i, length in enumerate(s["lens"]):
            at, k = at + length, slice(at, at + length)
            init = x.new_zeros(H, N, P) if f["h0"] is None else f["h0"][i]
            yk, last = walk(B[k], x[k] * d[k][..., None], C[k], a[k], init)
            y[k] = yk + f["D"][:, None] * x[k]
            ends.append(last)
            if not case["train"]:
                continue
            dht = torch.zeros_like(init) if f["dht"] is None else f["dht"][i]
            # out_t = sum_s of the pair weights times v_s, whichever of the three is read out
            dC[k] = walk(x[k] * d[k][..., None], B[k], dy[k], a[k], init.transpose(-1, -2))[0]
            # the adjoint runs from the end: R_t = C_t dy_t^T + a_{t+1} R_{t+1}
            back = lambda t: torch.flip(t, [0])  # noqa: E731
            a_next = torch.cat([a[k][1:], a.new_ones(1, H)]) if length else a[k]
            xr, first = walk(back(C[k]), back(dy[k]), back(B[k]), back(a_next), dht)
            br, _ = walk(back(dy[k]), back(C[k]), back(x[k]), back(a_next), dht.transpose(-1, -2))
            xr, br = back(xr), back(br)
            dh0.append(first * a[k][0][:, None, None] if length else first)
            dx[k] += d[k][..., None] * xr
            dB[k] = d[k][..., None] * br
            # d/dg_t = <R_t, a_t S_{t-1}>: what the later outputs and the last state read of what came before t
            read, written = (yk * dy[k]).sum(-1), d[k] * (xr * x[k]).sum(-1)
            dg = back(torch.cumsum(back(read - written), 0)) + (dht * last).sum((-1, -2))
            dd[k] = f["A"] * dg + (xr * x[k]).sum(-1)
            dA = dA + (d[k] * dg).sum(0)
        out = {"y": y.view(f["x"].shape)}
        if case["state"]:
            out["other"] = torch.stack(ends)
        if case["train"]:
            shared = lambda t: t.view(-1, G, H // G, N).sum(2).view(f["B"].shape)  # noqa: E731
            draw_dt = dd * sig(flat(raw))
            out.update({"dx": dx.view(f["x"].shape), "ddt": draw_dt.view(f["dt"].shape), "dA": dA, "dB": shared(dB),
                        "dC": shared(dC), "dD": (x * dy).sum((0, 2)), "ddt_bias": draw_dt.sum(0)})
            if case["state"]:
                out["dh0"] = torch.stack(dh0)
        return out
