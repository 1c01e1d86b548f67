"""The operators of a gated recurrent block as timed cases: the gated linear recurrence with its gradients and its
single-token step, and the gated feed-forward block with its gradients.

A case is a dict of plain values; ``op`` names the operator:

* ``scan``  ``linear_recurrence.gated_recurrence``: h_t = a_t h_{t-1} + u_t for each channel, a_t = exp(A sigmoid(r_t)),
  u_t = sqrt(1 - a_t^2) sigmoid(i_t) x_t, y_t = act(z_t) h_t, for a dense batch or packed sequences; with ``train`` the
  gradients of every input come back too;
* ``step``  ``linear_recurrence.gated_recurrence_step``: one token for each sequence on top of its state;
* ``ffn``   ``feed_forward.gated_feed_forward``: (act(x Wg^T) * (x Wu^T)) Wd^T, forward or with gradients.
"""
import math
import random

import torch

own = False  # True: the calls of this package; False: the same operators from elementary torch operations

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CHUNK = 256  # tokens whose sums the plain recurrence takes from one common origin


def listed():
    return [
        # one layer's recurrence on a full event (60 thousand hits, 512 channels), gated output, gates from projections
        {"name": "scan_event", "op": "scan", "n": 1, "T": 60000, "packed": False, "D": 512, "input_gate": True,
         "gate": "silu", "normalize": True, "dtype": "bf16", "state": False, "train": False},
        # 24 small events of very different lengths in one packed call, each on top of a state and returning it, as chunks
        # of a stream are worked through
        {"name": "scan_packed", "op": "scan", "n": 24, "T": 15000, "packed": True, "D": 192, "input_gate": True,
         "gate": "silu", "normalize": True, "dtype": "fp16", "state": True, "train": False},
        # a short prompt of two sequences in the exact type, sizes off every tile, the recurrence alone
        {"name": "scan_short", "op": "scan", "n": 2, "T": 77, "packed": False, "D": 97, "input_gate": False,
         "gate": "none", "normalize": False, "dtype": "fp32", "state": True, "train": False},
        # a training step's share of one layer on a full event
        {"name": "scan_train_event", "op": "scan", "n": 1, "T": 60000, "packed": False, "D": 512, "input_gate": True,
         "gate": "silu", "normalize": True, "dtype": "bf16", "state": False, "train": True},
        # the same in the exact type on a small packed batch, with states (truncated back-propagation)
        {"name": "scan_train_exact", "op": "scan", "n": 5, "T": 6007, "packed": True, "D": 128, "input_gate": True,
         "gate": "sigmoid", "normalize": True, "dtype": "fp32", "state": True, "train": True},
        # serving: one new token of one sequence
        {"name": "step_one", "op": "step", "n": 1, "D": 512, "input_gate": True, "gate": "silu", "normalize": True,
         "dtype": "bf16"},
        # serving: one new token for each of 250 sequences
        {"name": "step_many", "op": "step", "n": 250, "D": 1024, "input_gate": True, "gate": "silu", "normalize": True,
         "dtype": "bf16"},
        # serving: the feed-forward block for one token, latency
        {"name": "ffn_token", "op": "ffn", "rows": 1, "D": 128, "F": 512, "act": "silu", "dtype": "bf16", "train": False},
        # the feed-forward block of one layer on a full event
        {"name": "ffn_event", "op": "ffn", "rows": 60000, "D": 128, "F": 512, "act": "silu", "dtype": "bf16",
         "train": False},
        # the same in a training step
        {"name": "ffn_train_event", "op": "ffn", "rows": 60000, "D": 128, "F": 512, "act": "silu", "dtype": "bf16",
         "train": True},
        # a training step of a wide block: the largest call
        {"name": "ffn_train_wide", "op": "ffn", "rows": 8192, "D": 768, "F": 2048, "act": "silu", "dtype": "bf16",
         "train": True},
        # a training step of a small block in the exact type, rows off every tile
        {"name": "ffn_train_exact", "op": "ffn", "rows": 1501, "D": 96, "F": 256, "act": "sigmoid", "dtype": "fp32",
         "train": True},
    ]


def _spread(rng, lo, hi):
    return min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng):
    op = rng.choice(["scan", "scan", "scan", "step", "ffn", "ffn", "ffn"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    gates = {"input_gate": rng.random() < 0.75, "gate": rng.choice(["none", "silu", "silu", "sigmoid", "linear"]),
             "normalize": rng.random() < 0.75}
    if op == "scan":
        D = rng.choice([8, 24, 33, 64, 96, 100, 128, 192, 250, 256, 384, 512, 640, 768, 1024, 2048])
        tokens = _spread(rng, 1, min(60000, 60000 * 512 // D // (2 if dtype == "fp32" else 1)))
        packed = rng.random() < 0.5
        n = min(_spread(rng, 1, 32), tokens)
        return {"op": op, "n": n, "T": tokens if packed else max(1, tokens // n), "packed": packed, "D": D, **gates,
                "dtype": dtype, "state": rng.random() < 0.5, "train": rng.random() < 0.5}
    if op == "step":
        return {"op": op, "n": _spread(rng, 1, 250), "D": rng.choice([24, 33, 96, 128, 250, 512, 768, 1024, 2048]), **gates,
                "dtype": dtype}
    D, F = 8 * _spread(rng, 1, 128), 8 * _spread(rng, 4, 352)
    most = 8192 * 768 * 2048 // (16 if dtype == "fp32" else 1)
    return {"op": op, "rows": _spread(rng, 1, max(1, min(60000, most // (D * F)))), "D": D, "F": F,
            "act": rng.choice(["silu", "silu", "sigmoid", "none"]), "dtype": dtype, "train": rng.random() < 0.5}


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


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    randn = lambda *s: torch.randn(*s, generator=gen, device=dev)  # noqa: E731
    rand = lambda *s: torch.rand(*s, generator=gen, device=dev)  # noqa: E731
    state = {"case": case}
    leaf = lambda t: t.requires_grad_(True) if case.get("train") else t  # noqa: E731

    if case["op"] == "ffn":
        rows, D, F = case["rows"], case["D"], case["F"]
        # x comes from a norm, the weights are at their initial scale
        state["x"] = leaf(randn(rows, D).to(dtype))
        state["w_gate"], state["w_up"] = (leaf((randn(F, D) / math.sqrt(D)).to(dtype)) for _ in range(2))
        state["w_down"] = leaf((randn(D, F) / math.sqrt(F)).to(dtype))
        if case["train"]:
            state["dy"] = randn(rows, D).to(dtype)
        return state

    n, D = case["n"], case["D"]
    if case["op"] == "scan":
        lens = _lengths(case, seed)
        state["lens"], state["cu"], shape = lens, None, (n, case["T"])
        if case["packed"]:
            bounds = [0]
            for length in lens:
                bounds.append(bounds[-1] + length)
            state["cu"], shape = torch.tensor(bounds, dtype=torch.int64, device=dev), (1, case["T"])
    else:
        shape = (n,)
    # the two gates are columns of one projection, x and z of another
    r, i = randn(*shape, 2 * D).to(dtype).split([D, D], dim=-1)
    x, z = randn(*shape, 2 * D).to(dtype).split([D, D], dim=-1)
    state["x"], state["decay_gate"] = leaf(x.detach()), leaf(r.detach())
    state["input_gate"] = leaf(i.detach()) if case["input_gate"] else None
    state["gate"] = None if case["gate"] == "none" else leaf(z.detach())
    # the usual initial values: a token with an open gate keeps 0.9 .. 0.999 of the state
    state["A"] = leaf(torch.log(0.9 + 0.099 * rand(D)))
    if case["op"] == "step":
        state["state"] = randn(n, D)
        state["new_state"] = torch.empty_like(state["state"])
        return state
    state["h0"] = leaf(randn(n, D)) if case["state"] else None
    if case["train"]:
        state["dy"] = randn(*shape, D).to(dtype)
        state["dht"] = randn(n, D) if case["state"] else None
    return state


# ----------------------------------------------------------------------------------------------------- plain forms
ACT = {"none": None, "linear": None, "silu": "silu", "sigmoid": "sigmoid"}


def _sigmoid(t):
    return 1.0 / (1.0 + torch.exp(-t))


def _act(name, t):
    return {"silu": lambda v: v * _sigmoid(v), "sigmoid": _sigmoid}.get(name, lambda v: v)(t)


def _decay_and_input(s):
    """log a_t and u_t of every token, in 32 bits."""
    log_a = s["A"].float() * _sigmoid(s["decay_gate"].float())
    u = s["x"].float()
    if s["input_gate"] is not None:
        u = u * _sigmoid(s["input_gate"].float())
    if s["case"]["normalize"]:
        u = u * torch.sqrt(-torch.expm1(2.0 * log_a))
    return log_a, u


def _plain_scan(s):
    lens, D = s["lens"], s["case"]["D"]
    n, L, dev = len(lens), max(CHUNK, -(-max(lens) // CHUNK) * CHUNK), s["x"].device
    nc = L // CHUNK
    sizes = torch.tensor(lens, device=dev)
    seq = torch.repeat_interleave(torch.arange(n, device=dev), sizes)
    index = seq * L + torch.arange(sum(lens), device=dev) - (torch.cumsum(sizes, 0) - sizes)[seq]
    # sequences padded to whole chunks by tokens that leave the state as it is
    chunks = lambda t: torch.zeros(n * L, D, device=dev).index_copy(0, index, t.reshape(-1, D)).view(n, nc, CHUNK, D)  # noqa: E731
    log_a, u = _decay_and_input(s)
    # sums of many exponents, and what is scaled by their exponentials: 64 bits
    g = chunks(log_a).double().cumsum(2)
    inner = g.exp() * (chunks(u).double() * torch.exp(-g)).cumsum(2)
    total, local = g[:, :, -1], inner[:, :, -1]
    h0 = torch.zeros(n, 1, D, device=dev, dtype=torch.float64) if s["h0"] is None else s["h0"].double().unsqueeze(1)
    ends = torch.cat([torch.zeros_like(total[:, :1]), total.cumsum(1)], dim=1)
    before = torch.ones(nc + 1, nc + 1, dtype=torch.bool, device=dev).tril().unsqueeze(-1)
    carry = (ends.unsqueeze(2) - ends.unsqueeze(1)).masked_fill(~before, -math.inf).exp()
    states = (carry * torch.cat([h0, local], dim=1).unsqueeze(1)).sum(2)
    h = (inner + g.exp() * states[:, :-1].unsqueeze(2)).float().reshape(n * L, D)[index].view(s["x"].shape)
    y = h if s["gate"] is None else h * _act(s["case"]["gate"], s["gate"].float())
    return y.to(s["x"].dtype), (states[:, -1].float() if s["case"]["state"] else None)


def _plain_step(s):
    log_a, u = _decay_and_input(s)
    new = s["state"] * torch.exp(log_a) + u
    y = new if s["gate"] is None else new * _act(s["case"]["gate"], s["gate"].float())
    return y.to(s["x"].dtype), new


def _plain_ffn(s):
    x, wg, wu, wd = (s[k].float() for k in ("x", "w_gate", "w_up", "w_down"))
    hidden = _act(s["case"]["act"], torch.matmul(x, wg.t())) * torch.matmul(x, wu.t())
    return torch.matmul(hidden, wd.t()).to(s["x"].dtype), None


# ------------------------------------------------------------------------------------------------------------- run
def _own_scan(s):
    from lampa_amd.linear_recurrence import gated_recurrence

    case = s["case"]
    return gated_recurrence(s["x"], s["decay_gate"], s["A"], input_gate=s["input_gate"], gate=s["gate"],
                            gate_activation=ACT[case["gate"]], normalize=case["normalize"], initial_state=s["h0"],
                            output_final_state=case["state"], cu_seqlens=s["cu"])


def _own_step(s):
    from lampa_amd.linear_recurrence import gated_recurrence_step

    y = gated_recurrence_step(s["x"], s["decay_gate"], s["A"], s["state"], input_gate=s["input_gate"], gate=s["gate"],
                              gate_activation=ACT[s["case"]["gate"]], normalize=s["case"]["normalize"],
                              new_state=s["new_state"])
    return y, s["new_state"]


def _own_ffn(s):
    from lampa_amd.feed_forward import gated_feed_forward

    return gated_feed_forward(s["x"], s["w_gate"], s["w_up"], s["w_down"], activation=ACT[s["case"]["act"]]), None


LEAVES = {"scan": ("x", "decay_gate", "A", "input_gate", "gate", "h0"), "ffn": ("x", "w_gate", "w_up", "w_down")}


def run(state):
    case = state["case"]
    if own:
        forward = {"scan": _own_scan, "step": _own_step, "ffn": _own_ffn}
    else:
        forward = {"scan": _plain_scan, "step": _plain_step, "ffn": _plain_ffn}
    y, other = forward[case["op"]](state)
    out = {"y": y} if other is None else {"y": y, "state": other}
    if case.get("train"):
        names = [k for k in LEAVES[case["op"]] if state[k] is not None]
        into = [(y, state["dy"])] + ([] if other is None else [(other, state["dht"])])
        grads = torch.autograd.grad([o for o, _ in into], [state[k] for k in names], [g for _, g in into])
        out = {k: t.detach() for k, t in out.items()}
        out.update({"d" + k: g for k, g in zip(names, grads)})
    return out


# ------------------------------------------------------------------------------------------------------------ work
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "ffn":
        rows, D, F = case["rows"], case["D"], case["F"]
        # forward: three products; gradients: of the hidden values, of x (two) and of the weights (three)
        return {"bytes": e * (rows * D * (4 if case["train"] else 2) + 3 * D * F * (2 if case["train"] else 1)),
                "flops": 2 * rows * D * F * (9 if case["train"] else 3)}
    inputs = 2 + int(case["input_gate"]) + int(case["gate"] != "none")
    if case["op"] == "step":
        return {"bytes": case["n"] * case["D"] * (8 + e * (inputs + 1)), "flops": 20 * case["n"] * case["D"]}
    size = (case["T"] if case["packed"] else case["n"] * case["T"]) * case["D"]
    state = case["n"] * case["D"] * 4 if case["state"] else 0
    if case["train"]:  # the inputs and dy read, y and the inputs' gradients written
        return {"bytes": size * e * (2 * inputs + 2) + 4 * state, "flops": 60 * size}
    return {"bytes": size * e * (inputs + 1) + 2 * state, "flops": 20 * size}


# ----------------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    """The operators from their definitions in 64 bits: the recurrence token by token (pieces of a sequence side by side,
    the state then handed from piece to piece), its gradients from the adjoint recurrence, the feed-forward block's from the
    product rule."""
    s = prepare(case, seed)
    with torch.no_grad():
        f = {k: (t.detach().double() if torch.is_tensor(t) and t.is_floating_point() else t) for k, t in s.items()}
        sig = lambda t: torch.special.expit(t)  # noqa: E731
        one = lambda t: torch.ones_like(t)  # noqa: E731
        act = {"silu": lambda t: (t * sig(t), sig(t) * (1 + t * (1 - sig(t)))),
               "sigmoid": lambda t: (sig(t), sig(t) * (1 - sig(t)))}

        if case["op"] == "ffn":
            x, wg, wu, wd = f["x"], f["w_gate"], f["w_up"], f["w_down"]
            pre, up = x @ wg.T, x @ wu.T
            value, slope = act.get(case["act"], lambda t: (t, one(t)))(pre)
            out = {"y": (value * up) @ wd.T}
            if case["train"]:
                dh = f["dy"] @ wd
                dpre, dup = dh * up * slope, dh * value
                out.update({"dx": dpre @ wg + dup @ wu, "dw_gate": dpre.T @ x, "dw_up": dup.T @ x,
                            "dw_down": f["dy"].T @ (value * up)})
            return out

        sr = sig(f["decay_gate"])
        log_a = f["A"] * sr
        a = torch.exp(log_a)
        si = one(a) if f["input_gate"] is None else sig(f["input_gate"])
        m = torch.sqrt(-torch.expm1(2 * log_a)) if case["normalize"] else one(a)
        u = m * si * f["x"]
        if f["gate"] is None:
            value, slope = one(a), torch.zeros_like(a)
        else:
            value, slope = act.get(case["gate"], lambda t: (t, one(t)))(f["gate"])
        if case["op"] == "step":
            new = a * f["state"] + u
            return {"y": new * value, "state": new}

        def walk(a, u, init):
            """h_t = a_t h_{t-1} + u_t from `init`, all h_t [T, D]: token by token in pieces of about the square root of the
            length, all pieces at once, then the pieces joined."""
            T = a.shape[0]
            if T == 0:
                return u.clone()
            size = max(1, int(math.sqrt(T)))
            m = -(-T // size)
            pad = lambda t, fill: torch.cat([t, t.new_full((m * size - T, t.shape[1]), fill)]).view(m, size, -1)  # noqa: E731
            a, u = pad(a, 1.0), pad(u, 0.0)
            h = torch.empty_like(u)
            cur = torch.zeros_like(u[:, 0])
            for t in range(size):
                cur = a[:, t] * cur + u[:, t]
                h[:, t] = cur
            reach = torch.cumprod(a, 1)
            carried = init
            for i in range(m):
                h[i] += reach[i] * carried
                carried = h[i, -1]
            return h.reshape(m * size, -1)[:T]

        D = case["D"]
        flat = lambda t: t.reshape(-1, D)  # noqa: E731
        a, u, value, slope, sr, si, m, x = (flat(t) for t in (a, u, value, slope, sr, si, m, f["x"]))
        h, ends, at = torch.empty_like(u), [], 0
        if case["train"]:
            dy = flat(f["dy"])
            G, before, dh0 = torch.empty_like(u), torch.empty_like(u), []
        for k, length in enumerate(s["lens"]):
            at, sl = at + length, slice(at, at + length)
            init = u.new_zeros(D) if f["h0"] is None else f["h0"][k]
            h[sl] = walk(a[sl], u[sl], init)
            ends.append(h[sl][-1] if length else init)
            if not case["train"]:
                continue
            last = torch.zeros_like(init) if f["dht"] is None else f["dht"][k]
            if not length:
                dh0.append(last)
                continue
            before[sl] = torch.cat([init.unsqueeze(0), h[sl][:-1]])
            a_next = torch.cat([a[sl][1:], a.new_ones(1, D)])
            # the adjoint runs from the end: G_t = dy_t act(z_t) + a_{t+1} G_{t+1}
            G[sl] = torch.flip(walk(torch.flip(a_next, [0]), torch.flip((dy * value)[sl], [0]), last), [0])
            dh0.append(a[sl][0] * G[sl][0])
        out = {"y": (h * value).view(f["x"].shape)}
        if case["state"]:
            out["state"] = torch.stack(ends)
        if case["train"]:
            shaped = lambda t: t.view(f["x"].shape)  # noqa: E731
            dlog = G * a * before
            if case["normalize"]:  # d m / d log a = -a^2 / m
                dlog = dlog - G * si * x * a * a / m
            out.update({"dx": shaped(G * m * si), "ddecay_gate": shaped(dlog * f["A"] * sr * (1 - sr)),
                        "dA": (dlog * sr).sum(0)})
            if f["input_gate"] is not None:
                out["dinput_gate"] = shaped(G * m * x * si * (1 - si))
            if f["gate"] is not None:
                out["dgate"] = shaped(dy * h * slope)
            if case["state"]:
                out["dh0"] = torch.stack(dh0)
        return out
