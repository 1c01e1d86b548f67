"""A gated-delta layer and the `lshgd`-style block built from this package's operators.

``GatedDeltaLayer`` follows ``GatedDeltaProduct`` with one householder step (``models/hattention/
modeling_gated_deltaproduct.py:317-625``): q/k/v projections -> short convolution + SiLU -> l2-normalised chunkwise
gated-delta forward with decay g = -exp(A_log) softplus(a + dt_bias) and write strength beta = sigmoid(b) -> RMS norm
gated by swish(g_proj(x)) -> output projection. ``LshgdBlock`` is the benchmark block: input linear, LSH bucket sort of
the hits, pre-norm residual layers (the fused add + norm of ``GatedDeltaProductBlock.forward``, ``:1029-1056``), unsort
and an embedding head. The projections are plain library GEMMs (one fused GEMM per layer for q|k|v|g|b|a); everything
else runs in this package's HIP kernels. Forward only.

``StateSpaceLayer`` and ``StateSpaceBlock`` are the state-space counterpart (the mixer and residual wiring behind
``models/baselines/full_mamba2.py:221-430``): projection -> short convolution + SiLU -> selective scan -> gated norm -> output
projection, with the norms at the borders fused with the residual add. They train (every operator has its gradients), take
packed sequences, and continue from caches with whole prompts or one token at a time.

``GatedRecurrentLayer``, ``GatedFeedForward`` and ``GatedRecurrentBlock`` are a block of a mixer with a per-channel recurrence and a
gated feed-forward block behind each mixer (the wiring of ``GatedDeltaProductBlock``, ``modeling_gated_deltaproduct.py:995-1056``,
whose second half is the reference's ``GatedMLP``, ``:310-324``), trained, prefilled and stepped in the same way.
"""
import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import lsh
from .feed_forward import gated_feed_forward
from .gated_delta import chunk_gated_delta_rule
from .layer_ops import (PROJ_CONV_HIDDEN, FusedRMSNormSwishGate, RMSNorm, ShortConvolution, _sequences, causal_conv1d,
                        causal_conv1d_split, causal_conv1d_step, gdr_gates, norm_proj, norm_proj_supported, proj_conv, residual_norm)
from .linear_recurrence import gated_recurrence, gated_recurrence_step
from .state_space import state_space_scan, state_space_step


class GatedDeltaLayer(nn.Module):
    def __init__(self, hidden_size: int = 128, head_dim: int = 64, num_heads: int = 8, expand_v: float = 1,
                 conv_size: int = 4, norm_eps: float = 1e-6, allow_neg_eigval: bool = False):
        super().__init__()
        self.hidden_size, self.head_dim, self.num_heads = hidden_size, head_dim, num_heads
        self.key_dim = num_heads * head_dim
        self.value_dim = int(self.key_dim * expand_v)
        self.head_v_dim = int(head_dim * expand_v)
        self.allow_neg_eigval = allow_neg_eigval
        self.q_proj = nn.Linear(hidden_size, self.key_dim, bias=False)
        self.k_proj = nn.Linear(hidden_size, self.key_dim, bias=False)
        self.v_proj = nn.Linear(hidden_size, self.value_dim, bias=False)
        self.g_proj = nn.Linear(hidden_size, self.value_dim, bias=False)
        self.b_proj = nn.Linear(hidden_size, num_heads, bias=False)
        self.a_proj = nn.Linear(hidden_size, num_heads, bias=False)
        self.q_conv1d = ShortConvolution(self.key_dim, conv_size, activation="silu")
        self.k_conv1d = ShortConvolution(self.key_dim, conv_size, activation="silu")
        self.v_conv1d = ShortConvolution(self.value_dim, conv_size, activation="silu")
        # decay parameters as in modeling_gated_deltaproduct.py:420-437
        A = torch.empty(num_heads, dtype=torch.float32).uniform_(0, 16)
        self.A_log = nn.Parameter(torch.log(A))
        dt = torch.exp(torch.rand(num_heads) * (math.log(0.1) - math.log(0.001)) + math.log(0.001)).clamp(min=1e-4)
        self.dt_bias = nn.Parameter(dt + torch.log(-torch.expm1(-dt)))
        self.o_norm = FusedRMSNormSwishGate(self.head_v_dim, eps=norm_eps)
        self.o_proj = nn.Linear(self.value_dim, hidden_size, bias=False)
        self._fused = None

    def _fused_weight(self):
        parts = (self.q_proj.weight, self.k_proj.weight, self.v_proj.weight, self.g_proj.weight, self.b_proj.weight,
                 self.a_proj.weight)
        key = tuple((p.data_ptr(), p._version, p.dtype) for p in parts)
        if self._fused is None or self._fused[0] != key:
            self._fused = (key, torch.cat([p.detach() for p in parts], dim=0).contiguous())
        return self._fused[1]

    @torch.no_grad()
    def forward(self, hidden_states: torch.Tensor, cu_seqlens=None, initial_state=None, output_final_state=False,
                residual=None, next_norm=None):
        """hidden_states [B, T, hidden] -> (o [B, T, hidden], final_state or None). With ``residual`` and ``next_norm``
        (an ``RMSNorm``) the layer also applies the residual add and that norm and returns
        ((next_norm(o + residual), o + residual), final_state): the pre-norm wiring of a stack of layers, fused into
        the output projection kernel when the shapes allow it."""
        B, T, _ = hidden_states.shape
        H, dk, dv, kd, vd = self.num_heads, self.head_dim, self.head_v_dim, self.key_dim, self.value_dim
        convs = (self.q_conv1d, self.k_conv1d, self.v_conv1d)
        fused = (cu_seqlens is None and hidden_states.dtype == torch.bfloat16 and self.hidden_size == PROJ_CONV_HIDDEN
                 and kd == vd and kd % 256 == 0 and (2 * H) % 8 == 0)
        if fused:  # projections, convolutions and SiLU in one kernel: the projection output never reaches memory
            (q, k, v), xg, xba = proj_conv(hidden_states, self._fused_weight(), [c.weight for c in convs],
                                           [c.bias for c in convs], kd, vd)
            xb, xa = xba[..., :H], xba[..., H:]
        else:
            proj = F.linear(hidden_states, self._fused_weight())                 # [B, T, 2 kd + 2 vd + 2 H]
            cols = [0, kd, 2 * kd, 2 * kd + vd, 2 * kd + 2 * vd, 2 * kd + 2 * vd + H, 2 * kd + 2 * vd + 2 * H]
            xq, xk, xv, xg, xb, xa = (proj[..., cols[i]:cols[i + 1]] for i in range(6))
            if kd == vd:                                                         # one launch over the q | k | v columns
                q, k, v = causal_conv1d_split(proj[..., :cols[3]], [c.weight for c in convs], [c.bias for c in convs],
                                              "silu", cu_seqlens)
            else:
                q, k, v = (causal_conv1d(t, c.weight.reshape(t.shape[-1], -1), c.bias, None, "silu", cu_seqlens)
                           for t, c in zip((xq, xk, xv), convs))
        g, beta = gdr_gates(xa, xb, self.A_log, self.dt_bias, 2.0 if self.allow_neg_eigval else 1.0)
        o, state = chunk_gated_delta_rule(q.view(B, T, H, dk), k.view(B, T, H, dk), v.view(B, T, H, dv), g, beta,
                                          initial_state=initial_state, output_final_state=output_final_state,
                                          cu_seqlens=cu_seqlens, use_qk_l2norm_in_kernel=True)
        gate = xg.unflatten(-1, (H, dv))
        if norm_proj_supported(o, self.hidden_size) and self.o_proj.weight.dtype == torch.bfloat16:  # norm + gate + GEMM
            if residual is not None and residual.dtype == torch.bfloat16 and next_norm.bias is None:
                return norm_proj(o, gate, self.o_norm.weight, self.o_proj.weight, self.o_norm.eps, residual=residual,
                                 next_norm_weight=next_norm.weight, next_eps=next_norm.eps), state
            out = norm_proj(o, gate, self.o_norm.weight, self.o_proj.weight, self.o_norm.eps)
        else:
            out = self.o_proj(self.o_norm(o, gate).reshape(B, T, vd))
        return (out if residual is None else next_norm(out, residual, True)), state


class LshgdBlock(nn.Module):
    """Input linear -> LSH bucket sort of the hits -> ``n_layers`` pre-norm residual gated-delta layers -> final norm ->
    unsort -> embedding head. Parameters are created under the caller's seed with torch's default Linear / Conv1d
    initialisation (Kaiming-uniform)."""

    def __init__(self, in_dim: int = 24, hidden: int = 128, n_layers: int = 4, num_heads: int = 8, head_dim: int = 64,
                 out_dim: int = 24, coord_dim: int = 4, n_tables: int = 3, n_proj: int = 4, bucket_width: float = 0.5,
                 lsh_seed: int = 1):
        super().__init__()
        self.input = nn.Linear(in_dim, hidden)
        self.norms = nn.ModuleList([RMSNorm(hidden, eps=1e-6) for _ in range(n_layers)])
        self.layers = nn.ModuleList([GatedDeltaLayer(hidden, head_dim, num_heads) for _ in range(n_layers)])
        self.norm_f = RMSNorm(hidden, eps=1e-6)
        self.head = nn.Linear(hidden, out_dim)
        self.n_tables, self.n_proj, self.bucket_width = n_tables, n_proj, bucket_width
        gen = torch.Generator().manual_seed(lsh_seed)
        alpha = torch.normal(0.0, 1.0, (coord_dim, n_tables * n_proj), generator=gen)
        beta = torch.rand(n_tables * n_proj, generator=gen) * bucket_width
        # kept as bit patterns so that module.to(bfloat16) leaves the float32 hash parameters alone
        self.register_buffer("lsh_alpha_bits", alpha.view(torch.int32))
        self.register_buffer("lsh_beta_bits", beta.view(torch.int32))
        self._flags_host = None  # pinned copy of the LSH stage's flag fields (one per table), made on first use

    @property
    def lsh_alpha(self) -> torch.Tensor:
        return self.lsh_alpha_bits.view(torch.float32)

    @property
    def lsh_beta(self) -> torch.Tensor:
        return self.lsh_beta_bits.view(torch.float32)

    @torch.no_grad()
    def order(self, coords: torch.Tensor, check: bool = True):
        """Sequence order of the hits: the stable bucket-sort permutation of the first hash table (int32 [N]).
        ``check=True`` reads the flag field of the stage at once (one host synchronisation): when a workgroup of the
        one-launch kernel gave up a wait (``lsh.META_GAVE_UP``) the stage runs again as separate kernels, which wait for
        nothing; a key that does not fit 32 bits raises. ``check=False`` returns ``(perm, pending)`` instead and leaves
        the flags to ``_flags_of(pending)``: they are copied to pinned host memory behind the kernel, so that the caller
        can queue its other launches first and look at them without draining the stream."""
        args = (coords.float(), self.lsh_alpha, self.lsh_beta, self.bucket_width, self.n_tables, self.n_proj)
        out = lsh.lsh_bucket_sort(*args, return_ids=False)
        if not check:
            if self._flags_host is None:
                self._flags_host = torch.empty(self.n_tables, dtype=torch.int32, pin_memory=True)
            self._flags_host.copy_(out["meta"][..., -1], non_blocking=True)
            done = torch.cuda.Event()
            done.record()
            return out["perm"][0], done
        flags = lsh.decode_meta_flags(out["meta"])
        if bool(flags["gave_up"].any()):
            return self._order_with_separate_kernels(args)
        if bool(flags["key_overflow"][0]):
            raise lsh.LampaError("LshgdBlock: the bucket key of the first hash table does not fit 32 bits; the "
                                 "sequence order would be meaningless")
        return out["perm"][0]

    def _order_with_separate_kernels(self, args):
        lsh.one_launch_config(enabled=False)
        try:
            return lsh.lsh_bucket_sort(*args, return_ids=False, strict=True)["perm"][0]
        finally:
            lsh.one_launch_config(enabled=True)

    def _flags_of(self, done) -> int:
        """The flag fields of the last ``order(check=False)`` call, OR-ed over the tables (waits for that kernel only)."""
        done.synchronize()
        flags = 0
        for f in self._flags_host.tolist():
            flags |= f
        return flags

    @torch.no_grad()
    def forward(self, feats: torch.Tensor, coords: torch.Tensor, perm: torch.Tensor = None) -> torch.Tensor:
        """feats [N, in_dim], coords [N, coord_dim] -> [N, out_dim] in the parameters' dtype, in the input hit order.
        The LSH stage's flag field is looked at once per event, after every launch of the block has been queued: a
        one-launch kernel that gave up a wait (its permutation is then all -1) makes the block run again with the order
        from the separate kernels; a key overflow raises."""
        dtype = self.input.weight.dtype
        pending = None
        if perm is None:
            perm, pending = self.order(coords, check=False)
        x = self.input(feats.to(dtype))
        x = lsh.gather_rows(x[None], perm[None])                                 # [1, N, hidden], LSH order
        h, residual = self.norms[0](x, None, True)                               # residual = x, h = norm(x)
        for i, layer in enumerate(self.layers):                                  # residual <- out + residual; h = next norm
            next_norm = self.norms[i + 1] if i + 1 < len(self.layers) else self.norm_f
            (h, residual), _ = layer(h, residual=residual, next_norm=next_norm)
        h = lsh.scatter_rows(h, perm[None])[0]                                   # back to the input order
        out = self.head(h)
        if pending is not None:
            flags = self._flags_of(pending)
            if flags & lsh.META_GAVE_UP:
                args = (coords.float(), self.lsh_alpha, self.lsh_beta, self.bucket_width, self.n_tables, self.n_proj)
                return self.forward(feats, coords, perm=self._order_with_separate_kernels(args))
            if self._flags_host[0].item() & lsh.META_KEY_OVERFLOW:
                raise lsh.LampaError("LshgdBlock: the bucket key of the first hash table does not fit 32 bits; the "
                                     "sequence order would be meaningless")
        return out


class StateSpaceLayer(nn.Module):
    """in_proj -> z | x | B | C | dt; causal convolution + SiLU over x | B | C; selective scan with delta = softplus(dt + dt_bias),
    A = -exp(A_log) and the skip D; rms norm of silu(z) * y; out_proj. ``expand * hidden_size`` columns in heads of ``head_dim``,
    B and C shared by the heads of a group."""

    def __init__(self, hidden_size: int = 128, d_state: int = 64, head_dim: int = 64, expand: int = 2, n_groups: int = 1,
                 conv_size: int = 4, norm_eps: float = 1e-5):
        super().__init__()
        inner = expand * hidden_size
        if inner % head_dim or (inner // head_dim) % n_groups:
            raise ValueError(f"StateSpaceLayer: {inner} columns do not divide into heads of {head_dim} and {n_groups} groups")
        self.hidden_size, self.d_state, self.head_dim, self.n_groups = hidden_size, d_state, head_dim, n_groups
        self.inner, self.num_heads, self.conv_size, self.norm_eps = inner, inner // head_dim, conv_size, norm_eps
        self.conv_dim = inner + 2 * n_groups * d_state
        self.in_proj = nn.Linear(hidden_size, inner + self.conv_dim + self.num_heads, bias=False)
        bound = conv_size ** -0.5
        self.conv_weight = nn.Parameter(torch.empty(self.conv_dim, conv_size).uniform_(-bound, bound))
        self.conv_bias = nn.Parameter(torch.empty(self.conv_dim).uniform_(-bound, bound))
        self.A_log = nn.Parameter(torch.log(torch.empty(self.num_heads).uniform_(1, 16)))
        step = torch.exp(torch.rand(self.num_heads) * (math.log(0.1) - math.log(0.001)) + math.log(0.001)).clamp(min=1e-4)
        self.dt_bias = nn.Parameter(step + torch.log(-torch.expm1(-step)))
        self.D = nn.Parameter(torch.ones(self.num_heads))
        self.norm_weight = nn.Parameter(torch.ones(inner))
        self.out_proj = nn.Linear(inner, hidden_size, bias=False)

    def _split(self, hidden):
        return self.in_proj(hidden).split([self.inner, self.conv_dim, self.num_heads], dim=-1)

    def _heads(self, xbc):
        gn = self.n_groups * self.d_state
        x, B, C = xbc.split([self.inner, gn, gn], dim=-1)
        return x.unflatten(-1, (self.num_heads, self.head_dim)), *(t.unflatten(-1, (self.n_groups, self.d_state)) for t in (B, C))

    def _out(self, y, z):
        return self.out_proj(residual_norm(y.flatten(-2), None, self.norm_weight, gate=z, gate_activation="silu", eps=self.norm_eps))

    def forward(self, hidden_states: torch.Tensor, cu_seqlens=None, cache=None, output_cache: bool = False):
        """hidden_states [B, T, hidden] -> (out [B, T, hidden], cache or None). ``cache`` = (the last inputs of the convolution
        [sequences, conv_dim, conv_size], the states [sequences, heads, d_state, head_dim] float32) as a call or ``step`` left
        them; no gradient runs through the convolution's part. ``cu_seqlens`` as ``state_space_scan`` takes it."""
        cu_seqlens = _sequences("StateSpaceLayer", cu_seqlens, *hidden_states.shape[:2], hidden_states.device)
        z, xbc, dt = self._split(hidden_states)
        conv_cache, state = (None, None) if cache is None else cache
        conv = causal_conv1d(xbc, self.conv_weight, self.conv_bias, activation="silu", cu_seqlens=cu_seqlens,
                             initial_state=conv_cache, output_final_state=output_cache)
        xbc, conv_cache = conv if output_cache else (conv, None)
        x, B, C = self._heads(xbc)
        y, state = state_space_scan(x, dt, -torch.exp(self.A_log.float()), B, C, D=self.D, dt_bias=self.dt_bias, dt_softplus=True,
                                    initial_state=state, output_final_state=output_cache, cu_seqlens=cu_seqlens)
        return self._out(y, z), (conv_cache, state) if output_cache else None

    @torch.no_grad()
    def step(self, hidden_states: torch.Tensor, cache):
        """One token for each sequence: hidden_states [sequences, hidden] -> [sequences, hidden]; the cache is moved on in place."""
        z, xbc, dt = self._split(hidden_states)
        xbc = causal_conv1d_step(xbc, cache[0], self.conv_weight, self.conv_bias, "silu")
        x, B, C = self._heads(xbc)
        y = state_space_step(x, dt, -torch.exp(self.A_log.float()), B, C, cache[1], D=self.D, dt_bias=self.dt_bias, dt_softplus=True)
        return self._out(y, z)


class StateSpaceBlock(nn.Module):
    """``n_layers`` pre-norm residual ``StateSpaceLayer``s and a final norm. The residual add, its learned scale
    (``residual_scale``: one value per channel and layer, starting at the given number) and the next norm are one operator;
    ``residual_in_fp32`` keeps the stream in float32 beside 16-bit layers."""

    def __init__(self, hidden_size: int = 128, n_layers: int = 4, residual_scale: float = None, residual_in_fp32: bool = True,
                 norm_eps: float = 1e-5, **layer_args):
        super().__init__()
        self.layers = nn.ModuleList([StateSpaceLayer(hidden_size, norm_eps=norm_eps, **layer_args) for _ in range(n_layers)])
        self.norm_weights = nn.ParameterList([nn.Parameter(torch.ones(hidden_size)) for _ in range(n_layers + 1)])
        self.scales = None if residual_scale is None else nn.ParameterList(
            [nn.Parameter(torch.full((hidden_size,), float(residual_scale))) for _ in range(n_layers)])
        self.residual_in_fp32, self.norm_eps = residual_in_fp32, norm_eps

    def _enter(self, x):
        h = residual_norm(x, None, self.norm_weights[0], eps=self.norm_eps)
        return h, x.float() if self.residual_in_fp32 else x

    def _border(self, i, out, residual):
        return residual_norm(out, residual, self.norm_weights[i + 1], residual_scale=None if self.scales is None else self.scales[i],
                             eps=self.norm_eps)

    def forward(self, x: torch.Tensor, cu_seqlens=None, caches=None, output_caches: bool = False):
        """x [B, T, hidden] -> (normed output [B, T, hidden], the layers' caches or None)."""
        cu_seqlens = _sequences("StateSpaceBlock", cu_seqlens, *x.shape[:2], x.device)
        h, residual = self._enter(x)
        new = []
        for i, layer in enumerate(self.layers):
            out, cache = layer(h, cu_seqlens, None if caches is None else caches[i], output_caches)
            new.append(cache)
            h, residual = self._border(i, out, residual)
        return h, new if output_caches else None

    @torch.no_grad()
    def step(self, x: torch.Tensor, caches):
        """One token for each sequence: x [sequences, hidden]; the caches are moved on in place."""
        h, residual = self._enter(x)
        for i, layer in enumerate(self.layers):
            h, residual = self._border(i, layer.step(h, caches[i]), residual)
        return h


class GatedFeedForward(nn.Module):
    """``GatedMLP`` (``modeling_gated_deltaproduct.py:310-324``): down_proj(act(gate_proj(x)) * up_proj(x)). Without
    ``intermediate_size`` it is two thirds of ``hidden_ratio * hidden_size``, rounded up to a multiple of 256."""

    def __init__(self, hidden_size: int = 128, hidden_ratio: float = 4, intermediate_size: int = None, activation: str = "silu"):
        super().__init__()
        if intermediate_size is None:
            intermediate_size = 256 * -(-int(hidden_size * hidden_ratio * 2 / 3) // 256)
        self.hidden_size, self.intermediate_size, self.activation = hidden_size, intermediate_size, activation
        self.gate_proj = nn.Linear(hidden_size, intermediate_size, bias=False)
        self.up_proj = nn.Linear(hidden_size, intermediate_size, bias=False)
        self.down_proj = nn.Linear(intermediate_size, hidden_size, bias=False)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        """x [..., hidden] -> [..., hidden]. Under autocast in its type, as the linear layers it stands for."""
        tensors = x, self.gate_proj.weight, self.up_proj.weight, self.down_proj.weight
        if torch.is_autocast_enabled("cuda"):
            dtype = torch.get_autocast_dtype("cuda")
            tensors = [t if t.dtype == torch.float64 else t.to(dtype) for t in tensors]
        return gated_feed_forward(*tensors, self.activation)


class GatedRecurrentLayer(nn.Module):
    """in_proj -> x | z; causal convolution + SiLU over x; decay and input gates from it; gated linear recurrence with
    A = -exp(A_log), its output gated by silu(z); out_proj. ``expand * hidden_size`` channels."""

    def __init__(self, hidden_size: int = 128, expand: int = 2, conv_size: int = 4):
        super().__init__()
        inner = expand * hidden_size
        self.hidden_size, self.inner, self.conv_size = hidden_size, inner, conv_size
        self.in_proj = nn.Linear(hidden_size, 2 * inner, bias=False)
        bound = conv_size ** -0.5
        self.conv_weight = nn.Parameter(torch.empty(inner, conv_size).uniform_(-bound, bound))
        self.conv_bias = nn.Parameter(torch.empty(inner).uniform_(-bound, bound))
        self.gate_proj = nn.Linear(inner, 2 * inner)
        # a token with an open decay gate keeps 0.9 .. 0.999 of the state
        self.A_log = nn.Parameter(torch.log(-torch.log(torch.empty(inner).uniform_(0.9, 0.999))))
        self.out_proj = nn.Linear(inner, hidden_size, bias=False)

    def _gates(self, x):
        return self.gate_proj(x).split([self.inner, self.inner], dim=-1)

    def forward(self, hidden_states: torch.Tensor, cu_seqlens=None, cache=None, output_cache: bool = False):
        """hidden_states [B, T, hidden] -> (out [B, T, hidden], cache or None). ``cache`` = (the last inputs of the convolution
        [sequences, inner, conv_size], the states [sequences, inner] float32) as a call or ``step`` left them; no gradient runs
        through the convolution's part. ``cu_seqlens`` as ``gated_recurrence`` takes it."""
        cu_seqlens = _sequences("GatedRecurrentLayer", cu_seqlens, *hidden_states.shape[:2], hidden_states.device)
        x, z = self.in_proj(hidden_states).split([self.inner, self.inner], dim=-1)
        conv_cache, state = (None, None) if cache is None else cache
        conv = causal_conv1d(x, self.conv_weight, self.conv_bias, activation="silu", cu_seqlens=cu_seqlens,
                             initial_state=conv_cache, output_final_state=output_cache)
        x, conv_cache = conv if output_cache else (conv, None)
        r, i = self._gates(x)
        y, state = gated_recurrence(x, r, -torch.exp(self.A_log.float()), input_gate=i, gate=z, gate_activation="silu",
                                    initial_state=state, output_final_state=output_cache, cu_seqlens=cu_seqlens)
        return self.out_proj(y), (conv_cache, state) if output_cache else None

    @torch.no_grad()
    def step(self, hidden_states: torch.Tensor, cache):
        """One token for each sequence: hidden_states [sequences, hidden] -> [sequences, hidden]; the cache is moved on in place."""
        x, z = self.in_proj(hidden_states).split([self.inner, self.inner], dim=-1)
        x = causal_conv1d_step(x, cache[0], self.conv_weight, self.conv_bias, "silu")
        r, i = self._gates(x)
        y = gated_recurrence_step(x, r, -torch.exp(self.A_log.float()), cache[1], input_gate=i, gate=z, gate_activation="silu")
        return self.out_proj(y)


class GatedRecurrentBlock(nn.Module):
    """``n_layers`` pre-norm residual pairs of a ``GatedRecurrentLayer`` and a ``GatedFeedForward``, and a final norm. The residual
    add and the next norm are one operator; ``residual_in_fp32`` keeps the stream in float32 beside 16-bit layers."""

    def __init__(self, hidden_size: int = 128, n_layers: int = 4, hidden_ratio: float = 4, intermediate_size: int = None,
                 residual_in_fp32: bool = True, norm_eps: float = 1e-5, **layer_args):
        super().__init__()
        self.layers = nn.ModuleList([GatedRecurrentLayer(hidden_size, **layer_args) for _ in range(n_layers)])
        self.feed_forward = nn.ModuleList([GatedFeedForward(hidden_size, hidden_ratio, intermediate_size) for _ in range(n_layers)])
        self.norm_weights = nn.ParameterList([nn.Parameter(torch.ones(hidden_size)) for _ in range(2 * n_layers + 1)])
        self.residual_in_fp32, self.norm_eps = residual_in_fp32, norm_eps

    def _run(self, x, mix):
        """x through all pairs; ``mix(i, h)`` is layer i's mixer."""
        h = residual_norm(x, None, self.norm_weights[0], eps=self.norm_eps)
        residual = x.float() if self.residual_in_fp32 else x
        for i, feed_forward in enumerate(self.feed_forward):
            h, residual = residual_norm(mix(i, h), residual, self.norm_weights[2 * i + 1], eps=self.norm_eps)
            h, residual = residual_norm(feed_forward(h), residual, self.norm_weights[2 * i + 2], eps=self.norm_eps)
        return h

    def forward(self, x: torch.Tensor, cu_seqlens=None, caches=None, output_caches: bool = False):
        """x [B, T, hidden] -> (normed output [B, T, hidden], the layers' caches or None)."""
        cu_seqlens = _sequences("GatedRecurrentBlock", cu_seqlens, *x.shape[:2], x.device)
        new = [None] * len(self.layers)

        def mix(i, h):
            out, new[i] = self.layers[i](h, cu_seqlens, None if caches is None else caches[i], output_caches)
            return out

        return self._run(x, mix), new if output_caches else None

    @torch.no_grad()
    def step(self, x: torch.Tensor, caches):
        """One token for each sequence: x [sequences, hidden]; the caches are moved on in place."""
        return self._run(x, lambda i, h: self.layers[i].step(h, caches[i]))
