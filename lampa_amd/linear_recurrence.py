"""The gated linear recurrence of a recurrent mixer, for prompts and for single tokens, on the GPU.

For every sequence and channel, with a state h in float32::

    a_t = exp(A sigmoid(decay_gate_t))
    h_t = a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(input_gate_t) x_t          y_t = act(gate_t) h_t

``gated_recurrence`` runs it over whole sequences (dense or packed) and is differentiable; ``gated_recurrence_step`` runs one
token for each sequence on a kept state. It is the per-channel counterpart of ``state_space_scan`` (the mixers it stands beside:
``models/baselines/full_mamba2.py:221-430``) and follows its names, state handling and return tuples. GPU tensors only; there is
no CPU path.
"""
import functools
import struct
import weakref
from typing import Optional

import torch
from torch.autograd.graph import increment_version

from . import _capi
from ._capi import check, ptr, stream_of
from .gated_delta import _direct
from .layer_ops import _ACT, _DTYPES, _on_device, _plain_f32, _same_device, _sequences, _wants_grad

MAX_CHANNELS = 1 << 20
MAX_STRIDE = 1 << 20  # elements between tokens: the kernels form offsets inside a tile in 32 bits

# lampa_lr_args: 19 pointers, 7 int64, 6 int32
_ARGS = struct.Struct("=19Q7q6i")


def _rows(t, D):
    """(t, elements between tokens) of t [B, T, D] as the kernels read it; a copy where tokens do not lie evenly or lie too far
    apart (a token of each of several long sequences)."""
    if t is None:
        return None, D
    B, T, _ = t.shape
    sb, step, inner = t.stride()
    if T == 1:
        step = sb if B > 1 else D
    if (inner == 1 or D == 1) and D <= step <= MAX_STRIDE and (B == 1 or T == 1 or sb == T * step):
        return t, step
    return torch.empty((B, T, D), dtype=t.dtype, device=t.device).copy_(t.detach()), D


@functools.lru_cache(maxsize=4096)
def _sizes(B, T, D, n_seq, packed, dtype, backward):
    """(tiles, bytes of a pass's workspace) of a call."""
    args = _ARGS.pack(*(0,) * 9, int(packed), *(0,) * 9, 0, B * T, T, D, D, D, D, n_seq, D, dtype, 0, 0, 0)
    lib = _capi.lib()
    return check(lib.lampa_lr_slots(args), "lampa_lr_slots"), check(lib.lampa_lr_workspace_bytes(args, backward), "lampa_lr_workspace_bytes")


def _pack(x, r, i, z, A, h0, y, ht, tiles, cu, grads, ws, size, act, normalize, n_seq):
    (x, xs), (r, rs), (i, is_), (z, zs) = x, r, i, z
    B, T, D = x.shape
    pointers = [0 if t is None else t.data_ptr() for t in (x, r, i, z, A, h0, y, ht, tiles, cu, *grads, ws)]
    return _ARGS.pack(*pointers, size, B * T, T, xs, rs, is_, zs, n_seq, D, _DTYPES[x.dtype], act, int(normalize), 0)


_NO_GRADS = (None,) * 8


def _scan_launch(x, r, A, i, z, act, normalize, h0, want_final, cu, keep=False):
    """(y, final state or None, what the gradients need beside the inputs: the states before each tile)."""
    B, T, D = x.shape
    n_seq = B if cu is None else cu.numel() - 1
    dev = x.device
    slots, size = _sizes(B, T, D, n_seq, cu is not None, _DTYPES[x.dtype], 0)
    y = torch.empty((B, T, D), dtype=x.dtype, device=dev)
    ht = torch.empty((n_seq, D), dtype=torch.float32, device=dev) if want_final else None
    tiles = torch.empty((slots, D), dtype=torch.float32, device=dev) if keep else None
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    held = _rows(x, D), _rows(r, D), _rows(i, D), _rows(z, D), _plain_f32(A), _plain_f32(h0)  # copies among them live until the launch
    args = _pack(*held, y, ht, tiles, cu, _NO_GRADS, ws, size, act, normalize, n_seq)
    with _on_device(dev.index):
        check(_capi.lib().lampa_lr_scan_fwd(args, stream_of(y)), "lampa_lr_scan_fwd")
    return y, ht, tiles


def _scan_backward(x, r, A, i, z, act, normalize, h0, cu, tiles, dy, dht):
    B, T, D = x.shape
    n_seq = B if cu is None else cu.numel() - 1
    dev = x.device
    _, size = _sizes(B, T, D, n_seq, cu is not None, _DTYPES[x.dtype], 1)
    h0 = _plain_f32(h0)
    if dy is None:
        dy = torch.zeros((B, T, D), dtype=x.dtype, device=dev)
    elif dy.dtype != x.dtype or not dy.is_contiguous():
        dy = dy.to(x.dtype).contiguous()
    dx, dr = torch.empty_like(dy), torch.empty_like(dy)
    di = None if i is None else torch.empty_like(dy)
    dz = None if z is None else torch.empty_like(dy)
    dA = torch.empty(D, dtype=torch.float32, device=dev)
    dh0 = None if h0 is None else torch.empty((n_seq, D), dtype=torch.float32, device=dev)
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    dht = _plain_f32(dht)
    held = _rows(x, D), _rows(r, D), _rows(i, D), _rows(z, D), _plain_f32(A), h0  # copies among them live until the launch
    args = _pack(*held, None, None, tiles, cu, (dy, dht, dx, dr, di, dz, dA, dh0), ws, size, act, normalize, n_seq)
    with _on_device(dev.index):
        check(_capi.lib().lampa_lr_scan_bwd(args, stream_of(dx)), "lampa_lr_scan_bwd")
    return dx, dr, dA, di, dz, dh0


class _GatedRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, r, A, i, z, h0, act, normalize, want_final, cu, keep):
        ctx.set_materialize_grads(False)
        y, ht, tiles = _scan_launch(x, r, A, i, z, act, normalize, h0, want_final, cu, keep)
        if keep:
            ctx.save_for_backward(x, r, A, i, z, h0, cu, tiles)
        # The gradients do not read the final state, but one through it would be that of the state as it was returned: a state that has
        # been moved on in place is noticed as long as somebody holds it.
        ctx.final = (weakref.ref(ht), ht._version) if keep and want_final else None
        ctx.act, ctx.normalize = act, normalize
        return y, ht

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dht):
        x, r, A, i, z, h0, cu, tiles = ctx.saved_tensors
        final = None if ctx.final is None else ctx.final[0]()
        if final is not None and final._version != ctx.final[1]:
            raise RuntimeError("gated_recurrence: the final state has been modified by an inplace operation (a step that moved it "
                               "on) before the gradients of the call that returned it; give gated_recurrence_step a new_state")
        dx, dr, dA, di, dz, dh0 = _scan_backward(x, r, A, i, z, ctx.act, ctx.normalize, h0, cu, tiles, dy, dht)
        if A.dtype != torch.float32:
            dA = dA.to(A.dtype)
        if h0 is not None and h0.dtype != torch.float32:
            dh0 = dh0.to(h0.dtype)
        return dx, dr, dA, di, dz, dh0, None, None, None, None, None


def _check_operands(what, x, decay_gate, A, input_gate, gate, gate_activation, dims):
    if gate_activation not in _ACT:
        raise ValueError(f"Activation `{gate_activation}` not supported yet.")
    if gate_activation is not None and gate is None:
        raise ValueError(f"{what}: gate_activation without a gate")
    if x.dim() != dims or x.shape[-1] < 1 or x.shape[-1] > MAX_CHANNELS:
        raise ValueError(f"{what}: expected x [{'B, T, ' if dims == 3 else 'n, '}D] with D in 1 .. {MAX_CHANNELS}, got {tuple(x.shape)}")
    if x.dtype not in _DTYPES:
        raise TypeError(f"{what}: x must be bfloat16, float16 or float32, got {x.dtype}")
    for name, t in (("decay_gate", decay_gate), ("input_gate", input_gate), ("gate", gate)):
        if t is not None and t.shape != x.shape:
            raise ValueError(f"{what}: {name} must have x's shape {tuple(x.shape)}, got {tuple(t.shape)}")
        if t is not None and t.dtype != x.dtype:
            raise TypeError(f"{what}: {name} must have x's type ({x.dtype}), got {t.dtype}")
    if tuple(A.shape) != (x.shape[-1],):
        raise ValueError(f"{what}: A must have shape ({x.shape[-1]},), one value per channel, got {tuple(A.shape)}")
    if not A.is_floating_point():
        raise TypeError(f"{what}: A must be a floating-point tensor, got {A.dtype}")


def gated_recurrence(x: torch.Tensor, decay_gate: torch.Tensor, A: torch.Tensor, input_gate: Optional[torch.Tensor] = None,
                     gate: Optional[torch.Tensor] = None, gate_activation: Optional[str] = None, normalize: bool = True,
                     initial_state: Optional[torch.Tensor] = None, output_final_state: bool = False,
                     cu_seqlens: Optional[torch.Tensor] = None):
    """x, decay_gate, input_gate, gate [B, T, D] of one type (they may be column slices of wider tensors); A [D], the log of what a
    token with an open decay gate keeps: at most 0 (above 0 the normalised recurrence is NaN; without ``normalize`` it grows, and past
    float32's range within a sequence it may be NaN where the recurrence, on zeros, is not).
    ``input_gate`` None: a factor of 1; ``gate`` None: y = h; ``gate_activation`` ``None`` / ``'sigmoid'`` / ``'silu'`` /
    ``'swish'``; ``normalize=False`` leaves the factor sqrt(1 - a^2) out. Any D up to 2^20. Returns (y [B, T, D] in x's type,
    final state [sequences, D] float32 or None).

    With ``cu_seqlens`` [sequences + 1] B must be 1 and the sequences lie one after the other: it starts at 0, never decreases
    and ends at T. A tensor on the host is checked; one on the GPU is not read by the host (so a call can be captured in a
    graph): boundaries outside the tokens are moved inside, none lies before an earlier one, and tokens behind the last boundary
    come back as zero (their gradients too, whatever they hold).

    A value that is not finite reaches its channel's tokens from its own on, as in the recurrence, never earlier ones; in
    gradients of a sequence it may reach every token of its channel. Differentiable in every floating-point input (first order);
    repeated calls give the same bits. Where a token's log decay is 0 in float32 (A is 0, or its gate's sigmoid is) the slope
    through sqrt(1 - a^2) is taken as 0. The backward raises where the final state it returned has been moved on in place since: use
    ``gated_recurrence_step(..., new_state=)`` until then."""
    what = "gated_recurrence"
    _same_device(what, x, decay_gate, A, input_gate, gate, initial_state)
    _check_operands(what, x, decay_gate, A, input_gate, gate, gate_activation, 3)
    cu = _sequences(what, cu_seqlens, x.shape[0], x.shape[1], x.device)
    n_seq = x.shape[0] if cu is None else cu.numel() - 1
    if n_seq < 1:
        raise ValueError(f"{what}: the batch must hold at least one sequence")
    if initial_state is not None:
        if tuple(initial_state.shape) != (n_seq, x.shape[-1]):
            raise ValueError(f"{what}: initial_state must have shape {(n_seq, x.shape[-1])} ([sequences, D]), got "
                             f"{tuple(initial_state.shape)}")
        if not initial_state.is_floating_point():
            raise TypeError(f"{what}: initial_state must be a floating-point tensor, got {initial_state.dtype}")
    act, want = _ACT[gate_activation], bool(output_final_state)
    if _direct(x, decay_gate, A, input_gate, gate, initial_state):
        y, ht, _ = _scan_launch(x, decay_gate, A, input_gate, gate, act, bool(normalize), initial_state, want, cu)
        return y, ht
    keep = _wants_grad(x, decay_gate, A, input_gate, gate, initial_state)
    return _GatedRecurrence.apply(x, decay_gate, A, input_gate, gate, initial_state, act, bool(normalize), want, cu, keep)


def _step_rows(t, D):
    """(t, elements between rows) of t [n, D] whose rows are contiguous."""
    if t is None:
        return None, D
    step, inner = t.stride()
    if t.shape[0] == 1:
        step = D
    return (t, step) if (inner == 1 or D == 1) and step >= D else (t.contiguous(), D)


def _step_launch(x, r, A, state, i, z, new_state, act, normalize):
    target = state if new_state is None else new_state
    increment_version(target)  # written through its pointer: a backward that saved it must notice
    n, D = x.shape
    (x, xs), (r, rs), (i, is_), (z, zs) = _step_rows(x, D), _step_rows(r, D), _step_rows(i, D), _step_rows(z, D)
    A = _plain_f32(A)
    y = torch.empty((n, D), dtype=x.dtype, device=x.device)
    with _on_device(x.get_device()):
        check(_capi.lib().lampa_lr_step(ptr(x), xs, ptr(r), rs, ptr(i), is_, ptr(z), zs, ptr(A), ptr(state), ptr(target), ptr(y), n, D,
                                        _DTYPES[x.dtype], act, int(normalize), stream_of(y)), "lampa_lr_step")
    return y


class _Step(torch.autograd.Function):
    """A step in a graph: traced, or never differentiated (the backward raises)."""

    @staticmethod
    def forward(ctx, *args):
        return _step_launch(*args)

    @staticmethod
    def backward(ctx, dy):
        raise NotImplementedError("lampa_amd implements the forward pass of this operator only")


def gated_recurrence_step(x: torch.Tensor, decay_gate: torch.Tensor, A: torch.Tensor, state: torch.Tensor,
                          input_gate: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                          gate_activation: Optional[str] = None, normalize: bool = True,
                          new_state: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token for each of n sequences on top of ``state`` [n, D] (float32, contiguous): x and the gates [n, D], everything else
    as in ``gated_recurrence``. Returns y [n, D] in x's type. ``state`` is moved on in place, or, with ``new_state`` (same shape, no
    shared memory), left as it is and the next state written there. Forward only: the backward raises."""
    what = "gated_recurrence_step"
    _same_device(what, x, decay_gate, A, state, input_gate, gate, new_state)
    _check_operands(what, x, decay_gate, A, input_gate, gate, gate_activation, 2)
    for name, t in (("state", state), ("new_state", new_state)):
        if t is None:
            continue
        if tuple(t.shape) != tuple(x.shape):
            raise ValueError(f"{what}: {name} must have shape {tuple(x.shape)} ([n, D]), got {tuple(t.shape)}")
        if t.dtype != torch.float32 or not t.is_contiguous():
            raise ValueError(f"{what}: {name} must be float32 and contiguous, as it is read or written in place")
    if new_state is not None and new_state is not state:
        a, b, size = state.data_ptr(), new_state.data_ptr(), state.numel() * 4
        if a != b and a < b + size and b < a + size:
            raise ValueError(f"{what}: new_state overlaps state")
    if x.shape[0] == 0:
        return torch.empty_like(x)
    args = x, decay_gate, A, state, input_gate, gate, new_state, _ACT[gate_activation], bool(normalize)
    # a traced call has to be in the graph as a function; asking `_direct` takes a microsecond of a step's 13
    if _wants_grad(x, decay_gate, A, input_gate, gate, state) or torch._C._get_tracing_state() is not None:
        return _Step.apply(*args)
    return _step_launch(*args)
