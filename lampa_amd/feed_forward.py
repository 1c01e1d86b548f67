"""The gated feed-forward block behind a mixer, on the GPU::

    y = (act(x w_gate^T) * (x w_up^T)) w_down^T

``gated_feed_forward`` is the operator of the reference's ``GatedMLP`` (``models/hattention/modeling_gated_deltaproduct.py:310-324``)
with its gradients; the layer is ``lampa_amd.block.GatedFeedForward``. GPU tensors only; there is no CPU path.
"""
import functools
import struct
from typing import Optional

import torch

from . import _capi
from ._capi import check, stream_of
from .gated_delta import _direct
from .layer_ops import _ACT, _DTYPES, _on_device, _packed, _same_device, _wants_grad

MAX_WIDTH = 1 << 17   # of D and F
MAX_STRIDE = 1 << 20  # elements between rows of x: offsets inside a tile are formed in 32 bits

# lampa_ff_args: 11 pointers, 3 int64, 4 int32
_ARGS = struct.Struct("=11Q3q4i")


def _matrix(x):
    """x [..., D] as (rows, elements between them): itself where its rows lie evenly, 16-byte aligned and not too far apart, else a copy."""
    D = x.shape[-1]
    if x.dim() == 2 and x.is_contiguous() and x.data_ptr() % 16 == 0:
        return x, D
    x2 = x.detach().reshape(-1, D)
    step = x2.stride(0) if x2.shape[0] > 1 else D
    if x2.stride(1) != 1 or step < D or step % 8 or step > MAX_STRIDE or x2.data_ptr() % 16:
        x2, step = torch.empty(x2.shape, dtype=x2.dtype, device=x2.device).copy_(x2), D
    return x2, step


@functools.lru_cache(maxsize=4096)
def _workspace(rows, D, F, dtype, backward, wanted):
    """Bytes of a pass's workspace; ``wanted``: the gradients of x, w_gate, w_up and w_down that are asked for."""
    args = _ARGS.pack(0, 0, 0, 0, 0, 0, *wanted, 0, 0, rows, D, D, F, dtype, 0)
    return check(_capi.lib().lampa_ff_workspace_bytes(args, backward), "lampa_ff_workspace_bytes")


def _launch(call, name, x, w_gate, w_up, w_down, act, y, dy, grads):
    x2, step = _matrix(x)
    rows, D = x2.shape
    F, code, dev = w_gate.shape[0], _DTYPES[x.dtype], x.device
    w_gate, w_up, w_down = _packed(w_gate), _packed(w_up), _packed(w_down)
    grads = tuple([0 if g is None else g.data_ptr() for g in grads])
    size = _workspace(rows, D, F, code, int(dy is not None), tuple([int(g != 0) for g in grads]))
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    args = _ARGS.pack(x2.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), w_down.data_ptr(), 0 if y is None else y.data_ptr(),
                      0 if dy is None else dy.data_ptr(), *grads, ws.data_ptr() if size else 0, size, rows, step, D, F, code, act)
    with _on_device(dev.index):
        check(call(args, stream_of(x)), name)


_NO_GRADS = (None,) * 4


def _forward(x, w_gate, w_up, w_down, act):
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    _launch(_capi.lib().lampa_ff_fwd, "lampa_ff_fwd", x, w_gate, w_up, w_down, act, y, None, _NO_GRADS)
    return y


class _GatedFeedForward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, act):
        ctx.save_for_backward(x, w_gate, w_up, w_down)
        ctx.act = act
        return _forward(x, w_gate, w_up, w_down, act)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        tensors = ctx.saved_tensors
        x = tensors[0]
        make = torch.empty if x.numel() else torch.zeros  # without rows nothing is launched
        grads = [make(t.shape, dtype=t.dtype, device=t.device) if need else None for t, need in zip(tensors, ctx.needs_input_grad)]
        if dy.dtype != x.dtype:
            dy = dy.to(x.dtype)
        _launch(_capi.lib().lampa_ff_bwd, "lampa_ff_bwd", *tensors, ctx.act, None, _packed(dy), grads)
        return (*grads, None)


def gated_feed_forward(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
                       activation: Optional[str] = "silu") -> torch.Tensor:
    """x [..., D] (rows may be column slices of a wider tensor); w_gate, w_up [F, D], w_down [D, F] of x's type (as ``nn.Linear``
    keeps them); ``activation`` of the gate ``None`` / ``'sigmoid'`` / ``'silu'`` / ``'swish'``. D and F multiples of 8, up to
    2^17. Returns [..., D] in x's type.

    Products have fp32 sums; for 16-bit types the hidden values act(.) * (.) (and, in the gradients, theirs) are rounded to the type
    as the next product's operands (in float16 a hidden value past its range is infinite), which makes an output's error about 1.4
    times its own rounding. With few rows what that rounding leaves is kept as well, and the error is the output's rounding alone: for
    D <= 128 up to 32 768 rows (the weights' gradients up to 4 096), else up to 64. A row's last bits thus depend on how many rows a call
    has. Where an operand is infinite, what the formula makes infinite may be NaN. Differentiable in every tensor (first
    order; the gradients compute the hidden values again, so nothing but the inputs is kept; repeated calls give the same bits)."""
    what = "gated_feed_forward"
    _same_device(what, x, w_gate, w_up, w_down)
    if activation not in _ACT:
        raise ValueError(f"Activation `{activation}` not supported yet.")
    if x.dim() < 1 or w_gate.dim() != 2 or w_gate.shape != w_up.shape or w_gate.shape[1] != x.shape[-1] or \
            tuple(w_down.shape) != (w_gate.shape[1], w_gate.shape[0]):
        raise ValueError(f"{what}: expected x [..., D], w_gate and w_up [F, D] and w_down [D, F], got {tuple(x.shape)}, "
                         f"{tuple(w_gate.shape)}, {tuple(w_up.shape)} and {tuple(w_down.shape)}")
    F, D = w_gate.shape
    if D < 8 or F < 8 or D % 8 or F % 8 or D > MAX_WIDTH or F > MAX_WIDTH:
        raise ValueError(f"{what}: D and F must be multiples of 8 up to {MAX_WIDTH}, got {D} and {F}")
    if x.dtype not in _DTYPES or any(t.dtype != x.dtype for t in (w_gate, w_up, w_down)):
        raise TypeError(f"{what}: x and the weights must have one type (bfloat16, float16 or float32), got {x.dtype}, {w_gate.dtype}, "
                        f"{w_up.dtype} and {w_down.dtype}")
    act = _ACT[activation]
    if _direct(x) and not _wants_grad(w_gate, w_up, w_down):  # a module's weights without gradients too
        return _forward(x, w_gate, w_up, w_down, act)
    return _GatedFeedForward.apply(x, w_gate, w_up, w_down, act)
