"""The gated feed-forward block behind a mixer, on the GPU::

    y = (act(x w_gate^T) * (x w_up^T)) w_down^T

``gated_feed_forward`` is the operator of the reference's ``GatedMLP`` (``models/hattention/modeling_gated_deltaproduct.py:310-324``)
with its gradients; the layer is ``lampa_amd.block.GatedFeedForward``. GPU tensors only; there is no CPU path.
"""
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
    x2 = x.detach().reshape(-1, x.shape[-1])
    step = x2.stride(0) if x2.shape[0] > 1 else x2.shape[1]
    if (x2.shape[1] > 1 and x2.stride(1) != 1) or step < x2.shape[1] or step % 8 or step > MAX_STRIDE or x2.data_ptr() % 16:
        x2, step = torch.empty(x2.shape, dtype=x2.dtype, device=x2.device).copy_(x2), x2.shape[1]
    return x2, step


def _launch(name, backward, x, weights, act, y=None, dy=None, grads=(None,) * 4):
    x2, step = _matrix(x)
    rows, D = x2.shape
    p = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    w = [_packed(t.detach()) for t in weights]
    pack = lambda ws, size: _ARGS.pack(p(x2), *(p(t) for t in w), p(y), p(dy), *(p(t) for t in grads), p(ws), size, rows, step, D,  # noqa: E731
                                       w[0].shape[0], _DTYPES[x.dtype], act)
    lib = _capi.lib()
    with _on_device(x.get_device()):
        size = check(lib.lampa_ff_workspace_bytes(pack(None, 0), backward), "lampa_ff_workspace_bytes")
        ws = torch.empty(size, dtype=torch.uint8, device=x.device) if size else None
        check(getattr(lib, name)(pack(ws, size), stream_of(x)), name)


def _forward(x, w_gate, w_up, w_down, act):
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    _launch("lampa_ff_fwd", 0, x, (w_gate, w_up, w_down), act, y=y)
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
        grads = tuple(make(t.shape, dtype=t.dtype, device=t.device) if need else None
                      for t, need in zip(tensors, ctx.needs_input_grad))
        _launch("lampa_ff_bwd", 1, x, tensors[1:], ctx.act, dy=_packed(dy.to(x.dtype)), grads=grads)
        return (*grads, None)


def gated_feed_forward(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
                       activation: Optional[str] = "silu") -> torch.Tensor:
    """x [..., D] (rows may be column slices of a wider tensor); w_gate, w_up [F, D], w_down [D, F] of x's type (as ``nn.Linear``
    keeps them); ``activation`` of the gate ``None`` / ``'sigmoid'`` / ``'silu'`` / ``'swish'``. D and F multiples of 8, up to
    2^17. Returns [..., D] in x's type.

    Products have fp32 sums; for 16-bit types the hidden values act(.) * (.) (and, in the gradients, theirs) are rounded to the type
    as the next product's operands. Differentiable in every tensor (first order; the gradients compute the hidden values again, so
    nothing but the inputs is kept; repeated calls give the same bits)."""
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
    if _direct(x, w_gate, w_up, w_down) or not _wants_grad(x, w_gate, w_up, w_down):
        return _forward(x, w_gate, w_up, w_down, act)
    return _GatedFeedForward.apply(x, w_gate, w_up, w_down, act)
