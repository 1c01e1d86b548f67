"""The operators either side of the gated-delta forward in a layer: the depthwise causal short convolution and the
(gated) RMS norm, as gfx950 kernels behind the reference's names.

Mirrors ``causal_conv1d`` / ``ShortConvolution`` (``models/hattention/short_convolution.py:426-458,528-721``) and
``rms_norm_gated`` / ``rms_norm`` / ``FusedRMSNormGated`` / ``FusedRMSNormSwishGate`` / ``RMSNorm``
(``models/hattention/fused_norm.py:856-878,1003-1104,2094-2354``). ``causal_conv1d`` and ``residual_norm`` are
differentiable, everything else is forward only; GPU tensors only (no CPU fallback).
"""
import contextlib
import weakref
from typing import Optional, Tuple

import torch
import torch.nn as nn
from torch.autograd import forward_ad as _forward_ad
from torch.autograd.graph import increment_version

from . import _capi
from ._capi import check, ptr, require_cuda, stream_of

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_ACT = {None: 0, "silu": 1, "swish": 1, "sigmoid": 2}


class _ForwardOnly(torch.autograd.Function):
    """Lets the operators take part in a graph that is never differentiated; backward raises."""

    @staticmethod
    def forward(ctx, fn, *tensors):
        return fn()

    @staticmethod
    def backward(ctx, *grads):
        raise NotImplementedError("lampa_amd implements the forward pass of this operator only")


def _code(dtype) -> int:
    if dtype not in _DTYPES:
        raise TypeError(f"lampa_amd: unsupported dtype {dtype} (bfloat16, float16 or float32)")
    return _DTYPES[dtype]


_current_device = getattr(torch._C, "_cuda_getDevice", None)
_here = contextlib.nullcontext()


def _on_device(device: int):
    """The launches of a call go to its tensors' device, whichever is current."""
    return _here if device == _current_device() else torch.cuda.device(device)


def _same_device(what, *tensors) -> int:
    device = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != device:
            require_cuda(*tensors)
            raise ValueError(f"{what}: all tensors must be on one device, got cuda:{device} and {t.device}")
    if device < 0:
        require_cuda(*tensors)
    return device


def _wants_grad(*tensors) -> bool:
    """Whether a call has to go through its autograd function: a gradient can be asked for, or forward-mode gradients are being
    computed (the function raises where one of its inputs has a tangent; past it the tangent would be dropped)."""
    if _forward_ad._current_level >= 0:
        return True
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _plain_f32(t):
    """t in float32 and contiguous, for its pointer: t itself where it is."""
    if t is None or (t.dtype == torch.float32 and t.is_contiguous()):
        return t
    return t.detach().to(torch.float32).contiguous()


def _tokens(t: torch.Tensor, inner: int):
    """(t, elements from one token to the next) of t [B, T, ...] whose dimensions behind T hold `inner` contiguous elements;
    a copy only where the tokens do not lie evenly."""
    if t.is_contiguous():
        return t, inner
    B, T = t.shape[:2]
    expect = 1
    for size, stride in zip(reversed(t.shape[2:]), reversed(t.stride()[2:])):
        if size != 1 and stride != expect:
            return t.contiguous(), inner
        expect *= size
    step = t.stride(1) if T > 1 else t.stride(0) if B > 1 else inner
    if step < inner or (B > 1 and T > 1 and t.stride(0) != T * step):
        return t.contiguous(), inner
    return t, step


def _sequences(what, cu_seqlens, batch, tokens, device):
    """Boundaries as a device int64 tensor. On the host they are checked; on the device they are taken as they are (nothing
    waits for the GPU, and a captured graph may be replayed with others): the kernels hold them inside the tensors."""
    if cu_seqlens is None:
        return None
    if batch != 1:
        raise ValueError(f"{what}: the batch size must be 1 rather than {batch} when cu_seqlens is given; flatten "
                         f"variable-length inputs first")
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2 or cu_seqlens.is_floating_point() or cu_seqlens.dtype == torch.bool:
        raise ValueError(f"{what}: cu_seqlens must hold at least two whole numbers, got {cu_seqlens.dtype} "
                         f"{tuple(cu_seqlens.shape)}")
    if not cu_seqlens.is_cuda:
        cu = cu_seqlens.tolist()
        if cu[0] != 0 or cu[-1] != tokens or any(b < a for a, b in zip(cu[:-1], cu[1:])):
            raise ValueError(f"{what}: cu_seqlens must start at 0, never decrease and end at the number of tokens ({tokens}); "
                             f"got first = {cu[0]}, last = {cu[-1]}")
    return cu_seqlens.to(device=device, dtype=torch.int64).contiguous()


_F32_CACHE = {}


def _root(t: torch.Tensor) -> torch.Tensor:
    return t._base if t._base is not None else t


def _stamp(t: torch.Tensor):
    r = _root(t)
    return (id(r), tuple(t.shape), tuple(t.stride()), t.storage_offset())


def _fresh(entry, parts) -> bool:
    """A remembered copy is valid while every source object is alive, unmoved and unmodified in place."""
    return entry is not None and all(ref() is _root(p) and ver == _root(p)._version and addr == p.data_ptr()
                                     for (ref, ver, addr), p in zip(entry[0], parts))


def _remember(key, parts, value):
    if len(_F32_CACHE) > 512:
        _F32_CACHE.clear()
    _F32_CACHE[key] = ([(weakref.ref(_root(p)), _root(p)._version, p.data_ptr()) for p in parts], value)
    return value


def _f32(t: Optional[torch.Tensor], device) -> Optional[torch.Tensor]:
    """fp32 contiguous copy of a small parameter on ``device``. Copies are remembered per source tensor object and
    dropped when it is modified in place, moved or freed, so a layer does not convert its weights on every call
    (edits made through ``.data`` bypass the version counter and are not noticed)."""
    if t is None:
        return None
    if t.dtype == torch.float32 and t.is_contiguous() and t.device == torch.device(device):
        return t.detach()
    key = ("one", _stamp(t), str(device))
    entry = _F32_CACHE.get(key)
    if _fresh(entry, [t]):
        return entry[1]
    return _remember(key, [t], t.detach().to(device=device, dtype=torch.float32).contiguous())


def _cat_f32(parts, device) -> torch.Tensor:
    key = ("cat", tuple(_stamp(p) for p in parts), str(device))
    entry = _F32_CACHE.get(key)
    if _fresh(entry, parts):
        return entry[1]
    return _remember(key, parts,
                     torch.cat([p.detach().to(device=device, dtype=torch.float32) for p in parts]).contiguous())


# ----------------------------------------------------------------------------------------------- short convolution
@torch.no_grad()
def _conv_launch(x2: torch.Tensor, weight, bias, residual2, activation, cu_seqlens, t_len: int, parts: int = 1):
    """x2 [tokens, D] (last dim contiguous, any row stride) -> y [tokens, D] contiguous, or [parts, tokens, D / parts]
    when the columns are split over ``parts`` output tensors."""
    n, D = x2.shape
    W = weight.shape[-1]
    split = D // parts
    y = torch.empty((n, D) if parts == 1 else (parts, n, split), dtype=x2.dtype, device=x2.device)
    if n == 0:
        return y
    cu = None if cu_seqlens is None else cu_seqlens.to(device=x2.device, dtype=torch.int64).contiguous()
    check(_capi.lib().lampa_causal_conv1d_fwd(
        ptr(x2), x2.stride(0), n, D, W, ptr(weight), ptr(bias), ptr(residual2),
        0 if residual2 is None else residual2.stride(0), ptr(cu), 0 if cu is None else cu.numel() - 1, t_len,
        _ACT[activation], _code(x2.dtype), ptr(y), split, split if parts > 1 else 0, n * split, stream_of(x2)),
        "lampa_causal_conv1d_fwd")
    return y


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[B, T, D] -> [B*T, D] view with a contiguous last dimension (copies only when it has to)."""
    B, T, D = t.shape
    if t.stride(-1) != 1 or (B > 1 and t.stride(0) != T * t.stride(1)) or t.stride(1) % 8 or t.data_ptr() % 16:
        t = t.contiguous()
    return t.as_strided((B * T, D), (t.stride(1), 1))


def _conv_operands(x, weight, bias):
    """x as rows of D, the taps and the bias in fp32 (a copy of this call's own)."""
    D = x.shape[-1]
    x2, step = _tokens(x, D)
    if step % 8 or x2.data_ptr() % 16:
        x2, step = x2.contiguous(), D
        if x2.data_ptr() % 16:
            x2 = x2.clone()
    return x2, step, _plain_f32(weight), _plain_f32(bias)


@torch.no_grad()
def _conv_state_launch(x, weight, bias, activation, cu, past, want_last):
    B, T, D = x.shape
    W = weight.shape[-1]
    n_seq = B if cu is None else cu.numel() - 1
    x2, step, w32, b32 = _conv_operands(x, weight, bias)
    past = None if past is None else past.detach().to(x.dtype).contiguous()
    y = torch.empty((B, T, D), dtype=x.dtype, device=x.device)
    last = torch.empty((n_seq, D, W), dtype=x.dtype, device=x.device) if want_last else None
    with _on_device(x.get_device()):
        check(_capi.lib().lampa_causal_conv1d_state_fwd(
            ptr(x2), step, B * T, D, W, ptr(w32), ptr(b32), ptr(past), ptr(cu), n_seq, T, _ACT[activation], _code(x.dtype),
            ptr(y), ptr(last), stream_of(x)), "lampa_causal_conv1d_state_fwd")
    return y, last


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, past, forward, activation, cu):
        y, last = forward()
        ctx.save_for_backward(x, weight, bias, past, cu)
        ctx.activation = activation
        ctx.residual_dtype = None if residual is None else residual.dtype
        if last is not None:
            ctx.mark_non_differentiable(last)
        return y, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, _):
        x, weight, bias, past, cu = ctx.saved_tensors
        B, T, D = x.shape
        if x.numel() == 0:
            zero = lambda i, t: torch.zeros_like(t) if ctx.needs_input_grad[i] else None  # noqa: E731
            return (zero(0, x), zero(1, weight), zero(2, bias),
                    dy.to(ctx.residual_dtype) if ctx.needs_input_grad[3] else None, None, None, None, None)
        w2 = weight.reshape(D, -1)
        W = w2.shape[1]
        x2, step, w32, b32 = _conv_operands(x, w2, bias)
        past = None if past is None else past.detach().to(x.dtype).contiguous()
        g = dy.to(x.dtype).contiguous()
        if g.data_ptr() % 16:
            g = g.clone()
        dx = torch.empty((B, T, D), dtype=x.dtype, device=x.device)
        dwb = torch.empty((D, W + 1), dtype=torch.float32, device=x.device)
        lib = _capi.lib()
        with _on_device(x.get_device()):
            size = check(lib.lampa_causal_conv1d_bwd_workspace_bytes(B * T, D, W, _code(x.dtype)),
                         "lampa_causal_conv1d_bwd_workspace_bytes")
            ws = torch.empty(size, dtype=torch.uint8, device=x.device)
            check(lib.lampa_causal_conv1d_bwd(
                ptr(x2), step, ptr(g), B * T, D, W, ptr(w32), ptr(b32), ptr(past), ptr(cu), B if cu is None else cu.numel() - 1,
                T, _ACT[ctx.activation], _code(x.dtype), ptr(dx), ptr(dwb), ptr(ws), size, stream_of(x)),
                "lampa_causal_conv1d_bwd")
        dw = dwb[:, :W].to(weight.dtype).reshape(weight.shape) if ctx.needs_input_grad[1] else None
        db = dwb[:, W].to(bias.dtype).reshape(bias.shape) if ctx.needs_input_grad[2] else None
        return dx, dw, db, dy.to(ctx.residual_dtype) if ctx.needs_input_grad[3] else None, None, None, None, None


def causal_conv1d(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                  residual: Optional[torch.Tensor] = None, activation: Optional[str] = None,
                  cu_seqlens: Optional[torch.Tensor] = None, initial_state: Optional[torch.Tensor] = None,
                  output_final_state: bool = False):
    """``short_convolution.py:426-458``: x [B, T, D], weight [D, W] (tap W-1 on the current token), bias [D],
    residual [B, T, D]; activation ``None`` / ``'silu'`` / ``'swish'``; with ``cu_seqlens`` B must be 1 and taps never
    cross a sequence start. Returns [B, T, D] in x's dtype (fp32 arithmetic). Differentiable in x, weight, bias and residual
    (first order; repeated calls give the same bits); rows behind the last boundary of cu_seqlens have gradients of zero, and
    nothing of them, whatever they hold, enters the others.

    ``initial_state`` [sequences, D, W] holds the W inputs before each sequence (a cache as ``causal_conv1d_step`` and
    ``ShortConvolution`` keep it; its oldest column is not read), and ``output_final_state`` returns (y, the W inputs up to
    each sequence's end). Both are data handed from call to call: no gradient runs through them. With either, cu_seqlens is
    taken as ``state_space_scan`` takes it and there is no ``residual``."""
    require_cuda(x, weight, bias, residual, initial_state)
    if activation not in (None, "silu", "swish"):
        raise ValueError(f"Activation `{activation}` not supported yet.")
    if x.dim() != 3:
        raise ValueError("causal_conv1d: x must be [B, T, D]")
    B, T, D = x.shape
    if cu_seqlens is not None and B != 1:
        raise ValueError("causal_conv1d: batch size must be 1 when cu_seqlens is given")
    with_state = initial_state is not None or output_final_state
    if not with_state:
        require_cuda(cu_seqlens)
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"causal_conv1d: the residual must have x's shape {tuple(x.shape)}, got {tuple(residual.shape)}")
    if bias is not None and bias.numel() != D:
        raise ValueError(f"causal_conv1d: the bias must hold {D} values, got {tuple(bias.shape)}")
    if weight is None:
        weight = torch.ones(D, 1, device=x.device)
    grad = _wants_grad(x, weight, bias, residual)
    if with_state or grad:
        what = "causal_conv1d"
        _same_device(what, x, weight, bias, residual, initial_state)
        if weight.numel() % D or (with_state and (weight.shape[0] != D or (bias is not None and tuple(bias.shape) != (D,)))):
            raise ValueError(f"{what}: expected weight [{D}, W] and bias [{D}], got {tuple(weight.shape)} and "
                             f"{None if bias is None else tuple(bias.shape)}")
        W = weight.numel() // D
        cu = _sequences(what, cu_seqlens, B, T, x.device)
    if with_state:
        n_seq = B if cu is None else cu.numel() - 1
        if residual is not None:
            raise ValueError(f"{what}: no residual together with initial_state or output_final_state")
        if initial_state is not None and tuple(initial_state.shape) != (n_seq, D, W):
            raise ValueError(f"{what}: initial_state must have shape {(n_seq, D, W)} ([sequences, D, W]), got "
                             f"{tuple(initial_state.shape)}")
        if initial_state is not None and initial_state.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{what}: no gradient runs through initial_state; pass it detached")
        forward = lambda: _conv_state_launch(x, weight.reshape(D, W), bias, activation, cu, initial_state,  # noqa: E731
                                             output_final_state)
    else:
        if grad:  # a training step's weights are new every time
            w32, b32 = _plain_f32(weight.detach().reshape(D, -1)), _plain_f32(bias)
        else:
            w32, b32 = _f32(weight.reshape(D, -1), x.device), _f32(bias, x.device)
        res2 = None if residual is None else _rows(residual.to(x.dtype))
        x2 = _rows(x)
        forward = lambda: (_conv_launch(x2, w32, b32, res2, activation, cu_seqlens, max(T, 1)).view(B, T, D), None)  # noqa: E731
    if grad:
        y, last = _CausalConv.apply(x, weight, bias, residual, initial_state, forward, activation, cu)
    else:
        y, last = forward()
    return (y, last) if output_final_state else y


def _conv_step_launch(x, cache, weight, bias, activation, target):
    n, D = x.shape
    step = x.stride(0) if n > 1 else D
    if step < D or (D > 1 and x.stride(1) != 1):
        x, step = x.contiguous(), D
    w32, b32 = _plain_f32(weight), _plain_f32(bias)
    y = torch.empty((n, D), dtype=x.dtype, device=x.device)
    with _on_device(x.get_device()):
        check(_capi.lib().lampa_causal_conv1d_step(ptr(x), step, ptr(cache), ptr(target), ptr(w32), ptr(b32), _ACT[activation],
                                                   _code(x.dtype), ptr(y), n, D, weight.numel() // D, stream_of(x)),
              "lampa_causal_conv1d_step")
    return y


def causal_conv1d_step(x: torch.Tensor, cache: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                       activation: Optional[str] = None, new_cache: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token for each of n sequences: x [n, D], ``cache`` [n, D, W] (x's type, contiguous) with the last W inputs, weight
    [D, W], bias [D], W <= 8, any D. Returns y [n, D]; the cache is moved on in place, or, with ``new_cache`` (same shape, no
    shared memory), left as it is and the next one written there. The arithmetic of ``causal_conv1d``, token by token.
    Forward only: the backward raises."""
    what = "causal_conv1d_step"
    _same_device(what, x, cache, weight, bias, new_cache)
    if activation not in (None, "silu", "swish"):
        raise ValueError(f"Activation `{activation}` not supported yet.")
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f"{what}: x must be [n, D], got {tuple(x.shape)}")
    n, D = x.shape
    if weight.numel() % D or weight.shape[0] != D or weight.numel() == 0 or (bias is not None and tuple(bias.shape) != (D,)):
        raise ValueError(f"{what}: expected weight [{D}, W] and bias [{D}], got {tuple(weight.shape)} and "
                         f"{None if bias is None else tuple(bias.shape)}")
    W = weight.numel() // D
    for name, t in (("cache", cache), ("new_cache", new_cache)):
        if t is not None and (tuple(t.shape) != (n, D, W) or t.dtype != x.dtype or not t.is_contiguous()):
            raise ValueError(f"{what}: {name} must be a contiguous {x.dtype} tensor of shape {(n, D, W)}, got {t.dtype} "
                             f"{tuple(t.shape)}")
    if new_cache is not None and new_cache is not cache:
        a, b, size = cache.data_ptr(), new_cache.data_ptr(), cache.numel() * cache.element_size()
        if a != b and a < b + size and b < a + size:
            raise ValueError(f"{what}: new_cache overlaps cache")
    if n == 0:
        return torch.empty_like(x)
    target = cache if new_cache is None else new_cache
    increment_version(target)  # written through its pointer: a backward that saved it must notice
    if _wants_grad(x, weight, bias, cache):
        return _ForwardOnly.apply(lambda: _conv_step_launch(x, cache, weight, bias, activation, target), x, weight, bias, cache)
    return _conv_step_launch(x, cache, weight, bias, activation, target)


@torch.no_grad()
def causal_conv1d_split(x: torch.Tensor, weights, biases=None, activation: Optional[str] = None,
                        cu_seqlens: Optional[torch.Tensor] = None):
    """One launch for several convolutions of equal width over adjacent column blocks of x [B, T, n * D] (the q | k | v
    columns of a fused projection): weights = n tensors [D, W] (or [D, 1, W]), biases = None or n tensors [D].
    Returns n contiguous tensors [B, T, D]. Same arithmetic as ``causal_conv1d`` on each block."""
    require_cuda(x, cu_seqlens, *weights)
    B, T, Dall = x.shape
    n = len(weights)
    D = Dall // n
    if Dall != n * D or any(w.numel() != weights[0].numel() or w.shape[0] != D for w in weights):
        raise ValueError("causal_conv1d_split: the column blocks must have equal width")
    if cu_seqlens is not None and B != 1:
        raise ValueError("causal_conv1d_split: batch size must be 1 when cu_seqlens is given")
    w32 = _cat_f32([w.reshape(D, -1) for w in weights], x.device)
    b32 = None if biases is None or biases[0] is None else _cat_f32(list(biases), x.device)
    y = _conv_launch(_rows(x), w32, b32, None, activation, cu_seqlens, max(T, 1), parts=n)
    return tuple(y[i].view(B, T, D) for i in range(n))


PROJ_CONV_HIDDEN = 128  # contraction length the fused projection kernel is built for


@torch.no_grad()
def proj_conv(x: torch.Tensor, weight: torch.Tensor, conv_weights, conv_biases, conv_split: int, plain_cols: int,
              tokens_per_wg: int = 0):
    """Fused bias-free projections + short convolution (4 taps) + SiLU: x [B, T, 128] bf16, weight [n_cols, 128] bf16
    (the projection weights one after the other), conv_weights = tensors [conv_split, 4] (or [conv_split, 1, 4]) for
    the first len(conv_weights) * conv_split columns, conv_biases = None or matching tensors. Returns
    (conv outputs: tuple of [B, T, conv_split], plain [B, T, plain_cols], tail [B, T, rest]); the projection output
    itself is never written. Same arithmetic as ``F.linear`` in bf16 followed by ``causal_conv1d(..., 'silu')``."""
    require_cuda(x, weight, *conv_weights)
    B, T, K = x.shape
    n_cols = weight.shape[0]
    n_conv = len(conv_weights) * conv_split
    tail = n_cols - n_conv - plain_cols
    if x.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16 or K != PROJ_CONV_HIDDEN or weight.shape[1] != K:
        raise ValueError("proj_conv: bf16 x [B, T, 128] and weight [n_cols, 128] expected")
    if any(w.shape[0] != conv_split or w.shape[-1] != 4 for w in conv_weights) or tail < 0:
        raise ValueError("proj_conv: conv_weights must be [conv_split, 4] each and fit the columns of weight")
    x2 = _rows(x)
    weight = weight.detach().contiguous()
    cw = _cat_f32([w.reshape(conv_split, 4) for w in conv_weights], x.device)
    cb = None if conv_biases is None or conv_biases[0] is None else _cat_f32(list(conv_biases), x.device)
    n = B * T
    y_conv = torch.empty((len(conv_weights), n, conv_split), dtype=x.dtype, device=x.device)
    y_plain = torch.empty((n, plain_cols), dtype=x.dtype, device=x.device)
    y_tail = torch.empty((n, tail), dtype=x.dtype, device=x.device)
    check(_capi.lib().lampa_proj_conv_fwd(ptr(x2), x2.stride(0), n, max(T, 1), K, ptr(weight), n_cols, ptr(cw), ptr(cb), n_conv,
                                          conv_split, ptr(y_conv), plain_cols, ptr(y_plain) if plain_cols else None, tail,
                                          ptr(y_tail) if tail else None, tokens_per_wg, stream_of(x)), "lampa_proj_conv_fwd")
    return (tuple(y_conv[i].view(B, T, conv_split) for i in range(len(conv_weights))), y_plain.view(B, T, plain_cols),
            y_tail.view(B, T, tail))


def norm_proj_supported(o: torch.Tensor, n_out: int) -> bool:
    """Shapes the fused gated-norm + output-projection kernel is built for."""
    return o.dtype == torch.bfloat16 and o.dim() == 4 and o.shape[2] * o.shape[3] == 512 and o.shape[3] == 64 and n_out == 128


@torch.no_grad()
def norm_proj(o: torch.Tensor, g: torch.Tensor, norm_weight: Optional[torch.Tensor], weight: torch.Tensor,
              eps: float = 1e-5, tokens_per_wg: int = 0, residual: Optional[torch.Tensor] = None,
              next_norm_weight: Optional[torch.Tensor] = None, next_eps: float = 1e-5):
    """``o_proj(FusedRMSNormSwishGate(o, g))`` in one kernel: o, g [B, T, 8, 64] bf16 (g may be a view with a token
    stride), norm_weight [64] or None, weight [128, 512] bf16 -> [B, T, 128]. The normalised tensor is rounded to bf16
    as the two-step route stores it, but never written. With ``residual`` [B, T, 128] (bf16) the kernel also applies the
    residual add and the next pre-norm, ``RMSNorm(next_norm_weight, next_eps)(y, residual, prenorm=True)``, and returns
    (normalised [B, T, 128], residual + y [B, T, 128])."""
    require_cuda(o, g, norm_weight, weight)
    if not norm_proj_supported(o, weight.shape[0]) or weight.dtype != torch.bfloat16 or weight.shape[1] != 512:
        raise ValueError("norm_proj: bf16 o [B, T, 8, 64] and weight [128, 512] expected")
    B, T, H, D = o.shape
    o = o.contiguous()
    g = g.to(o.dtype)
    if not (g.stride(-1) == 1 and g.stride(-2) == D and g.stride(1) % 8 == 0 and g.data_ptr() % 16 == 0
            and (B == 1 or g.stride(0) == T * g.stride(1))):
        g = g.contiguous()
    w32 = _f32(norm_weight, o.device)
    weight = weight.detach().contiguous()
    y = torch.empty((B, T, weight.shape[0]), dtype=o.dtype, device=o.device)
    res_out, nw32 = None, None
    if residual is not None:
        require_cuda(residual, next_norm_weight)
        if residual.shape != y.shape or residual.dtype != o.dtype:
            raise ValueError("norm_proj: residual must be bf16 [B, T, 128]")
        residual = residual.contiguous()
        res_out = torch.empty_like(y)
        nw32 = _f32(next_norm_weight, o.device)
    check(_capi.lib().lampa_norm_proj_fwd(ptr(o), ptr(g), g.stride(1), ptr(w32), ptr(weight), B * T, H, D, weight.shape[0],
                                          float(eps), ptr(y), ptr(residual), ptr(nw32), float(next_eps), ptr(res_out),
                                          tokens_per_wg, stream_of(o)), "lampa_norm_proj_fwd")
    return y if residual is None else (y, res_out)


class ShortConvolution(nn.Conv1d):
    """``short_convolution.py:528-721``: depthwise causal convolution over the time axis of a [B, T, D] tensor with
    an optional SiLU, a cache of the last W inputs per sequence ([N, D, W]) and a one-token ``step``."""

    def __init__(self, hidden_size: int, kernel_size: int, bias: bool = False, activation: Optional[str] = 'silu',
                 use_fast_conv1d: Optional[bool] = True, device=None, dtype=None, **kwargs):
        super().__init__(in_channels=hidden_size, out_channels=hidden_size, kernel_size=kernel_size, groups=hidden_size,
                         bias=bias, padding=kernel_size - 1, device=device, dtype=dtype)
        self.hidden_size = hidden_size
        self.activation = None
        if kernel_size % 2 != 0:
            raise ValueError("Kernel size must be the power of 2")
        if activation is not None:
            assert activation in ['silu', 'swish'], f"Activation `{activation}` not supported yet."
            self.activation = activation
        self.use_fast_conv1d = False  # one implementation here: the HIP kernel

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
                cache: Optional[torch.Tensor] = None, output_final_state: bool = False,
                cu_seqlens: Optional[torch.LongTensor] = None, **kwargs) -> Tuple[torch.Tensor, torch.Tensor]:
        B, T, D, W = *x.shape, self.kernel_size[0]
        N = B if cu_seqlens is None else len(cu_seqlens) - 1
        if mask is not None:
            if cu_seqlens is not None:
                raise ValueError("`mask` and `cu_seqlens` cannot be provided at the same time")
            x = x.mul_(mask.unsqueeze(-1))
        if output_final_state and cache is None:
            cache = x.new_zeros(N, D, W)
        if cache is not None and B * T == N:
            return self.step(x, residual, cache, cu_seqlens)
        if cache is not None:
            with torch.no_grad():
                if cu_seqlens is not None:
                    cu = cu_seqlens.to(x.device).long()
                    idx = cu[1:, None] - W + torch.arange(W, device=x.device)[None]          # [N, W]
                    ok = idx >= torch.maximum(cu[:-1], cu[1:] - W)[:, None]
                    rows = x[0][idx.clamp(min=0)] * ok[..., None].to(x.dtype)                # [N, W, D]
                    cache.copy_(rows.transpose(1, 2))
                else:
                    cache[:, :, -min(W, T):].copy_(x[..., -min(W, T):, :].transpose(1, 2))
        y = causal_conv1d(x=x, weight=self.weight.reshape(D, W), bias=self.bias, residual=residual,
                          activation=self.activation, cu_seqlens=cu_seqlens)
        return y, cache

    def step(self, x: torch.Tensor, residual: Optional[torch.Tensor], cache: torch.Tensor,
             cu_seqlens: Optional[torch.LongTensor] = None):
        """One token per sequence: the cache is moved on in place, and the convolution runs over its W columns. Differentiable in x, the
        taps and the bias, as the call on more tokens is; no gradient runs through the cache. Computed and returned in the
        cache's type: a cache wider than x keeps its bits."""
        shape = x.shape
        x = x.to(cache.dtype)
        D, W = self.hidden_size, self.kernel_size[0]
        weight = self.weight.reshape(D, W)
        held = cache.contiguous()
        if _wants_grad(x, weight, self.bias):
            past = held.detach().clone()  # the backward's own: the cache moves on
            y, last = causal_conv1d(x.reshape(-1, 1, D), weight, self.bias, activation=self.activation, initial_state=past,
                                    output_final_state=True)
            with torch.no_grad():
                cache.copy_(last)
        else:
            with torch.no_grad():
                y = causal_conv1d_step(x.reshape(-1, D), held, weight, self.bias, self.activation)
                if held is not cache:
                    cache.copy_(held)
        y = y.reshape(shape)
        if residual is not None:
            y = y + residual
        return y, cache

    @property
    def state_size(self) -> int:
        return self.hidden_size * self.kernel_size


# ------------------------------------------------------------------------------------------------------ RMS norm
@torch.no_grad()
def _norm_launch(x2, g2, weight, bias, residual2, residual_dtype, eps, activation, g_group=0, g_group_stride=0):
    rows, D = x2.shape
    y = torch.empty_like(x2)
    want_res_out = residual2 is not None or (residual_dtype is not None and residual_dtype != x2.dtype)
    res_out = torch.empty((rows, D), dtype=residual_dtype, device=x2.device) if want_res_out else None
    if rows:
        check(_capi.lib().lampa_rms_norm_fwd(
            ptr(x2), ptr(g2), ptr(weight), ptr(bias), ptr(residual2), ptr(res_out), ptr(y), None, rows, D, float(eps),
            _ACT[activation] if g2 is not None else 0, _code(x2.dtype),
            _code(residual_dtype) if want_res_out else _code(x2.dtype), g_group, g_group_stride, stream_of(x2)),
            "lampa_rms_norm_fwd")
    return y, (res_out if res_out is not None else x2)


def _rms_norm_any(x, g, weight, bias, activation, residual, eps, prenorm, residual_in_fp32):
    require_cuda(x, g, weight, bias, residual)
    shape = x.shape
    D = shape[-1]
    x2 = x.reshape(-1, D).contiguous()
    g2, g_group, g_group_stride = None, 0, 0
    if g is not None:
        g = g.to(x.dtype)
        # [..., T, H, D] view of the g_proj columns of a wider projection output: read in place
        if (g.dim() >= 3 and not g.is_contiguous() and g.stride(-1) == 1 and g.stride(-2) == D and g.stride(-3) % 8 == 0
                and g.data_ptr() % 16 == 0 and g.stride(-3) >= g.shape[-2] * D
                and all(g.stride(i) == g.stride(i + 1) * g.shape[i + 1] for i in range(g.dim() - 3))):
            g2, g_group, g_group_stride = g, g.shape[-2], g.stride(-3)
        else:
            g2 = g.reshape(-1, D).contiguous()
    if residual is not None:
        assert residual.shape == shape
    res2 = None if residual is None else residual.reshape(-1, D).contiguous()
    residual_dtype = res2.dtype if res2 is not None else (torch.float32 if residual_in_fp32 else None)
    w32, b32 = _f32(weight, x.device), _f32(bias, x.device)

    def fn():
        y, res_out = _norm_launch(x2, g2, w32, b32, res2, residual_dtype, eps, activation, g_group, g_group_stride)
        return (y.reshape(shape), res_out.reshape(shape)) if prenorm else y.reshape(shape)

    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, g, weight, bias, residual)):
        return _ForwardOnly.apply(fn, x)
    return fn()


def rms_norm_gated(x: torch.Tensor, g: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, activation: str = 'swish',
                   residual: Optional[torch.Tensor] = None, prenorm: bool = False, residual_in_fp32: bool = False,
                   eps: float = 1e-6):
    """``fused_norm.py:856-878``: y = rmsnorm(x + residual) * weight + bias, times ``g * sigmoid(g)`` ('swish' /
    'silu') or ``sigmoid(g)`` ('sigmoid'); the norm runs over the last dimension. ``prenorm`` also returns x + residual."""
    if activation not in ('swish', 'silu', 'sigmoid'):
        raise ValueError(f"Unsupported activation: {activation}")
    return _rms_norm_any(x, g, weight, bias, activation, residual, eps, prenorm, residual_in_fp32)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, residual: torch.Tensor = None, eps: float = 1e-5,
             prenorm: bool = False, residual_in_fp32: bool = False):
    """``fused_norm.py:2094-2112``: y = rmsnorm(x + residual) * weight + bias; ``prenorm`` also returns x + residual."""
    return _rms_norm_any(x, None, weight, bias, None, residual, eps, prenorm, residual_in_fp32)


_GATE_NONE, _GATE_TOKEN, _GATE_SEQUENCE = 0, 1, 2


def _packed(t):
    """Contiguous and 16-byte aligned, as the row kernels read it."""
    if t is None or (t.is_contiguous() and t.data_ptr() % 16 == 0):
        return t
    t = t.detach().contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _vec32(t):
    return _packed(_plain_f32(t))


def _norm_sizes(x, gate):
    D = x.shape[-1]
    rows = x.numel() // D
    if gate is None:
        return rows, max(rows, 1), D, _GATE_NONE
    if gate.shape == x.shape:
        return rows, max(rows, 1), D, _GATE_TOKEN
    return rows, max(x.shape[1], 1), D, _GATE_SEQUENCE


def _residual_norm_launch(x, residual, weight, post_weight, gate, act, scale, eps):
    rows, seq_rows, D, kind = _norm_sizes(x, gate)
    x_, r_, g_ = _packed(x), _packed(residual), _packed(gate)
    w, pw, sc = _vec32(weight), _vec32(post_weight), _vec32(scale)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    out = None if residual is None else torch.empty(x.shape, dtype=residual.dtype, device=x.device)
    with _on_device(x.get_device()):
        check(_capi.lib().lampa_residual_norm_fwd(ptr(x_), ptr(r_), ptr(w), ptr(pw), ptr(g_), kind, act, ptr(sc), rows, seq_rows, D,
                                                  float(eps), _code(x.dtype), _code((x if residual is None else residual).dtype),
                                                  ptr(y), ptr(out), stream_of(x)), "lampa_residual_norm_fwd")
    return y, out


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, post_weight, gate, scale, act, eps):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, residual, weight, post_weight, gate, scale)
        ctx.act, ctx.eps = act, eps
        return _residual_norm_launch(x, residual, weight, post_weight, gate, act, scale, eps)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dres):
        x, residual, weight, post_weight, gate, scale = ctx.saved_tensors
        rows, seq_rows, D, kind = _norm_sizes(x, gate)
        x_, r_, g_ = _packed(x), _packed(residual), _packed(gate)
        w, pw, sc = _vec32(weight), _vec32(post_weight), _vec32(scale)
        dy = None if dy is None else _packed(dy.to(x.dtype))
        dres = None if dres is None or residual is None else _packed(dres.to(residual.dtype))
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        res_dtype = (x if residual is None else residual).dtype
        dr = None if residual is None else torch.empty(x.shape, dtype=res_dtype, device=x.device)
        make = torch.empty if rows else torch.zeros  # without rows nothing is launched
        need = ctx.needs_input_grad
        vec = lambda t, wanted: make(D, dtype=torch.float32, device=x.device) if t is not None and wanted else None  # noqa: E731
        dw, dpw, dsc = vec(weight, need[2]), vec(post_weight, need[3]), vec(scale, need[5])
        dg = make(gate.shape, dtype=gate.dtype, device=x.device) if gate is not None and need[4] else None
        lib = _capi.lib()
        with _on_device(x.get_device()):
            size = check(lib.lampa_residual_norm_bwd_workspace_bytes(rows, seq_rows, D), "lampa_residual_norm_bwd_workspace_bytes")
            ws = torch.empty(max(size, 1), dtype=torch.uint8, device=x.device)
            check(lib.lampa_residual_norm_bwd(ptr(x_), ptr(r_), ptr(w), ptr(pw), ptr(g_), kind, ctx.act, ptr(sc), ptr(dy), ptr(dres),
                                              rows, seq_rows, D, float(ctx.eps), _code(x.dtype), _code(res_dtype), ptr(dx),
                                              ptr(dr), ptr(dg), ptr(dw), ptr(dpw), ptr(dsc), ptr(ws), size, stream_of(x)),
                  "lampa_residual_norm_bwd")
        cast = lambda g, t: None if g is None else g.to(t.dtype)  # noqa: E731
        return dx, dr, cast(dw, weight), cast(dpw, post_weight), dg, cast(dsc, scale), None, None


def residual_norm(x: torch.Tensor, residual: Optional[torch.Tensor], weight: Optional[torch.Tensor] = None,
                  post_weight: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                  gate_activation: Optional[str] = None, residual_scale: Optional[torch.Tensor] = None, eps: float = 1e-5):
    """The border between two blocks in one pass: x [..., D] is a block's output, ``residual`` (x's shape; x's type or
    float32) the stream it is added to::

        a = rms_norm(x, post_weight)            (x itself without post_weight)
        r = residual + residual_scale * act(gate) * a
        y = rms_norm(r, weight)

    Returns (y in x's type, r in the residual's type), or y alone where there is no residual (None): the gated norm behind a mixer,
    norm of act(gate) * a. y comes from the unrounded r. ``weight``, ``post_weight`` and
    ``residual_scale`` are [D] or None; ``gate`` has x's shape and type, or [B, 1, D] beside x [B, T, D] (one gate for each
    sequence); ``gate_activation`` ``None`` / ``'sigmoid'`` / ``'silu'`` / ``'swish'``. D a multiple of 8, at most 8192.
    Differentiable in every tensor (first order; repeated calls give the same bits)."""
    what = "residual_norm"
    _same_device(what, x, residual, weight, post_weight, gate, residual_scale)
    if gate_activation not in _ACT:
        raise ValueError(f"Activation `{gate_activation}` not supported yet.")
    if x.dim() < 1 or (residual is not None and residual.shape != x.shape):
        raise ValueError(f"{what}: x and residual must have one shape [..., D], got {tuple(x.shape)} and "
                         f"{None if residual is None else tuple(residual.shape)}")
    D = x.shape[-1]
    if D < 8 or D % 8 or D > 8192:
        raise ValueError(f"{what}: the last dimension must be a multiple of 8 and at most 8192, got {D}")
    if _code(x.dtype) != _code((x if residual is None else residual).dtype) and residual.dtype != torch.float32:
        raise TypeError(f"{what}: the residual must have x's type ({x.dtype}) or be float32, got {residual.dtype}")
    for name, t in (("weight", weight), ("post_weight", post_weight), ("residual_scale", residual_scale)):
        if t is not None and (tuple(t.shape) != (D,) or not t.is_floating_point()):
            raise ValueError(f"{what}: {name} must be a floating-point tensor of shape ({D},), got {t.dtype} {tuple(t.shape)}")
    if gate is not None:
        if gate.shape != x.shape and not (x.dim() == 3 and tuple(gate.shape) == (x.shape[0], 1, D)):
            raise ValueError(f"{what}: the gate must have x's shape {tuple(x.shape)}, or [B, 1, D] beside x [B, T, D], got "
                             f"{tuple(gate.shape)}")
        if gate.dtype != x.dtype:
            raise TypeError(f"{what}: the gate must have x's type ({x.dtype}), got {gate.dtype}")
        if gate.shape != x.shape and x.shape[0] > 65535:
            raise ValueError(f"{what}: at most 65535 sequences with a gate each, got {x.shape[0]}")
    act = _ACT[gate_activation]
    if _wants_grad(x, residual, weight, post_weight, gate, residual_scale):
        y, r = _ResidualNorm.apply(x, residual, weight, post_weight, gate, residual_scale, act, eps)
    else:
        y, r = _residual_norm_launch(x, residual, weight, post_weight, gate, act, residual_scale, eps)
    return y if residual is None else (y, r)


class FusedRMSNormGated(nn.Module):
    """``fused_norm.py:1003-1064``."""

    def __init__(self, hidden_size: int, elementwise_affine: bool = True, eps: float = 1e-5, activation: str = 'swish',
                 device=None, dtype=None):
        super().__init__()
        self.hidden_size = hidden_size
        self.elementwise_affine = elementwise_affine
        self.eps = eps
        self.activation = activation
        if self.activation not in ['swish', 'silu', 'sigmoid']:
            raise ValueError(f"Unsupported activation: {self.activation}")
        if elementwise_affine:
            self.weight = nn.Parameter(torch.ones(hidden_size, device=device, dtype=dtype))
        else:
            self.register_parameter("weight", None)
        self.register_parameter("bias", None)

    def forward(self, x: torch.Tensor, g: torch.Tensor, residual: Optional[torch.Tensor] = None, prenorm: bool = False,
                residual_in_fp32: bool = False) -> torch.Tensor:
        return rms_norm_gated(x, g, self.weight, self.bias, self.activation, residual=residual, eps=self.eps,
                              prenorm=prenorm, residual_in_fp32=residual_in_fp32)


class FusedRMSNormSwishGate(FusedRMSNormGated):
    """``fused_norm.py:1088-1104``."""

    def __init__(self, hidden_size: int, elementwise_affine: bool = True, eps: float = 1e-5, device=None, dtype=None):
        super().__init__(hidden_size=hidden_size, elementwise_affine=elementwise_affine, eps=eps, device=device,
                         dtype=dtype)


class RMSNorm(nn.Module):
    """``fused_norm.py:2307-2354``."""

    def __init__(self, hidden_size: int, elementwise_affine: bool = True, bias: bool = False, eps: float = 1e-5):
        super().__init__()
        self.hidden_size = hidden_size
        self.elementwise_affine = elementwise_affine
        self.eps = eps
        self.register_parameter("weight", None)
        self.register_parameter("bias", None)
        if elementwise_affine:
            self.weight = nn.Parameter(torch.ones(hidden_size))
            if bias:
                self.bias = nn.Parameter(torch.zeros(hidden_size))

    def forward(self, x, residual=None, prenorm=False, residual_in_fp32=False):
        return rms_norm(x, self.weight, self.bias, residual=residual, eps=self.eps, prenorm=prenorm,
                        residual_in_fp32=residual_in_fp32)


# ----------------------------------------------------------------------------------------- decay and write gates
@torch.no_grad()
def gdr_gates(a: torch.Tensor, b: torch.Tensor, A_log: torch.Tensor, dt_bias: torch.Tensor, beta_scale: float = 1.0):
    """``modeling_gated_deltaproduct.py:541-547,568-570``: g = -exp(A_log) * softplus(a + dt_bias) and
    beta = sigmoid(b) * beta_scale, both fp32 [..., H]. a, b [..., H] may be column slices of a wider projection."""
    require_cuda(a, b, A_log, dt_bias)
    H = a.shape[-1]
    assert b.shape == a.shape and a.dtype == b.dtype

    def rows(t):
        if t.dim() >= 2 and t.stride(-1) == 1 and all(t.stride(i) == t.stride(i + 1) * t.shape[i + 1]
                                                      for i in range(t.dim() - 2)):
            return t, t.stride(-2) if t.dim() >= 2 else H
        t = t.contiguous()
        return t, H

    a2, a_stride = rows(a)
    b2, b_stride = rows(b)
    n = a.numel() // H
    g = torch.empty(a.shape, dtype=torch.float32, device=a.device)
    beta = torch.empty_like(g)
    A32, dt32 = _f32(A_log, a.device), _f32(dt_bias, a.device)  # named: they must outlive the launch call
    if n:
        check(_capi.lib().lampa_gdr_gates_fwd(ptr(a2), a_stride, ptr(b2), b_stride, ptr(A32), ptr(dt32), n, H,
                                              float(beta_scale), _code(a.dtype), ptr(g), ptr(beta), stream_of(a)),
              "lampa_gdr_gates_fwd")
    return g, beta
