"""The selective scan of a state-space layer, for prompts and for single tokens, on the GPU.

For every sequence and head, with a state S [N, P] in float32 and a head's group of B and C shared by its heads::

    delta_t = softplus(dt_t + dt_bias)
    S_t = exp(delta_t A) S_{t-1} + delta_t B_t x_t^T          y_t = S_t^T C_t + D x_t

``state_space_scan`` runs it over whole sequences (dense or packed) and is differentiable; ``state_space_step`` runs one
token for each sequence on a kept state. It is the mixer behind the reference's LSH-ordered models
(``models/baselines/full_mamba2.py:221-430``, ``models/baselines/hmamba.py:356-460``), whose scan lives in a package the
reference imports. Names, state layout ([sequences, H, N, P], float32) and return tuples follow this package's
``chunk_gated_delta_rule``. GPU tensors only; there is no CPU path.
"""
import struct
import weakref
from typing import Optional

import torch
from torch.autograd.graph import increment_version

from . import _capi
from ._capi import check, ptr, require_cuda, stream_of
from .gated_delta import _direct
from .layer_ops import _DTYPES, _ForwardOnly, _on_device, _plain_f32, _same_device, _sequences, _tokens, _wants_grad

MAX_STATE = 128  # N of state_space_scan; state_space_step takes any
MAX_STRIDE = 1 << 24  # elements between tokens, as lampa_ss_scan_fwd takes them

# lampa_ss_args: 13 pointers, 8 int64, 10 int32, 11 pointers, one int64
_ARGS = struct.Struct("=13Q8q10i11Qq")


def _segment_tokens(longest: int, total: int, heads: int, N: int, dtype, grad: bool) -> int:
    """Length of the segments that run in parallel, a multiple of 64: as many workgroups as the chip holds at once, in one round.
    ``heads`` counts blocks of 64 columns. The chunk kernels (16-bit types) run two workgroups a CU, three without gradients and
    N <= 64; the token-serial ones (float32) one wave a workgroup, eight a CU. 60 000 tokens x 8 heads, segments of 256 / 640 /
    960 / 1920 tokens: forward at N = 64 120 / 95 / 108 / 167 us, with gradients at N = 128 996 / 893 / 779 / 977 us; fp32, 20 000 x
    8, with gradients at N = 64, 64 / 128 / 192 / 640 tokens: 1007 / 980 / 1266 / 3398 us. Segments of fewer tokens than `shortest`
    are not worth the two further launches of joining them: fp32 gradients of 6 007 tokens x 4 heads with 64 / 128 / 256 tokens 194 /
    305 / 549 us, but 77 tokens whole 27 us, in two segments 45; 16-bit forward of 15 000 x 6 with 64 / 256 / 512 tokens 37 / 45 / 63
    us, where 256 leave a quarter of the states to hold."""
    serial = dtype == torch.float32
    per_cu = 8 if serial else 3 if N <= 64 and not grad else 2
    shortest = 256 if not serial else 128 if longest <= 128 else 64
    seg = -(-total * heads // (256 * per_cu) // 64) * 64
    return max(shortest, min(seg, -(-longest // 64) * 64))


def _vectors(t, inner, width):
    """``_tokens`` as the kernels read them. A copy where tokens lie 2^24 elements apart or more (a token of each of several
    long sequences: the kernels form offsets within 64 rows in 32 bits), and where a 16-bit tensor's rows of ``width`` could be
    read in 16-byte pieces but for their place in memory (60 000 tokens x 8 heads of 64 one element off: 303 us read as they
    lie, 111 us aligned, a copy takes 25)."""
    t, step = _tokens(t, inner)
    if step >= MAX_STRIDE or (t.element_size() == 2 and width % 8 == 0 and (step % 8 or t.data_ptr() % 16)):
        return torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t), inner
    return t, step


def _pack(x, dt, A, B, C, D, bias, h0, y, ht, states, decay, cu, longest, seg, n_seq, softplus, for_grad, grad=None):
    (x, xs), (dt, dts), (B, bs), (C, cs) = x, dt, B, C
    H, P = x.shape[-2:]
    G, N = B.shape[-2:]
    p = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    total = x.shape[0] * x.shape[1]
    extra = [0] * 12 if grad is None else [p(t) for t in grad[0]] + [grad[1]]
    return _ARGS.pack(p(x), p(dt), p(B), p(C), p(A), p(D), p(bias), p(h0), p(y), p(ht), p(states), p(decay), p(cu), total,
                      longest, seg, xs, dts, bs, cs, H * P, n_seq, H, P, G, N, _DTYPES[x.dtype], _DTYPES[dt.dtype],
                      int(softplus), int(for_grad), 0, *extra)


def _scan_launch(x, dt, A, B, C, D, bias, softplus, h0, want_final, cu, keep=False):
    """(y, final state or None, kept): kept holds what the gradients need beside the inputs."""
    nb, T, H, P = x.shape
    G, N = B.shape[-2:]
    n_seq = nb if cu is None else cu.numel() - 1
    total, longest = nb * T, T
    dev = x.device
    x, dt = _vectors(x.detach(), H * P, P), _tokens(dt, H)
    B, C = _vectors(B.detach(), G * N, N), _vectors(C.detach(), G * N, N)
    A, D, bias, h0 = _plain_f32(A), _plain_f32(D), _plain_f32(bias), _plain_f32(h0)
    seg = _segment_tokens(longest, total, H * -(-P // 64), N, x[0].dtype, keep)
    single = longest <= seg
    y = torch.empty((nb, T, H, P), dtype=x[0].dtype, device=dev)
    ht = torch.empty((n_seq, H, N, P), dtype=torch.float32, device=dev) if want_final else None
    states = decay = None
    if not single:
        slots = n_seq * -(-T // seg) if cu is None else total // seg + n_seq + 1
        states = torch.empty((slots, H, N, P), dtype=torch.float32, device=dev)
        decay = torch.empty((slots, H), dtype=torch.float32, device=dev)
    with _on_device(dev.index):
        check(_capi.lib().lampa_ss_scan_fwd(
            _pack(x, dt, A, B, C, D, bias, h0, y, ht, states, decay, cu, longest, seg, n_seq, softplus, keep),
            stream_of(y)), "lampa_ss_scan_fwd")
    return y, ht, (states, decay, seg, n_seq, longest)


def _scan_backward(x, dt, A, B, C, D, bias, softplus, h0, cu, kept, dy, dht):
    states, decay, seg, n_seq, longest = kept
    dev = x.device
    nb, T, H, P = x.shape
    G, N = B.shape[-2:]
    dx, ddt, dB, dC = (torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (x, dt, B, C))
    dA = torch.empty(H, dtype=torch.float32, device=dev)
    dD = None if D is None else torch.empty_like(dA)
    dbias = None if bias is None else torch.empty_like(dA)
    dh0 = None if h0 is None else torch.empty((n_seq, H, N, P), dtype=torch.float32, device=dev)
    dy = torch.zeros((nb, T, H, P), dtype=x.dtype, device=dev) if dy is None else dy.to(x.dtype).contiguous()
    dht = _plain_f32(dht)
    if dy.data_ptr() % 16:
        dy = dy.clone()
    x_, dt_ = _vectors(x, H * P, P), _tokens(dt, H)
    B_, C_ = _vectors(B, G * N, N), _vectors(C, G * N, N)
    A, D, bias, h0 = _plain_f32(A), _plain_f32(D), _plain_f32(bias), _plain_f32(h0)
    pack = lambda ws, size: _pack(x_, dt_, A, B_, C_, D, bias, h0, None, None, states, decay, cu, longest, seg, n_seq,  # noqa: E731
                                  softplus, True, ((dy, dht, dx, ddt, dB, dC, dA, dD, dbias, dh0, ws), size))
    lib = _capi.lib()
    with _on_device(dev.index):
        size = check(lib.lampa_ss_bwd_workspace_bytes(pack(None, 0)), "lampa_ss_bwd_workspace_bytes")
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        check(lib.lampa_ss_scan_bwd(pack(ws, size), stream_of(dx)), "lampa_ss_scan_bwd")
    return dx, ddt, dA, dB, dC, dD, dbias, dh0


class _StateSpaceScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, bias, h0, softplus, want_final, cu, keep):
        ctx.set_materialize_grads(False)
        y, ht, kept = _scan_launch(x, dt, A, B, C, D, bias, softplus, h0, want_final, cu, keep=keep)
        if keep:
            ctx.save_for_backward(x, dt, A, B, C, D, bias, h0, cu, kept[0], kept[1])
        # The gradients do not read the final state, so it is not kept; but a gradient through it would be that of the state as
        # it was returned, so one that has been moved on in place is noticed as long as somebody holds it.
        ctx.final = (weakref.ref(ht), ht._version) if keep and want_final else None
        ctx.softplus, ctx.sizes = softplus, kept[2:]
        return y, ht if want_final else None

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dht):
        x, dt, A, B, C, D, bias, h0, cu, states, decay = ctx.saved_tensors
        final = None if ctx.final is None else ctx.final[0]()
        if final is not None and final._version != ctx.final[1]:
            raise RuntimeError("state_space_scan: the final state has been modified by an inplace operation (a step that moved it "
                               "on) before the gradients of the scan that returned it; give state_space_step a new_state")
        dx, ddt, dA, dB, dC, dD, dbias, dh0 = _scan_backward(x, dt, A, B, C, D, bias, ctx.softplus, h0, cu,
                                                             (states, decay, *ctx.sizes), dy, dht)
        as_type = lambda g, t: None if t is None else g.to(t.dtype)  # noqa: E731
        return (dx, ddt, as_type(dA, A), dB, dC, as_type(dD, D), as_type(dbias, bias), as_type(dh0, h0), None, None, None, None)


def _check_operands(what, x, dt, A, B, C, D, dt_bias, tokens):
    """Shapes and types of a call; `tokens`: the leading dimensions of x."""
    xs, bs, own = x.shape, B.shape, x.dtype
    if len(xs) != tokens + 2 or dt.shape != xs[:-1]:
        names = "B, T, " if tokens == 2 else "n, "
        raise ValueError(f"{what}: expected x [{names}H, P] and dt [{names}H], got {tuple(xs)} and {tuple(dt.shape)}")
    H = xs[-2]
    if len(bs) != tokens + 2 or bs != C.shape or bs[:tokens] != xs[:tokens] or bs[-2] < 1 or H % bs[-2]:
        names = "B, T, " if tokens == 2 else "n, "
        raise ValueError(f"{what}: expected B, C [{names}G, N] with G a divisor of the {H} heads, got {tuple(bs)} and "
                         f"{tuple(C.shape)}")
    if H < 1 or xs[-1] < 1 or bs[-1] < 1:
        raise ValueError(f"{what}: heads, columns and states must be at least 1, got H = {H}, P = {xs[-1]}, N = {bs[-1]}")
    for name, t in (("A", A), ("D", D), ("dt_bias", dt_bias)):
        if t is None:
            continue
        if t.dim() != 1 or t.shape[0] != H:
            raise ValueError(f"{what}: {name} must have shape ({H},), one value per head, got {tuple(t.shape)}")
        if not t.is_floating_point():
            raise TypeError(f"{what}: {name} must be a floating-point tensor, got {t.dtype}")
    if own not in _DTYPES or B.dtype != own or C.dtype != own or (dt.dtype != own and dt.dtype != torch.float32):
        raise TypeError(f"{what}: x, B and C must have one type (bfloat16, float16 or float32) and dt that type or float32, got "
                        f"{own}, {B.dtype}, {C.dtype} and {dt.dtype}")


def _check_state(what, name, state, shape):
    if tuple(state.shape) != shape:
        raise ValueError(f"{what}: {name} must have shape {shape} ([sequences, H, N, P]), got {tuple(state.shape)}")


def state_space_scan(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                     D: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None, dt_softplus: bool = False,
                     initial_state: Optional[torch.Tensor] = None, output_final_state: bool = False,
                     cu_seqlens: Optional[torch.Tensor] = None):
    """x [B, T, H, P]; dt [B, T, H] (x's type or float32); A [H] (decay rates, normally negative); B, C [B, T, G, N] with G
    dividing H (head h reads group h // (H // G)), N <= 128; D, dt_bias [H] or None. x, dt, B, C may be column slices of a
    wider tensor. ``dt_softplus`` puts dt + dt_bias through softplus (as it is above 20). Returns (y [B, T, H, P] in x's type,
    final state [sequences, H, N, P] float32 or None).

    With ``cu_seqlens`` [sequences + 1] B must be 1 and the sequences lie one after the other: it starts at 0, never decreases
    and ends at T. A tensor on the host is checked; one on the GPU is not read by the host (so a call can be captured in a
    graph): boundaries outside the tokens are moved inside, and tokens behind the last boundary come back as zero.

    A value that is not finite reaches the tokens from its own on, as in the recurrence, never earlier ones (in gradients a
    dy, B or C that is not finite may reach every token of its 64). Growth (delta A > 0) is taken as it is; where it passes
    float32's range within 64 tokens or a segment the result may be NaN where the recurrence, on zeros, is not.
    Differentiable in every floating-point input (first order); the gradients of B and C are summed over a group's heads in
    a fixed order, and repeated calls give the same bits. (Calls that differ in what else is asked for, gradients or the final
    state, may differ in the last bits of y: they run in other segments and hand states on with more bits.) The backward raises where
    the final state it returned has been moved on in place since: use ``state_space_step(..., new_state=)`` until then."""
    what = "state_space_scan"
    _same_device(what, x, dt, A, B, C, D, dt_bias, initial_state)
    _check_operands(what, x, dt, A, B, C, D, dt_bias, 2)
    H, P = x.shape[-2:]
    N = B.shape[-1]
    if N > MAX_STATE:
        raise ValueError(f"{what}: N must be at most {MAX_STATE}, got {N}")
    cu = _sequences(what, cu_seqlens, x.shape[0], x.shape[1], x.device)
    n_seq = x.shape[0] if cu is None else cu.numel() - 1
    if n_seq < 1:
        raise ValueError(f"{what}: the batch must hold at least one sequence")
    if initial_state is not None:
        _check_state(what, "initial_state", initial_state, (n_seq, H, N, P))
    if _direct(x, dt, A, B, C, D, dt_bias, initial_state):
        y, ht, _ = _scan_launch(x, dt, A, B, C, D, dt_bias, dt_softplus, initial_state, output_final_state, cu)
        return y, ht
    # a call that goes through the function without gradients (parameters under no_grad) is launched as the direct one
    keep = _wants_grad(x, dt, A, B, C, D, dt_bias, initial_state)
    return _StateSpaceScan.apply(x, dt, A, B, C, D, dt_bias, initial_state, bool(dt_softplus), bool(output_final_state), cu, keep)


def _rows(t, inner):
    """(t, elements from one row to the next) of t [n, ...] whose rows are contiguous."""
    return (t, inner) if t.is_contiguous() else _tokens(t.unsqueeze(0), inner)


def _step_launch(x, dt, A, B, C, D, dt_bias, softplus, state, new_state):
    n, H, P = x.shape
    G, N = B.shape[-2:]
    (x, xs), (dt, dts), (B, bs), (C, cs) = _rows(x, H * P), _rows(dt, H), _rows(B, G * N), _rows(C, G * N)
    A, D, dt_bias = _plain_f32(A), _plain_f32(D), _plain_f32(dt_bias)
    y = torch.empty((n, H, P), dtype=x.dtype, device=x.device)
    with _on_device(x.get_device()):
        check(_capi.lib().lampa_ss_step(ptr(x), xs, ptr(dt), dts, ptr(B), bs, ptr(C), cs, ptr(A), ptr(D), ptr(dt_bias),
                                        ptr(state), ptr(new_state), ptr(y), n, H, P, G, N, _DTYPES[x.dtype],
                                        _DTYPES[dt.dtype], int(softplus), stream_of(y)), "lampa_ss_step")
    return y


def state_space_step(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                     state: torch.Tensor, D: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None,
                     dt_softplus: bool = False, new_state: Optional[torch.Tensor] = None):
    """One token for each of n sequences on top of ``state`` [n, H, N, P] (float32, contiguous): x [n, H, P], dt [n, H],
    B, C [n, G, N], everything else as in ``state_space_scan``; any N. Returns y [n, H, P] in x's type. ``state`` is moved on
    in place, or, with ``new_state`` (same shape, no shared memory), left as it is and the next state written there. Forward
    only: the backward raises."""
    what = "state_space_step"
    _same_device(what, x, dt, A, B, C, D, dt_bias, state, new_state)
    _check_operands(what, x, dt, A, B, C, D, dt_bias, 1)
    shape = (x.shape[0], x.shape[1], B.shape[-1], x.shape[2])
    for name, t in (("state", state), ("new_state", new_state)):
        if t is None:
            continue
        _check_state(what, name, t, shape)
        if t.dtype != torch.float32 or not t.is_contiguous():
            raise ValueError(f"{what}: {name} must be float32 and contiguous, as it is read or written in place")
    if new_state is not None and new_state is not state:
        a, b, size = state.data_ptr(), new_state.data_ptr(), state.numel() * 4
        if a != b and a < b + size and b < a + size:
            raise ValueError(f"{what}: new_state overlaps state")
    if x.shape[0] == 0:
        return torch.empty_like(x)
    target = state if new_state is None else new_state
    increment_version(target)  # written through its pointer: a backward that saved it must notice
    if _wants_grad(x, dt, A, B, C, D, dt_bias, state):
        return _ForwardOnly.apply(lambda: _step_launch(x, dt, A, B, C, D, dt_bias, dt_softplus, state, target),
                                  x, dt, A, B, C, D, dt_bias, state)
    return _step_launch(x, dt, A, B, C, D, dt_bias, dt_softplus, state, target)
