"""The selective state space scan and its short causal convolution on the gfx950 kernels
(``csrc/selective*.hip``, ``csrc/short_conv.hip``): prompts, training and in-place single tokens.

    z_t = bias + sum_j w_j x_{t - (K - 1) + j},  short_conv = act(z)
    d_t = softplus(delta_t + delta_bias),  S_t = exp(d_t A) S_{t-1} + d_t x_t B_t^T,  y_t = S_t C_t + D x_t

The recurrence beside the SSSD scan (:func:`verace_amd.sssd_scan`): the same [batch, time, heads, dim]
layouts, fp32 states handed from call to call, a differentiable scan and an opt-in in-place step.  Every
launcher enqueues on the current HIP stream of its tensors' device and allocates outputs and workspace
from torch's caching allocator.  There is no CPU path.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _lib
from .hip_kernels import _mask_bytes, _require_device, address, device_guard, refuse_tangents, traced

_ACT = {None: 0, "silu": 1}


def _same_device(like: torch.Tensor, **tensors) -> None:
    device = like.device
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise RuntimeError(f"verace_amd: {name} must be on {device}, got {t.device}")


def _grad_check(like: torch.Tensor, shape, **grads) -> None:
    for name, t in grads.items():
        if t is not None and (t.shape != shape or t.dtype != like.dtype or t.device != like.device):
            raise RuntimeError(f"verace_amd: {name} must be {tuple(shape)} {like.dtype} on {like.device}, "
                               f"got {tuple(t.shape)} {t.dtype} on {t.device}")


def _lengths(lengths: Optional[torch.Tensor], B: int, like: torch.Tensor) -> Optional[torch.Tensor]:
    if lengths is None:
        return None
    if tuple(lengths.shape) != (B,) or lengths.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"verace_amd: lengths must be [{B}] int32 or int64, got {tuple(lengths.shape)} {lengths.dtype}")
    _same_device(like, lengths=lengths)
    return lengths.contiguous()


def _own_state(state: torch.Tensor) -> None:
    """A state that a step may overwrite: not one that autograd follows."""
    if state.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("verace_amd: a state that requires grad cannot be updated in place (use the prompt form, or no_grad)")


def _inner(t: torch.Tensor, lead: int) -> torch.Tensor:
    """t with everything after its first ``lead`` dimensions contiguous (a copy only if it is not)."""
    if t.is_contiguous():
        return t
    expect = 1
    for size, stride in zip(reversed(t.shape[lead:]), reversed(t.stride()[lead:])):
        if size != 1 and stride != expect:
            return t.contiguous()
        expect *= size
    return t


_MAX_ROW = 1 << 23  # elements between tokens that the chunk kernels' 32-bit offsets reach


def _near(t: torch.Tensor) -> torch.Tensor:
    """t, or a copy where its tokens lie further apart than the backward takes."""
    return t if t.stride(1) <= _MAX_ROW else t.clone(memory_format=torch.contiguous_format)


# ------------------------------------------------------------------------------------ short convolution

def _conv_check(x, weight, bias, activation):
    _require_device(x, "x")
    _lib.dtype_code(x.dtype)
    C = x.shape[-1]
    if activation not in _ACT:
        raise RuntimeError(f"verace_amd: activation must be None or 'silu', got {activation!r}")
    if weight.dim() != 2 or weight.shape[0] != C or not 2 <= weight.shape[1] <= 4:
        raise RuntimeError(f"verace_amd: weight must be [{C}, 2 .. 4], got {tuple(weight.shape)}")
    if bias is not None and (tuple(bias.shape) != (C,) or bias.dtype != weight.dtype):
        raise RuntimeError(f"verace_amd: bias must be [{C}] {weight.dtype}, got {tuple(bias.shape)} {bias.dtype}")
    _lib.dtype_code(weight.dtype)
    _same_device(x, weight=weight, bias=bias)


def _conv_args(x, weight, bias, state, lengths, activation):
    """The lengths and the initial state of a call as the launchers take them."""
    if x.dim() != 3:
        raise RuntimeError(f"verace_amd: x must be [B, T, C], got {tuple(x.shape)}")
    _conv_check(x, weight, bias, activation)
    B, T, C = x.shape
    lengths = _lengths(lengths, B, x)
    if state is not None:
        if tuple(state.shape) != (B, weight.shape[1] - 1, C) or state.dtype != x.dtype:
            raise RuntimeError(f"verace_amd: initial_state must be {(B, weight.shape[1] - 1, C)} {x.dtype}, "
                               f"got {tuple(state.shape)} {state.dtype}")
        _same_device(x, initial_state=state)
        state = state.contiguous()
    return lengths, state


def _launch_conv(x, weight, bias, state, lengths, act):
    B, T, C = x.shape
    K = weight.shape[1]
    x, w = _inner(x, 2), weight.contiguous()
    b = None if bias is None else bias.contiguous()
    y = torch.empty(B, T, C, device=x.device, dtype=x.dtype)
    out = torch.empty(B, K - 1, C, device=x.device, dtype=x.dtype)
    with device_guard(x):
        _lib.check(_lib.load().vmi_short_conv(
            address(x), x.stride(1), x.stride(0), address(w), address(b), _lib.dtype_code(x.dtype), _lib.dtype_code(w.dtype), act,
            address(state), address(lengths), int(lengths is not None and lengths.dtype == torch.int64), address(y), address(out),
            B, T, C, K, _lib.raw_stream(x.device)), "vmi_short_conv")
    return y, out


def _launch_conv_bwd(x, weight, bias, state, lengths, act, dy, dout, need):
    """(dx, dweight, dbias, dstate) for dL/dy and dL/dlast rows (either may be None), None where not needed."""
    B, T, C = x.shape
    K = weight.shape[1]
    _grad_check(x, x.shape, dy=dy)
    _grad_check(x, (B, K - 1, C), d_last=dout)
    x, w = _inner(x, 2), weight.contiguous()
    b = None if bias is None else bias.contiguous()
    dy = None if dy is None else _inner(dy, 2)
    dout = None if dout is None else dout.contiguous()
    dx = torch.empty(B, T, C, device=x.device, dtype=x.dtype) if need[0] else None
    dw = torch.empty_like(w) if need[1] else None
    db = torch.empty_like(b) if b is not None and need[2] else None
    dstate = torch.empty_like(state) if state is not None and need[3] else None
    lib = _lib.load()
    ws, ws_bytes = None, ctypes.c_size_t(0)
    if not (dw is None and db is None):
        _lib.check(lib.vmi_short_conv_bwd_workspace_bytes(B, T, C, K, ctypes.byref(ws_bytes)),
                   "vmi_short_conv_bwd_workspace_bytes")
        ws = torch.empty(max(1, ws_bytes.value), device=x.device, dtype=torch.uint8)
    with device_guard(x):
        _lib.check(lib.vmi_short_conv_bwd(
            address(x), x.stride(1), x.stride(0), address(w), address(b), _lib.dtype_code(x.dtype),
            _lib.dtype_code(w.dtype), act, address(state), address(lengths),
            int(lengths is not None and lengths.dtype == torch.int64), address(dy), 0 if dy is None else dy.stride(1),
            0 if dy is None else dy.stride(0), address(dout), address(dx), address(dw), address(db), address(dstate),
            B, T, C, K, address(ws), ws_bytes.value, _lib.raw_stream(x.device)), "vmi_short_conv_bwd")
    return dx, dw, db, dstate


class ShortConvFunction(torch.autograd.Function):
    """:func:`short_conv` as an autograd node (only its inputs are kept)."""

    @staticmethod
    def forward(ctx, x, weight, bias, state, lengths, act):
        y, out = _launch_conv(x, weight, bias, state, lengths, act)
        ctx.save_for_backward(x, weight, bias, state, lengths)
        ctx.act = act
        ctx.set_materialize_grads(False)
        return y, out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dout):
        x, weight, bias, state, lengths = ctx.saved_tensors
        return (*_launch_conv_bwd(x, weight, bias, state, lengths, ctx.act, dy, dout, ctx.needs_input_grad[:4]), None, None)


def short_conv(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    initial_state: Optional[torch.Tensor] = None,
    lengths: Optional[torch.Tensor] = None,
    activation: Optional[str] = "silu",
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Causal depthwise convolution over time, differentiable once.

    x: [batch, seq_len, C] (rows may be slices of a wider projection); weight: [C, K], K = 2 .. 4,
    weight[:, K - 1] on the current token; bias: [C]; initial_state: the K - 1 rows before the first,
    [batch, K - 1, C] in x's dtype (zeros when None, never modified); lengths: [batch] on x's device,
    how many of a right-padded sequence's rows count (values outside 0 .. seq_len are clamped); activation
    "silu" or None.  Returns (y [batch, seq_len, C], the last K - 1 counted rows [batch, K - 1, C]); y
    behind a sequence's length is 0 and x there is not read.
    """
    lengths, state = _conv_args(x, weight, bias, initial_state, lengths, activation)
    refuse_tangents(x, weight, bias, state)
    if traced(x):
        return torch.ops.verace.short_conv(x, weight, bias, state, lengths, activation)
    act = _ACT[activation]
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, state)):
        return ShortConvFunction.apply(x, weight, bias, state, lengths, act)
    return _launch_conv(x, weight, bias, state, lengths, act)


def short_conv_step_(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: Optional[torch.Tensor],
    state: torch.Tensor,
    activation: Optional[str] = "silu",
    active_mask: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """One token of :func:`short_conv` per item with the state [batch, K - 1, C] (contiguous, x's dtype)
    moved up a row in place.  x: [batch, 1, C] or [batch, C].  Items whose ``active_mask`` [batch] is off
    keep their state and give zeros.  Returns y [batch, 1, C].  Not differentiable; a backward of a call that
    took this state raises, as after any in-place operation."""
    refuse_tangents(x, weight, bias, state)
    _own_state(state)
    if traced(x):
        _conv_step_check(x, weight, bias, state, activation, active_mask)
        return torch.ops.verace.short_conv_step_(x, weight, bias, state, activation, active_mask)
    y = _launch_conv_step(x, weight, bias, state, activation, active_mask)
    torch.autograd.graph.increment_version(state)
    return y


def _conv_step_check(x, weight, bias, state, activation, active_mask):
    """(B, K - 1, C) of a step's arguments."""
    _conv_check(x, weight, bias, activation)
    B, K1, C = state.shape if state.dim() == 3 else (-1, -1, -1)
    if K1 != weight.shape[1] - 1 or C != x.shape[-1] or state.dtype != x.dtype or not state.is_contiguous():
        raise RuntimeError(f"verace_amd: state must be a contiguous [B, {weight.shape[1] - 1}, {x.shape[-1]}] {x.dtype} "
                           f"tensor, got {tuple(state.shape)} {state.dtype}")
    if tuple(x.shape) not in ((B, 1, C), (B, C)):
        raise RuntimeError(f"verace_amd: x must hold one token for each of {B} items, got {tuple(x.shape)}")
    _same_device(x, state=state, active_mask=active_mask)
    return B, K1, C


def _launch_conv_step(x, weight, bias, state, activation, active_mask):
    B, K1, C = _conv_step_check(x, weight, bias, state, activation, active_mask)
    x2 = _inner(x.reshape(B, C), 1)
    mask = None if active_mask is None else _mask_bytes(active_mask.reshape(B))
    w = weight.contiguous()
    b = None if bias is None else bias.contiguous()
    y = torch.empty(B, 1, C, device=x.device, dtype=x.dtype)
    with device_guard(x):
        _lib.check(_lib.load().vmi_short_conv_step(
            address(x2), x2.stride(0), address(w), address(b), _lib.dtype_code(x.dtype), _lib.dtype_code(w.dtype), _ACT[activation],
            address(mask), address(state), address(y), B, C, K1 + 1, _lib.raw_stream(x.device)), "vmi_short_conv_step")
    return y


# ------------------------------------------------------------------------------------ selective scan

def _head_vector(t: Optional[torch.Tensor], H: int, name: str) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if t.dim() != 1 or t.shape[0] != H:
        raise RuntimeError(f"verace_amd: {name} must be [{H}], got {tuple(t.shape)}")
    if t.dtype == torch.float32 and t.is_contiguous():
        return t
    return t.to(torch.float32).contiguous()


def _scan_check(x, delta, A, Bm, Cm, D, delta_bias):
    """Shapes of x [B, T, H, P], delta [B, T, H], Bm, Cm [B, T, G, N]: (B, T, H, P, G, N)."""
    _require_device(x, "x")
    _lib.dtype_code(x.dtype)
    if x.dim() != 4:
        raise RuntimeError(f"verace_amd: x must be [B, T, H, P], got {tuple(x.shape)}")
    B, T, H, P = x.shape
    ds, bs = delta.shape, Bm.shape
    if ds != (B, T, H) and ds != (B, T, H, 1):
        raise RuntimeError(f"verace_amd: delta must be [B, T, H] = {(B, T, H)}, got {tuple(ds)}")
    if len(bs) != 4 or bs[0] != B or bs[1] != T or Cm.shape != bs:
        raise RuntimeError(f"verace_amd: B and C must be [B, T, G, N], got {tuple(bs)}, {tuple(Cm.shape)}")
    G, N = bs[2], bs[3]
    if G < 1 or H % G != 0:
        raise RuntimeError(f"verace_amd: {H} heads do not share {G} groups of B and C")
    if not 1 <= N <= 256 or not 1 <= P <= 1024:
        raise RuntimeError(f"verace_amd: built for head sizes 1 .. 1024 and state sizes 1 .. 256, got {P}, {N}")
    if Bm.dtype != x.dtype or Cm.dtype != x.dtype:
        raise RuntimeError(f"verace_amd: B and C must be {x.dtype}, got {Bm.dtype}, {Cm.dtype}")
    _lib.dtype_code(delta.dtype)
    _same_device(x, delta=delta, A=A, B=Bm, C=Cm, D=D, delta_bias=delta_bias)
    return B, T, H, P, G, N


def _state_check(x: torch.Tensor, state: Optional[torch.Tensor], N: int, name: str = "initial_state") -> None:
    if state is not None:
        want = (x.shape[0], x.shape[2], x.shape[3], N)
        if tuple(state.shape) != want:
            raise RuntimeError(f"verace_amd: {name} must be {want}, got {tuple(state.shape)}")
        if state.device != x.device:
            raise RuntimeError(f"verace_amd: {name} must be on {x.device}, got {state.device}")


def launch_selective_hip_scan(
    x: torch.Tensor,
    delta: torch.Tensor,
    A: torch.Tensor,
    B: torch.Tensor,
    C: torch.Tensor,
    D: Optional[torch.Tensor] = None,
    delta_bias: Optional[torch.Tensor] = None,
    softplus: bool = True,
    initial_state: Optional[torch.Tensor] = None,
    lengths: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """:func:`selective_scan` without autograd."""
    b, T, H, P, G, N = _scan_check(x, delta, A, B, C, D, delta_bias)
    lengths = _lengths(lengths, b, x)
    if delta.dim() == 4:
        delta = delta.squeeze(-1)
    A, D, bias = (_head_vector(t, H, n) for t, n in ((A, "A"), (D, "D"), (delta_bias, "delta_bias")))
    _state_check(x, initial_state, N)
    state = None if initial_state is None else initial_state.to(torch.float32).contiguous()
    x, delta, B, C = _inner(x, 2), _inner(delta, 2), _inner(B, 2), _inner(C, 2)
    y = torch.empty(b, T, H, P, device=x.device, dtype=x.dtype)
    out = torch.empty(b, H, P, N, device=x.device, dtype=torch.float32)
    code = _lib.dtype_code(x.dtype)
    lib = _lib.load()
    ws_bytes = ctypes.c_size_t(0)
    _lib.check(lib.vmi_selective_scan_workspace_bytes(b, T, H, P, G, N, code, ctypes.byref(ws_bytes)),
               "vmi_selective_scan_workspace_bytes")
    ws = torch.empty(ws_bytes.value, device=x.device, dtype=torch.uint8) if ws_bytes.value else None
    with device_guard(x):
        _lib.check(lib.vmi_selective_scan_fwd(
            address(x), x.stride(1), x.stride(0), address(delta), delta.stride(1), delta.stride(0), _lib.dtype_code(delta.dtype),
            address(A), address(B), B.stride(1), B.stride(0), address(C), C.stride(1), C.stride(0), address(D), address(bias),
            int(bool(softplus)), code, address(state), address(lengths),
            int(lengths is not None and lengths.dtype == torch.int64), address(y), address(out), b, T, H, P, G, N, address(ws),
            ws_bytes.value, _lib.raw_stream(x.device)), "vmi_selective_scan_fwd")
    return y, out


def launch_selective_hip_scan_bwd(x, delta, A, B, C, dy, D=None, delta_bias=None, softplus=True, initial_state=None,
                                  lengths=None, d_state=None, need_d_state=True):
    """Gradients of :func:`launch_selective_hip_scan` for dy = dL/dy [batch, seq_len, num_heads, head_dim] and
    d_state = dL/dfinal_state (None: zero): (dx, ddelta, dA, dB, dC, dD, ddelta_bias, dinitial_state), dx, dB and
    dC in x's dtype, ddelta in delta's, the others float32; dinitial_state None unless need_d_state."""
    b, T, H, P, G, N = _scan_check(x, delta, A, B, C, D, delta_bias)
    _grad_check(x, x.shape, dy=dy)
    lengths = _lengths(lengths, b, x)
    shape = delta.shape
    if delta.dim() == 4:
        delta = delta.squeeze(-1)
    _state_check(x, initial_state, N)
    _state_check(x, d_state, N, "d_state")
    state, d_state = (None if t is None else t.to(torch.float32).contiguous() for t in (initial_state, d_state))
    A, D, bias = (_head_vector(t, H, n) for t, n in ((A, "A"), (D, "D"), (delta_bias, "delta_bias")))
    x, B, C, dy = (_near(_inner(t, 2)) for t in (x, B, C, dy))
    delta = _inner(delta, 2)

    def new(like, dtype=None):
        return torch.empty(like.shape, device=x.device, dtype=dtype or like.dtype)
    dx, dd, dB, dC = new(x), new(delta), new(B), new(C)
    heads = torch.empty(3, H, device=x.device, dtype=torch.float32)
    d0 = torch.empty(b, H, P, N, device=x.device, dtype=torch.float32) if need_d_state else None
    if b == 0 or T == 0:
        heads.zero_()
        if d0 is not None:
            d0.zero_() if d_state is None else d0.copy_(d_state)
        return dx, dd.view(shape), heads[0], dB, dC, heads[1], heads[2], d0
    code = _lib.dtype_code(x.dtype)
    lib = _lib.load()
    ws_bytes = ctypes.c_size_t(0)
    _lib.check(lib.vmi_selective_scan_bwd_workspace_bytes(b, T, H, P, G, N, code, ctypes.byref(ws_bytes)),
               "vmi_selective_scan_bwd_workspace_bytes")
    ws = torch.empty(ws_bytes.value, device=x.device, dtype=torch.uint8)
    with device_guard(x):
        _lib.check(lib.vmi_selective_scan_bwd(
            address(x), x.stride(1), x.stride(0), address(delta), delta.stride(1), delta.stride(0), _lib.dtype_code(delta.dtype),
            address(A), address(B), B.stride(1), B.stride(0), address(C), C.stride(1), C.stride(0), address(D), address(bias),
            int(bool(softplus)), code, address(state), address(lengths),
            int(lengths is not None and lengths.dtype == torch.int64), address(dy), dy.stride(1), dy.stride(0),
            address(d_state), address(dx), address(dd), address(heads[0]), address(dB), address(dC), address(heads[1]), address(heads[2]),
            address(d0), b, T, H, P, G, N, address(ws), ws_bytes.value, _lib.raw_stream(x.device)),
            "vmi_selective_scan_bwd")
    return dx, dd.view(shape), heads[0], dB, dC, heads[1], heads[2], d0


def _rows_fit(x: torch.Tensor, B: torch.Tensor) -> None:
    if x.dim() == 4 and B.dim() == 4 and max(x.shape[2] * x.shape[3], B.shape[2] * B.shape[3]) > _MAX_ROW:
        raise RuntimeError(f"verace_amd: selective_scan is differentiable up to {_MAX_ROW} elements a token in x, B and C")


class SelectiveScanFunction(torch.autograd.Function):
    """:func:`selective_scan` as an autograd node: only the inputs are kept, the backward makes the states of
    every chunk again."""

    @staticmethod
    def forward(ctx, x, delta, A, B, C, D, delta_bias, softplus, initial_state, lengths):
        _rows_fit(x, B)
        y, state = launch_selective_hip_scan(x, delta, A, B, C, D, delta_bias, softplus, initial_state, lengths)
        ctx.save_for_backward(x, delta, A, B, C, D, delta_bias, initial_state, lengths)
        ctx.softplus = softplus
        ctx.set_materialize_grads(False)
        return y, state

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, d_state):
        x, delta, A, B, C, D, delta_bias, initial_state, lengths = ctx.saved_tensors
        dy = torch.zeros_like(x) if dy is None else dy
        need0 = initial_state is not None and ctx.needs_input_grad[8]
        dx, dd, dA, dB, dC, dD, dbias, d0 = launch_selective_hip_scan_bwd(
            x, delta, A, B, C, dy, D, delta_bias, ctx.softplus, initial_state, lengths, d_state, need0)
        return (dx, dd, dA.to(A.dtype), dB, dC, None if D is None else dD.to(D.dtype),
                None if delta_bias is None else dbias.to(delta_bias.dtype), None,
                d0.to(initial_state.dtype) if need0 else None, None)


def selective_scan(
    x: torch.Tensor,
    delta: torch.Tensor,
    A: torch.Tensor,
    B: torch.Tensor,
    C: torch.Tensor,
    D: Optional[torch.Tensor] = None,
    delta_bias: Optional[torch.Tensor] = None,
    softplus: bool = True,
    initial_state: Optional[torch.Tensor] = None,
    lengths: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Selective state space scan, differentiable once in every tensor argument but ``lengths``.

    x: [batch, seq_len, num_heads, head_dim]; delta: [batch, seq_len, num_heads] (any of the three
    dtypes); A: [num_heads] decay rates (negative for a decaying state); B, C: [batch, seq_len, groups, N]
    in x's dtype, a group shared by num_heads / groups consecutive heads; D, delta_bias: [num_heads];
    softplus: whether the step size is softplus(delta + delta_bias) or that sum itself; initial_state:
    [batch, num_heads, head_dim, N], zeros when None (never modified); lengths: [batch] on x's device, how
    many of a right-padded sequence's tokens count (values outside 0 .. seq_len are clamped).  x, delta, B
    and C may be slices of wider rows.  head_dim <= 1024, N <= 256.  Returns (y in x's dtype, final_state
    float32); y behind a sequence's length is 0 and nothing of the inputs there is used.

    bf16: each term of y and of the gradients of x, B and C is taken to 2^-16 of itself; the states and the other gradients
    are fp32 sums of the inputs as they are.  A NaN or an infinity in a token reaches no earlier output and no
    other row of its head (bf16: an infinity may come out as NaN), but in the backward the gradients of its chunk's other
    tokens and of earlier ones.  Tokens more than 2^23 elements apart run
    token by token, and the backward takes a copy of them; a token of more than 2^23 elements has no backward.
    """
    refuse_tangents(x, delta, A, B, C, D, delta_bias, initial_state)
    if traced(x):
        _scan_check(x, delta, A, B, C, D, delta_bias)
        _state_check(x, initial_state, B.shape[-1])
        for name, t in (("A", A), ("D", D), ("delta_bias", delta_bias)):
            _head_vector(t, x.shape[2], name)
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                           for t in (x, delta, A, B, C, D, delta_bias, initial_state)):
            _rows_fit(x, B)
        return torch.ops.verace.selective_scan(x, delta, A, B, C, D, delta_bias, softplus, initial_state,
                                               _lengths(lengths, x.shape[0], x))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                       for t in (x, delta, A, B, C, D, delta_bias, initial_state)):
        return SelectiveScanFunction.apply(x, delta, A, B, C, D, delta_bias, softplus, initial_state, lengths)
    return launch_selective_hip_scan(x, delta, A, B, C, D, delta_bias, softplus, initial_state, lengths)


def selective_step_(
    x: torch.Tensor,
    delta: torch.Tensor,
    A: torch.Tensor,
    B: torch.Tensor,
    C: torch.Tensor,
    state: torch.Tensor,
    D: Optional[torch.Tensor] = None,
    delta_bias: Optional[torch.Tensor] = None,
    softplus: bool = True,
    active_mask: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """One token of :func:`selective_scan` per item with ``state`` [batch, num_heads, head_dim, N] (float32,
    contiguous) updated in place.  x: [batch, 1, num_heads, head_dim] and delta, B, C alike, or all without
    the time dimension.  Items whose ``active_mask`` [batch] is off keep their state and give zeros.
    Returns y [batch, 1, num_heads, head_dim].  Only for callers that own the state; not differentiable, and a backward
    of a call that took this state raises, as after any in-place operation."""
    refuse_tangents(x, delta, A, B, C, state, D, delta_bias)
    _own_state(state)
    if traced(x):
        x, delta, A, B, C, D, delta_bias = _step_check(x, delta, A, B, C, state, D, delta_bias, active_mask)[:7]
        return torch.ops.verace.selective_step_(x, delta, A, B, C, state, D, delta_bias, softplus, active_mask)
    y = _launch_selective_step(x, delta, A, B, C, state, D, delta_bias, softplus, active_mask)
    torch.autograd.graph.increment_version(state)
    return y


def _step_check(x, delta, A, B, C, state, D, delta_bias, active_mask):
    """x, delta, A, B, C, D, delta_bias of a step as the launcher takes them, and the sizes."""
    if x.dim() == 3:
        x, delta, B, C = x.unsqueeze(1), delta.unsqueeze(1), B.unsqueeze(1), C.unsqueeze(1)
    b, T, H, P, G, N = _scan_check(x, delta, A, B, C, D, delta_bias)
    if T != 1:
        raise RuntimeError(f"verace_amd: selective_step_ takes one token per item, got {T}")
    if delta.dim() == 4:
        delta = delta.squeeze(-1)
    if tuple(state.shape) != (b, H, P, N) or state.dtype != torch.float32 or not state.is_contiguous():
        raise RuntimeError(f"verace_amd: state must be a contiguous float32 {(b, H, P, N)} tensor, "
                           f"got {tuple(state.shape)} {state.dtype}")
    _same_device(x, state=state, active_mask=active_mask)
    A, D, bias = (_head_vector(t, H, n) for t, n in ((A, "A"), (D, "D"), (delta_bias, "delta_bias")))
    return x, delta, A, B, C, D, bias, (b, H, P, G, N)


def _launch_selective_step(x, delta, A, B, C, state, D, delta_bias, softplus, active_mask):
    x, delta, A, B, C, D, bias, (b, H, P, G, N) = _step_check(x, delta, A, B, C, state, D, delta_bias, active_mask)
    x, delta, B, C = _inner(x, 2), _inner(delta, 2), _inner(B, 2), _inner(C, 2)
    mask = None if active_mask is None else _mask_bytes(active_mask.reshape(b))
    y = torch.empty(b, 1, H, P, device=x.device, dtype=x.dtype)
    with device_guard(x):
        _lib.check(_lib.load().vmi_selective_step(
            address(x), x.stride(0), address(delta), delta.stride(0), _lib.dtype_code(delta.dtype), address(A), address(B),
            B.stride(0), address(C), C.stride(0), address(D), address(bias), int(bool(softplus)), _lib.dtype_code(x.dtype),
            address(mask), address(state), address(y), b, H, P, G, N, _lib.raw_stream(x.device)), "vmi_selective_step")
    return y
