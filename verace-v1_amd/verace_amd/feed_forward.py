"""The feed-forward sub-block's products on the gfx950 kernels (``csrc/feed_forward*``, ``csrc/norm_quant.hip``): both gated
projections with their activation and product in one kernel, a projection with bias, activation and residual in its epilogue,
each differentiable, and the same over rows held in 8 bits; the norm with the residual's addition that makes such rows.

    gated_linear    h = a(x Wg^T) * b(x Wu^T)
    linear_add      y = residual + act(x W^T + bias)
    norm_add_quant  s = a + residual, n = rmsnorm(s) w, q scale = n
    quantize_rows   q scale = x

Weights have nn.Linear's layout.  8-bit tensors are float8_e4m3fn with one float32 scale a row (an output channel of a weight):
the value is q * scale.  Every launcher enqueues on the current HIP stream of its tensors' device and allocates outputs and
workspace from torch's caching allocator.  There is no CPU path.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _lib
from .hip_kernels import _require_device, address, device_guard, refuse_tangents, traced

E4M3 = torch.float8_e4m3fn
_LINEAR_ACT = {None: 0, "silu": 1, "gelu": 2}
_GATED_ACT = {"silu": 1, "situ": 3}
_MAX_ROW_BYTES = 1 << 24  # from a row to the next


def _code(dtype: torch.dtype) -> int:
    return _lib.VMI_E4M3 if dtype == E4M3 else _lib.dtype_code(dtype)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t [..., K] as [M, K] with rows as the kernels load them: contiguous, starting on 16 bytes, filled with zeros to whole
    16-byte pieces.  A view of t where it lies so, otherwise a copy."""
    k = t.shape[-1]
    t = t if t.dim() == 2 else t.reshape(-1, k)
    m, piece = t.shape[0], 16 // t.dtype.itemsize
    if k % piece == 0 and t.data_ptr() % 16 == 0 and (k <= 1 or t.stride(1) == 1):
        if m <= 1 or (t.stride(0) % piece == 0 and t.stride(0) >= k and t.stride(0) * t.dtype.itemsize < _MAX_ROW_BYTES):
            return t
    out = torch.empty(m, -(-k // piece) * piece, device=t.device, dtype=t.dtype)
    if out.shape[1] > k:
        out[:, k:].view(torch.uint8).zero_() if t.dtype == E4M3 else out[:, k:].zero_()
    out[:, :k].copy_(t)
    return out[:, :k]


def _ld(t: Optional[torch.Tensor]) -> int:
    """Elements from a row of [M, K] to the next, also where it has but one."""
    if t is None:
        return 0
    piece = 16 // t.dtype.itemsize
    return t.stride(0) if t.shape[0] > 1 else -(-t.shape[1] // piece) * piece


def _plain_rows(t: Optional[torch.Tensor], n: int) -> Optional[torch.Tensor]:
    """t [..., n] as [M, n] whose rows do not overlap, for the epilogue's reads."""
    if t is None:
        return None
    t = t if t.dim() == 2 else t.reshape(-1, n)
    return t if (n <= 1 or t.stride(1) == 1) and (t.shape[0] <= 1 or t.stride(0) >= n) else t.contiguous()


def _weight_check(x, name, w, scale_name, scale) -> None:
    K = x.shape[-1]
    if w.dim() != 2 or w.shape[1] != K or w.dtype != x.dtype or w.device != x.device:
        raise RuntimeError(f"verace_amd: {name} must be [N, {K}] {x.dtype} on {x.device}, "
                           f"got {tuple(w.shape)} {w.dtype} on {w.device}")
    _scale_check(x, scale_name, scale, (w.shape[0],))


def _scale_check(x, name, scale, shape) -> None:
    if (scale is not None) != (x.dtype == E4M3):
        raise RuntimeError(f"verace_amd: {name} belongs to float8_e4m3fn rows, and they to it (x is {x.dtype})")
    if scale is not None and (tuple(scale.shape) != tuple(shape) or scale.dtype != torch.float32 or scale.device != x.device):
        raise RuntimeError(f"verace_amd: {name} must be {tuple(shape)} float32 on {x.device}, "
                           f"got {tuple(scale.shape)} {scale.dtype} on {scale.device}")


def _x_check(x, x_scale, out_dtype) -> torch.dtype:
    """The result's dtype."""
    _require_device(x, "x")
    _code(x.dtype)
    if x.dim() < 1:
        raise RuntimeError("verace_amd: x must be [..., K]")
    _scale_check(x, "x_scale", x_scale, x.shape[:-1])
    if x.dtype != E4M3:
        if out_dtype not in (None, x.dtype):
            raise RuntimeError(f"verace_amd: out_dtype is for float8_e4m3fn rows; with {x.dtype} the result is {x.dtype}")
        return x.dtype
    out_dtype = torch.bfloat16 if out_dtype is None else out_dtype
    _lib.dtype_code(out_dtype)
    return out_dtype


def _vector(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return None if t is None else t.reshape(-1).contiguous()


def _workspace(query, *args, device) -> Tuple[Optional[torch.Tensor], int]:
    need = ctypes.c_size_t(0)
    _lib.check(getattr(_lib.load(), query)(*args, ctypes.byref(need)), query)
    return (torch.empty(need.value, device=device, dtype=torch.uint8) if need.value else None), need.value


def _no_grad_rows(**tensors) -> None:
    if torch.is_grad_enabled():
        for name, t in tensors.items():
            if t is not None and t.requires_grad:
                raise RuntimeError(f"verace_amd: {name} requires grad, and 8-bit rows have no gradients (run under no_grad)")


# ------------------------------------------------------------------------------------ gated projections

def _gated_check(x, w_gate, w_up, x_scale, gate_scale, up_scale, activation, beta1, beta2, out_dtype) -> torch.dtype:
    out_dtype = _x_check(x, x_scale, out_dtype)
    _weight_check(x, "w_gate", w_gate, "gate_scale", gate_scale)
    _weight_check(x, "w_up", w_up, "up_scale", up_scale)
    if w_up.shape != w_gate.shape:
        raise RuntimeError(f"verace_amd: w_up {tuple(w_up.shape)} != w_gate {tuple(w_gate.shape)}")
    if activation not in _GATED_ACT:
        raise RuntimeError(f"verace_amd: activation must be one of {tuple(_GATED_ACT)}, got {activation!r}")
    if activation == "situ" and not (0 < beta1 < float("inf") and 0 < beta2 < float("inf")):
        raise RuntimeError(f"verace_amd: beta1 and beta2 must be positive and finite, got {beta1}, {beta2}")
    return out_dtype


def _pair(w_gate, w_up):
    """Both weights' rows at one distance."""
    g, u = _rows(w_gate), _rows(w_up)
    if _ld(g) != _ld(u):
        g, u = _rows(w_gate.contiguous()), _rows(w_up.contiguous())
    return g, u


def _launch_gated(x, w_gate, w_up, x_scale, gate_scale, up_scale, act, beta1, beta2, out_dtype):
    F, K = w_gate.shape
    x2 = _rows(x)
    g, u = _pair(w_gate, w_up)
    out = torch.empty(*x.shape[:-1], F, device=x.device, dtype=out_dtype)
    with device_guard(x):
        _lib.check(_lib.load().vmi_gated_linear(
            address(x2), _ld(x2), address(_vector(x_scale)), address(g), _ld(g), address(_vector(gate_scale)), address(u), _ld(u),
            address(_vector(up_scale)), _code(x.dtype), act, beta1, beta2, address(out), F, _lib.dtype_code(out_dtype),
            x2.shape[0], F, K, _lib.raw_stream(x.device)), "vmi_gated_linear")
    return out


def _launch_gated_bwd(x, w_gate, w_up, act, beta1, beta2, dh, need):
    """(dx, dw_gate, dw_up) for dL/dh, None where not needed."""
    F, K = w_gate.shape
    if dh.shape != x.shape[:-1] + (F,) or dh.dtype != x.dtype or dh.device != x.device:
        raise RuntimeError(f"verace_amd: dh must be {tuple(x.shape[:-1] + (F,))} {x.dtype} on {x.device}, "
                           f"got {tuple(dh.shape)} {dh.dtype} on {dh.device}")
    x2, dh2 = _rows(x), _plain_rows(dh, F)
    g, u = _pair(w_gate, w_up)
    M = x2.shape[0]
    dx = torch.empty(x.shape, device=x.device, dtype=x.dtype) if need[0] else None
    dw = torch.empty(2, F, K, device=x.device, dtype=x.dtype) if need[1] or need[2] else None
    code = _code(x.dtype)
    ws, ws_bytes = _workspace("vmi_gated_linear_bwd_workspace_bytes", M, F, K, code, device=x.device)
    with device_guard(x):
        _lib.check(_lib.load().vmi_gated_linear_bwd(
            address(x2), _ld(x2), address(g), _ld(g), address(u), _ld(u), code, act, beta1, beta2, address(dh2),
            dh2.stride(0) if M > 1 else F, address(dx), address(dw), M, F, K, address(ws), ws_bytes,
            _lib.raw_stream(x.device)), "vmi_gated_linear_bwd")
    return dx, dw[0] if need[1] else None, dw[1] if need[2] else None


class GatedLinearFunction(torch.autograd.Function):
    """:func:`gated_linear` as an autograd node (only the inputs are kept)."""

    @staticmethod
    def forward(ctx, x, w_gate, w_up, act, beta1, beta2):
        ctx.save_for_backward(x, w_gate, w_up)
        ctx.form = (act, beta1, beta2)
        return _launch_gated(x, w_gate, w_up, None, None, None, act, beta1, beta2, x.dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        x, w_gate, w_up = ctx.saved_tensors
        return (*_launch_gated_bwd(x, w_gate, w_up, *ctx.form, dh, ctx.needs_input_grad[:3]), None, None, None)


def gated_linear(
    x: torch.Tensor,
    w_gate: torch.Tensor,
    w_up: torch.Tensor,
    x_scale: Optional[torch.Tensor] = None,
    gate_scale: Optional[torch.Tensor] = None,
    up_scale: Optional[torch.Tensor] = None,
    activation: str = "situ",
    beta1: float = 4.0,
    beta2: float = 25.0,
    out_dtype: Optional[torch.dtype] = None,
) -> torch.Tensor:
    """``h = a(x w_gate^T) * b(x w_up^T)`` in one kernel, [..., F].

    x: [..., K]; w_gate, w_up: [F, K], all bfloat16, float16 or float32.  ``activation`` "situ" (the layer's):
    a(z) = beta1 tanh(z / beta1) sigmoid(z), b(z) = beta2 tanh(z / beta2); "silu": a(z) = z sigmoid(z), b(z) = z.
    Sums and activations are fp32 and h is rounded once.  Differentiable once in x and both weights: the backward keeps the
    inputs alone, forms both projections again and rounds their gradients to x's dtype once, as operands of its products.

    8 bits: x and the weights float8_e4m3fn with ``x_scale`` [...], ``gate_scale``, ``up_scale`` [F] float32; h is
    ``out_dtype`` (bfloat16), without gradients.
    """
    out_dtype = _gated_check(x, w_gate, w_up, x_scale, gate_scale, up_scale, activation, beta1, beta2, out_dtype)
    refuse_tangents(x, w_gate, w_up)
    if x.dtype == E4M3:
        _no_grad_rows(x_scale=x_scale, gate_scale=gate_scale, up_scale=up_scale)
    if traced(x):
        return torch.ops.verace.gated_linear(x, w_gate, w_up, x_scale, gate_scale, up_scale, activation, beta1, beta2, out_dtype)
    act = _GATED_ACT[activation]
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad):
        return GatedLinearFunction.apply(x, w_gate, w_up, act, float(beta1), float(beta2))
    return _launch_gated(x, w_gate, w_up, x_scale, gate_scale, up_scale, act, beta1, beta2, out_dtype)


# ------------------------------------------------------------------------------------ projection with its epilogue

def _linear_check(x, weight, bias, residual, x_scale, weight_scale, activation, out_dtype) -> torch.dtype:
    out_dtype = _x_check(x, x_scale, out_dtype)
    _weight_check(x, "weight", weight, "weight_scale", weight_scale)
    if activation not in _LINEAR_ACT:
        raise RuntimeError(f"verace_amd: activation must be one of {tuple(_LINEAR_ACT)}, got {activation!r}")
    N = weight.shape[0]
    for name, t, shape in (("bias", bias, (N,)), ("residual", residual, (*x.shape[:-1], N))):
        if t is not None and (tuple(t.shape) != shape or t.dtype != out_dtype or t.device != x.device):
            raise RuntimeError(f"verace_amd: {name} must be {shape} {out_dtype} on {x.device}, "
                               f"got {tuple(t.shape)} {t.dtype} on {t.device}")
    return out_dtype


def _launch_linear(x, weight, bias, residual, x_scale, weight_scale, act, out_dtype):
    N, K = weight.shape
    x2, w, r = _rows(x), _rows(weight), _plain_rows(residual, N)
    M = x2.shape[0]
    out = torch.empty(*x.shape[:-1], N, device=x.device, dtype=out_dtype)
    with device_guard(x):
        _lib.check(_lib.load().vmi_linear_add(
            address(x2), _ld(x2), address(_vector(x_scale)), address(w), _ld(w), address(_vector(weight_scale)), _code(x.dtype),
            address(_vector(bias)), address(r), 0 if r is None else r.stride(0) if M > 1 else N, act, address(out), N,
            _lib.dtype_code(out_dtype), M, N, K, _lib.raw_stream(x.device)), "vmi_linear_add")
    return out


def _launch_linear_bwd(x, weight, bias, act, dy, need):
    """(dx, dweight, dbias) for dL/dy, None where not needed."""
    N, K = weight.shape
    if dy.shape != x.shape[:-1] + (N,) or dy.dtype != x.dtype or dy.device != x.device:
        raise RuntimeError(f"verace_amd: dy must be {tuple(x.shape[:-1] + (N,))} {x.dtype} on {x.device}, "
                           f"got {tuple(dy.shape)} {dy.dtype} on {dy.device}")
    x2, w, dy2 = _rows(x), _rows(weight), _rows(dy)
    M = x2.shape[0]
    dx = torch.empty(x.shape, device=x.device, dtype=x.dtype) if need[0] else None
    dw = torch.empty(N, K, device=x.device, dtype=x.dtype) if need[1] else None
    db = torch.empty(N, device=x.device, dtype=x.dtype) if need[2] and bias is not None else None
    code = _code(x.dtype)
    ws, ws_bytes = _workspace("vmi_linear_add_bwd_workspace_bytes", M, N, K, code, act, device=x.device)
    with device_guard(x):
        _lib.check(_lib.load().vmi_linear_add_bwd(
            address(x2), _ld(x2), address(w), _ld(w), code, address(_vector(bias)), act, address(dy2), _ld(dy2), address(dx),
            address(dw), address(db), M, N, K, address(ws), ws_bytes, _lib.raw_stream(x.device)), "vmi_linear_add_bwd")
    return dx, dw, db


class LinearAddFunction(torch.autograd.Function):
    """:func:`linear_add` as an autograd node (only the inputs are kept; the residual's gradient is dy)."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        ctx.save_for_backward(x, weight, bias)
        ctx.act = act
        return _launch_linear(x, weight, bias, residual, None, None, act, x.dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, bias = ctx.saved_tensors
        need = ctx.needs_input_grad
        grads = _launch_linear_bwd(x, weight, bias, ctx.act, dy, need) if any(need[:3]) else (None, None, None)
        return (*grads, dy if need[3] else None, None)


def linear_add(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    residual: Optional[torch.Tensor] = None,
    x_scale: Optional[torch.Tensor] = None,
    weight_scale: Optional[torch.Tensor] = None,
    activation: Optional[str] = None,
    out_dtype: Optional[torch.dtype] = None,
) -> torch.Tensor:
    """``y = residual + act(x weight^T + bias)`` in one kernel, [..., N].

    x: [..., K]; weight: [N, K]; bias: [N]; residual: [..., N], all of one dtype (bfloat16, float16, float32); ``activation``
    None, "silu" or "gelu" (z Phi(z)).  Sums and the epilogue are fp32 and y is rounded once.  Differentiable once in every
    tensor; the backward keeps x, weight and bias alone.

    8 bits: x and weight float8_e4m3fn with ``x_scale`` [...] and ``weight_scale`` [N] float32; bias, residual and y are
    ``out_dtype`` (bfloat16), without gradients.
    """
    out_dtype = _linear_check(x, weight, bias, residual, x_scale, weight_scale, activation, out_dtype)
    refuse_tangents(x, weight, bias, residual)
    if x.dtype == E4M3:
        _no_grad_rows(x_scale=x_scale, weight_scale=weight_scale, bias=bias, residual=residual)
    if traced(x):
        return torch.ops.verace.linear_add(x, weight, bias, residual, x_scale, weight_scale, activation, out_dtype)
    act = _LINEAR_ACT[activation]
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual)):
        return LinearAddFunction.apply(x, weight, bias, residual, act)
    return _launch_linear(x, weight, bias, residual, x_scale, weight_scale, act, out_dtype)


# ------------------------------------------------------------------------------------ rows in 8 bits

def _quant_check(a, residual, norm_weight) -> None:
    _require_device(a, "a")
    _lib.dtype_code(a.dtype)
    if a.dim() < 1 or a.shape[-1] < 1:
        raise RuntimeError(f"verace_amd: rows must be [..., d], got {tuple(a.shape)}")
    if residual is not None and (residual.shape != a.shape or residual.dtype != a.dtype or residual.device != a.device):
        raise RuntimeError(f"verace_amd: residual must be {tuple(a.shape)} {a.dtype} on {a.device}, "
                           f"got {tuple(residual.shape)} {residual.dtype} on {residual.device}")
    d = a.shape[-1]
    if norm_weight is not None and (tuple(norm_weight.shape) != (d,) or norm_weight.dtype not in (a.dtype, torch.float32)
                                    or norm_weight.device != a.device):
        raise RuntimeError(f"verace_amd: norm_weight must be [{d}] {a.dtype} or float32 on {a.device}, "
                           f"got {tuple(norm_weight.shape)} {norm_weight.dtype} on {norm_weight.device}")


def _launch_quant(a, residual, weight, norm: bool, eps: float, want_sum: bool):
    d = a.shape[-1]
    a2, r2 = _plain_rows(a, d), _plain_rows(residual, d)
    w = _vector(weight)
    q = torch.empty(a.shape, device=a.device, dtype=E4M3)
    scale = torch.empty(a.shape[:-1], device=a.device, dtype=torch.float32)
    s = torch.empty(a.shape, device=a.device, dtype=a.dtype) if want_sum else None
    code = _lib.dtype_code(a.dtype)
    with device_guard(a):
        _lib.check(_lib.load().vmi_norm_add_quant(
            address(a2), a2.stride(0), address(r2), 0 if r2 is None else r2.stride(0), address(w), code,
            code if w is None else _lib.dtype_code(w.dtype), int(norm), eps, address(s), address(q), address(scale),
            a2.shape[0], d, _lib.raw_stream(a.device)), "vmi_norm_add_quant")
    return s, q, scale


def norm_add_quant(
    a: torch.Tensor,
    residual: Optional[torch.Tensor] = None,
    norm_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``s = a + residual``, ``n = s / sqrt(mean s^2 + eps) * norm_weight`` and n in 8 bits: (s, q, scale).

    a, residual: [..., d] of one dtype (bfloat16, float16, float32); norm_weight: [d] of it or float32.  s has a's dtype, q is
    float8_e4m3fn, scale [...] float32: ``scale = max(max |n| / 448, 2^-126)``, ``q = n / scale`` to nearest, ties to even, from
    the unrounded sum in 64 bits.  A row with a NaN or an infinity in s * norm_weight has NaN for scale and q.  No gradients.
    """
    _quant_check(a, residual, norm_weight)
    refuse_tangents(a, residual, norm_weight)
    _no_grad_rows(a=a, residual=residual, norm_weight=norm_weight)
    if traced(a):
        return torch.ops.verace.norm_add_quant(a, residual, norm_weight, eps)
    return _launch_quant(a, residual, norm_weight, True, eps, True)


def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows [..., d] in 8 bits: (q float8_e4m3fn, scale [...] float32), scale and rounding as :func:`norm_add_quant`'s.  For
    a weight [N, K] the scales are its output channels'."""
    _quant_check(x, None, None)
    refuse_tangents(x)
    _no_grad_rows(x=x)
    if traced(x):
        return torch.ops.verace.quantize_rows(x)
    return _launch_quant(x, None, None, False, 0.0, False)[1:]
