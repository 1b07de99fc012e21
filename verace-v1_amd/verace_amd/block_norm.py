"""The norms either side of a block fused with its gate and residual scale (``csrc/gated_norm.hip``),
differentiable: the training form of what :func:`verace_amd.layer_ops.norm_add` does between a layer's
sub-blocks in inference, with a gate and a per-channel residual scale."""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _lib
from .hip_kernels import _require_device, address, device_guard, refuse_tangents, traced

_ACT = {"sigmoid": 0, "silu": 1}


def _rows(t: Optional[torch.Tensor], d: int) -> Optional[torch.Tensor]:
    """t as [rows, d] with contiguous rows (a view where its rows lie at one stride)."""
    if t is None:
        return None
    if t.dim() != 2:
        t = t.reshape(-1, d)
    return t if t.stride(1) == 1 or d == 1 else t.contiguous()


def _checked(y, residual, gate, norm_weight, scale, next_weight, activation):
    """The tensors of a call as the launchers take them."""
    _require_device(y, "y")
    shape, dtype, device = y.shape, y.dtype, y.device
    if len(shape) < 1 or shape[-1] < 1:
        raise RuntimeError(f"verace_amd: y must be [..., d], got {tuple(shape)}")
    _lib.dtype_code(dtype)
    d = shape[-1]
    if d > (4096 if dtype == torch.float32 else 8192):
        raise RuntimeError(f"verace_amd: rows of {d} {dtype} elements are too long for gated_norm_add")
    if activation not in _ACT:
        raise RuntimeError(f"verace_amd: activation must be one of {tuple(_ACT)}, got {activation!r}")
    if residual.shape != shape:
        raise RuntimeError(f"verace_amd: residual shape {tuple(residual.shape)} != y shape {tuple(shape)}")
    if gate is not None and gate.shape != shape:
        try:
            gate.expand(shape)
        except RuntimeError:
            raise RuntimeError(f"verace_amd: gate {tuple(gate.shape)} does not broadcast to {tuple(shape)}") from None
    for name, t in (("residual", residual), ("gate", gate)):
        if t is not None and (t.dtype != dtype or t.device != device):
            raise RuntimeError(f"verace_amd: {name} must be {dtype} on {device}, got {t.dtype} on {t.device}")
    w_dtype = None
    for name, t in (("norm_weight", norm_weight), ("scale", scale), ("next_weight", next_weight)):
        if t is None:
            continue
        if t.dim() != 1 or t.shape[0] != d or t.device != device or t.dtype not in (dtype, torch.float32):
            raise RuntimeError(f"verace_amd: {name} must be [{d}] {dtype} or float32 on {device}, "
                               f"got {tuple(t.shape)} {t.dtype} on {t.device}")
        if w_dtype is not None and t.dtype != w_dtype:
            raise RuntimeError("verace_amd: norm_weight, scale and next_weight must have one dtype")
        w_dtype = t.dtype
    return (y, residual, gate, *(None if t is None else t.contiguous() for t in (norm_weight, scale, next_weight)))


def _gate_rows(gate: Optional[torch.Tensor], y: torch.Tensor) -> Optional[torch.Tensor]:
    return None if gate is None else _rows(gate if gate.shape == y.shape else gate.expand(y.shape), y.shape[-1])


def _launch(y, residual, gate, w1, scale, w2, eps1, eps2, act, want_stats):
    d = y.shape[-1]
    y2, r2, g2 = _rows(y, d), _rows(residual, d), _gate_rows(gate, y)
    s = torch.empty(y.shape, device=y.device, dtype=y.dtype)
    n = None if w2 is None else torch.empty_like(s)
    stats = torch.empty(2, y2.shape[0], device=y.device, dtype=torch.float32) if want_stats else None
    w = next((t for t in (w1, scale, w2) if t is not None), None)
    with device_guard(y):
        _lib.check(_lib.load().vmi_gated_norm(
            address(y2), y2.stride(0), address(r2), r2.stride(0), address(g2), 0 if g2 is None else g2.stride(0), address(w1),
            address(scale), address(w2), _lib.dtype_code(y.dtype), _lib.dtype_code(y.dtype if w is None else w.dtype), act,
            eps1, eps2, address(s), address(n), address(stats), y2.shape[0], d, _lib.raw_stream(y.device)), "vmi_gated_norm")
    return s, n, stats


def _launch_bwd(y, residual, gate, w1, scale, w2, stats, act, ds, dn, need):
    """(dy, dresidual, dgate, dw1, dscale, dw2) for dL/ds and dL/dn (either may be None), None where not needed."""
    d = y.shape[-1]
    y2, r2, g2 = _rows(y, d), _rows(residual, d), _gate_rows(gate, y)
    for name, t in (("ds", ds), ("dn", None if w2 is None else dn)):
        if t is not None and (t.shape != y.shape or t.dtype != y.dtype or t.device != y.device):
            raise RuntimeError(f"verace_amd: {name} must be {tuple(y.shape)} {y.dtype} on {y.device}, "
                               f"got {tuple(t.shape)} {t.dtype} on {t.device}")
    if stats.shape != (2, y2.shape[0]) or stats.dtype != torch.float32 or not stats.is_contiguous() or stats.device != y.device:
        raise RuntimeError(f"verace_amd: stats must be a contiguous float32 {(2, y2.shape[0])} tensor on {y.device}, "
                           f"got {tuple(stats.shape)} {stats.dtype}")
    ds, dn = (None if t is None else t.contiguous() for t in (ds, dn))
    dy, dres, dgate = (torch.empty(y.shape, device=y.device, dtype=y.dtype) if f and t is not None else None
                       for f, t in zip(need[:3], (y, residual, gate)))
    shared = dgate is not None and gate.shape != y.shape  # summed in fp32 over what the gate was broadcast to
    if shared:
        dgate = torch.empty(y.shape, device=y.device, dtype=torch.float32)
    dw1, dscale, dw2 = (torch.empty_like(t) if f and t is not None else None
                        for f, t in zip(need[3:6], (w1, scale, w2)))
    w = next((t for t in (w1, scale, w2) if t is not None), None)
    code = _lib.dtype_code(y.dtype)
    lib = _lib.load()
    ws, ws_bytes = None, ctypes.c_size_t(0)
    if not (dw1 is None and dscale is None and dw2 is None):
        _lib.check(lib.vmi_gated_norm_bwd_workspace_bytes(y2.shape[0], d, code, ctypes.byref(ws_bytes)),
                   "vmi_gated_norm_bwd_workspace_bytes")
        ws = torch.empty(ws_bytes.value, device=y.device, dtype=torch.uint8)
    with device_guard(y):
        _lib.check(lib.vmi_gated_norm_bwd(
            address(y2), y2.stride(0), address(r2), r2.stride(0), address(g2), 0 if g2 is None else g2.stride(0),
            address(w1), address(scale), address(w2), code, _lib.dtype_code(y.dtype if w is None else w.dtype), act | 2 * shared,
            address(stats), address(ds), address(dn), address(dy), address(dres), address(dgate), address(dw1),
            address(dscale), address(dw2), y2.shape[0], d, address(ws), ws_bytes.value, _lib.raw_stream(y.device)),
            "vmi_gated_norm_bwd")
    if shared:
        dgate = dgate.sum_to_size(gate.shape).to(gate.dtype)
    return dy, dres, dgate, dw1, dscale, dw2


class GatedNormFunction(torch.autograd.Function):
    """:func:`gated_norm_add` as an autograd node (the inputs and two fp32 numbers a row are kept)."""

    @staticmethod
    def forward(ctx, y, residual, gate, w1, scale, w2, eps1, eps2, act):
        s, n, stats = _launch(y, residual, gate, w1, scale, w2, eps1, eps2, act, True)
        ctx.save_for_backward(y, residual, gate, w1, scale, w2, stats)
        ctx.act = act
        ctx.set_materialize_grads(False)
        return s, n

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, ds, dn):
        y, residual, gate, w1, scale, w2, stats = ctx.saved_tensors
        return (*_launch_bwd(y, residual, gate, w1, scale, w2, stats, ctx.act, ds, dn, ctx.needs_input_grad[:6]),
                None, None, None)


def gated_norm_add(
    y: torch.Tensor,
    residual: torch.Tensor,
    norm_weight: Optional[torch.Tensor] = None,
    gate: Optional[torch.Tensor] = None,
    scale: Optional[torch.Tensor] = None,
    next_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    next_eps: Optional[float] = None,
    activation: str = "silu",
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``s = residual + scale * act(gate) * rmsnorm(y; norm_weight, eps)`` and
    ``n = rmsnorm(s; next_weight, next_eps)`` in one pass over the rows: (s, n), n None without
    ``next_weight``.

    y, residual: [..., d] of one shape and dtype (rows may be slices of a wider tensor); gate: the same,
    or broadcastable to it (its gradient is then summed in fp32), through ``activation`` ("silu" or "sigmoid"); norm_weight, scale, next_weight:
    [d], all in y's dtype or all float32.  Each may be None and is then left out of the formula.
    d <= 8192 (float32: 4096).  Arithmetic is fp32 and each result is rounded once; n is formed from the
    unrounded s.  Differentiable once, in every tensor argument.
    """
    y, residual, gate, w1, sc, w2 = _checked(y, residual, gate, norm_weight, scale, next_weight, activation)
    refuse_tangents(y, residual, gate, w1, sc, w2)
    if traced(y):
        s, n, _ = torch.ops.verace.gated_norm(y, residual, gate, w1, sc, w2, eps, eps if next_eps is None else next_eps,
                                              activation)
        return s, None if w2 is None else n
    eps1, eps2 = float(eps), float(eps if next_eps is None else next_eps)
    act = _ACT[activation]
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (y, residual, gate, w1, sc, w2)):
        return GatedNormFunction.apply(y, residual, gate, w1, sc, w2, eps1, eps2, act)
    return _launch(y, residual, gate, w1, sc, w2, eps1, eps2, act, False)[:2]
