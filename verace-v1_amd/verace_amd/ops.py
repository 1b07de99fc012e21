"""The HIP launchers as torch operators (``torch.ops.verace.*``), with fake (meta) kernels and
autograd, so that FakeTensor / meta tracing and ``torch.compile(fullgraph=True)`` pass through
the scan instead of breaking the graph at a ctypes call.

Replaces, for tracing purposes, the reference's Triton launcher ``launch_sssd_triton_scan``
(``verace_v1/serving/triton_kernels.py:603-636``), which torch sees as an opaque Python call.

* ``verace::sssd_scan(q, k, v, delta, state?) -> (out, state_T)`` -- :func:`launch_sssd_hip_scan`;
  differentiable through ``verace::sssd_scan_bwd`` (:func:`launch_sssd_hip_scan_bwd`).
* ``verace::sssd_step_(q, k, v, delta, state!) -> out`` -- :func:`sssd_step_` (mutates state).
* ``verace::sssd_scan_fused(proj, H, D, mask?, rms_weight?, rms_eps, state?) -> (out, state_T)``.
* ``verace::sssd_step_fused_(proj, H, D, state!, mask?, rms_weight?, rms_eps) -> out`` --
  :func:`sssd_step_fused_` (mutates state).
* ``verace::cham_scan(q, k, v, gamma, h0_real?, h0_imag?) -> (out, h_real, h_imag)``.
* ``verace::cham_step_(q, k, v, gamma, h_real!, h_imag!, r_real!?, r_imag!?) -> out``.
* ``verace::cham_scan_fused(proj, h, mask?) -> (out, h_real, h_imag)`` -- :func:`launch_cham_hip_update_fused`.
* ``verace::cham_step_fused_(proj, h, h_real!, h_imag!, r_real!?, r_imag!?, mask?) -> out`` --
  :func:`cham_step_fused_` (mutates the states).
* ``verace::ns_retraction(h_real, h_imag, steps) -> (real, imag)``.
* ``verace::selective_scan(x, delta, A, B, C, D?, delta_bias?, softplus, state?, lengths?) -> (y, state_T)`` --
  differentiable through ``verace::selective_scan_bwd``; ``verace::selective_step_(..., state!, ...) -> y``.
* ``verace::short_conv(x, weight, bias?, state?, lengths?, activation?) -> (y, last rows)`` -- differentiable through
  ``verace::short_conv_bwd``; ``verace::short_conv_step_(x, weight, bias?, state!, activation?, mask?) -> y``.
* ``verace::gated_norm(y, residual, gate?, w1?, scale?, w2?, eps, next_eps, activation) -> (s, n, stats)`` -- differentiable
  through ``verace::gated_norm_bwd`` (n empty without w2).

The eager module path calls the launchers directly (no dispatcher overhead in a decode loop);
:class:`~verace_amd.SSSDAttention` switches to these operators while ``torch.compile`` traces.
"""
from __future__ import annotations

from typing import List, Optional, Tuple

import torch
from torch import Tensor

from . import block_norm as bn
from . import hip_kernels as hk
from . import selective as sel


@torch.library.custom_op("verace::sssd_scan", mutates_args=())
def sssd_scan(q: Tensor, k: Tensor, v: Tensor, delta: Tensor,
              state: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    return hk.launch_sssd_hip_scan(q, k, v, delta, state)


@sssd_scan.register_fake
def _sssd_scan_fake(q, k, v, delta, state=None):
    B, T, H, D = q.shape
    return torch.empty_like(q, memory_format=torch.contiguous_format), \
        q.new_empty((B, H, D, D), dtype=torch.float32)


@torch.library.custom_op("verace::sssd_scan_bwd", mutates_args=())
def sssd_scan_bwd(q: Tensor, k: Tensor, v: Tensor, delta: Tensor, psi_T: Tensor, d_out: Tensor,
                  d_psi_T: Optional[Tensor], need_d_psi0: bool
                  ) -> Tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    dq, dk, dv, dd, dpsi0 = hk.launch_sssd_hip_scan_bwd(q, k, v, delta, psi_T, d_out, d_psi_T,
                                                         need_d_psi0)
    if dpsi0 is None:  # an operator returns tensors only: an empty placeholder
        dpsi0 = q.new_empty((0,), dtype=torch.float32)
    return dq, dk, dv, dd, dpsi0


@sssd_scan_bwd.register_fake
def _sssd_scan_bwd_fake(q, k, v, delta, psi_T, d_out, d_psi_T, need_d_psi0):
    B, T, H, D = q.shape
    d = delta.squeeze(-1) if delta.dim() == 4 else delta
    dpsi0 = q.new_empty((B, H, D, D) if need_d_psi0 else (0,), dtype=torch.float32)
    return (torch.empty_like(q, memory_format=torch.contiguous_format), q.new_empty(q.shape),
            q.new_empty(q.shape), torch.empty_like(d, memory_format=torch.contiguous_format), dpsi0)


def _scan_setup(ctx, inputs, output):
    q, k, v, delta, state = inputs
    _, psi = output
    ctx.save_for_backward(q, k, v, delta, psi)
    ctx.state_dtype = None if state is None else state.dtype
    ctx.k_dtype, ctx.v_dtype, ctx.delta_shape = k.dtype, v.dtype, delta.shape


def _scan_backward(ctx, d_out, d_psi):
    q, k, v, delta, psi = ctx.saved_tensors
    need0 = ctx.state_dtype is not None and ctx.needs_input_grad[4]
    if d_out is None:
        d_out = torch.zeros_like(q)
    dq, dk, dv, dd, dpsi0 = torch.ops.verace.sssd_scan_bwd(q, k, v, delta, psi, d_out, d_psi, need0)
    return (dq, dk.to(ctx.k_dtype), dv.to(ctx.v_dtype), dd.view(ctx.delta_shape),
            dpsi0.to(ctx.state_dtype) if need0 else None)


sssd_scan.register_autograd(_scan_backward, setup_context=_scan_setup)


@torch.library.custom_op("verace::sssd_step_", mutates_args=("state",))
def sssd_step_(q: Tensor, k: Tensor, v: Tensor, delta: Tensor, state: Tensor) -> Tensor:
    return hk.sssd_step_(q, k, v, delta, state)


@sssd_step_.register_fake
def _sssd_step_fake(q, k, v, delta, state):
    B, H, D, _ = state.shape
    return q.new_empty((B, 1, H, D))


@torch.library.custom_op("verace::sssd_step_fused_", mutates_args=("state",))
def sssd_step_fused_(proj: Tensor, num_heads: int, head_dim: int, state: Tensor,
                     active_mask: Optional[Tensor], rms_weight: Optional[Tensor],
                     rms_eps: Optional[float]) -> Tensor:
    return hk.sssd_step_fused_(proj, num_heads, head_dim, state, active_mask, rms_weight, rms_eps)


@sssd_step_fused_.register_fake
def _sssd_step_fused_fake(proj, num_heads, head_dim, state, active_mask, rms_weight, rms_eps):
    return proj.new_empty((proj.shape[0], 1, num_heads, head_dim))


@torch.library.custom_op("verace::sssd_scan_fused", mutates_args=())
def sssd_scan_fused(proj: Tensor, num_heads: int, head_dim: int, active_mask: Optional[Tensor],
                    rms_weight: Optional[Tensor], rms_eps: Optional[float],
                    state: Optional[Tensor]) -> Tuple[Tensor, Tensor]:
    return hk.launch_sssd_hip_scan_fused(proj, num_heads, head_dim, active_mask, rms_weight,
                                         rms_eps, state)


@sssd_scan_fused.register_fake
def _sssd_scan_fused_fake(proj, num_heads, head_dim, active_mask, rms_weight, rms_eps, state):
    B, T, _ = proj.shape
    return (proj.new_empty((B, T, num_heads, head_dim)),
            proj.new_empty((B, num_heads, head_dim, head_dim), dtype=torch.float32))


@torch.library.custom_op("verace::cham_scan", mutates_args=())
def cham_scan(q: Tensor, k: Tensor, v: Tensor, gamma: Tensor, h0_real: Optional[Tensor],
              h0_imag: Optional[Tensor]) -> Tuple[Tensor, Tensor, Tensor]:
    init = None if h0_real is None else (h0_real, h0_imag)
    out, (hr, hi) = hk.launch_cham_hip_update(q, k, v, gamma, init)
    return out, hr, hi


@cham_scan.register_fake
def _cham_scan_fake(q, k, v, gamma, h0_real, h0_imag):
    B, T, h = q.shape
    return (torch.empty_like(q, memory_format=torch.contiguous_format),
            q.new_empty((B, h, h), dtype=torch.float32), q.new_empty((B, h, h), dtype=torch.float32))


@torch.library.custom_op("verace::cham_step_", mutates_args=("h_real", "h_imag", "r_real", "r_imag"))
def cham_step_(q: Tensor, k: Tensor, v: Tensor, gamma: Tensor, h_real: Tensor, h_imag: Tensor,
               r_real: Optional[Tensor], r_imag: Optional[Tensor]) -> Tensor:
    readout = None if r_real is None else (r_real, r_imag)
    return hk.cham_step_(q, k, v, gamma, (h_real, h_imag), readout)


@cham_step_.register_fake
def _cham_step_fake(q, k, v, gamma, h_real, h_imag, r_real, r_imag):
    B, h, _ = h_real.shape
    return q.new_empty((B, 1, h))


@torch.library.custom_op("verace::cham_scan_fused", mutates_args=())
def cham_scan_fused(proj: Tensor, holographic_dim: int,
                    active_mask: Optional[Tensor]) -> Tuple[Tensor, Tensor, Tensor]:
    out, (hr, hi) = hk.launch_cham_hip_update_fused(proj, holographic_dim, active_mask)
    return out, hr, hi


@cham_scan_fused.register_fake
def _cham_scan_fused_fake(proj, holographic_dim, active_mask):
    B, T, _ = proj.shape
    h = holographic_dim
    return (proj.new_empty((B, T, h)), proj.new_empty((B, h, h), dtype=torch.float32),
            proj.new_empty((B, h, h), dtype=torch.float32))


@torch.library.custom_op("verace::cham_step_fused_",
                         mutates_args=("h_real", "h_imag", "r_real", "r_imag"))
def cham_step_fused_(proj: Tensor, holographic_dim: int, h_real: Tensor, h_imag: Tensor,
                     r_real: Optional[Tensor], r_imag: Optional[Tensor],
                     active_mask: Optional[Tensor]) -> Tensor:
    readout = None if r_real is None else (r_real, r_imag)
    return hk.cham_step_fused_(proj, holographic_dim, (h_real, h_imag), readout, active_mask)


@cham_step_fused_.register_fake
def _cham_step_fused_fake(proj, holographic_dim, h_real, h_imag, r_real, r_imag, active_mask):
    return proj.new_empty((proj.shape[0], 1, holographic_dim))


@torch.library.custom_op("verace::ns_retraction", mutates_args=())
def ns_retraction(h_real: Tensor, h_imag: Tensor, steps: int) -> Tuple[Tensor, Tensor]:
    return hk.newton_schulz_unitary_retraction(h_real, h_imag, steps)


@ns_retraction.register_fake
def _ns_fake(h_real, h_imag, steps):
    return (h_real.new_empty(h_real.shape, dtype=torch.float32),
            h_real.new_empty(h_real.shape, dtype=torch.float32))


# ------------------------------------------------------------------------------------ selective state space layer

@torch.library.custom_op("verace::selective_scan", mutates_args=())
def selective_scan(x: Tensor, delta: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Optional[Tensor],
                   delta_bias: Optional[Tensor], softplus: bool, state: Optional[Tensor],
                   lengths: Optional[Tensor]) -> Tuple[Tensor, Tensor]:
    return sel.launch_selective_hip_scan(x, delta, A, B, C, D, delta_bias, softplus, state, lengths)


@selective_scan.register_fake
def _selective_scan_fake(x, delta, A, B, C, D, delta_bias, softplus, state, lengths):
    b, T, H, P = x.shape
    return x.new_empty((b, T, H, P)), x.new_empty((b, H, P, B.shape[-1]), dtype=torch.float32)


@torch.library.custom_op("verace::selective_scan_bwd", mutates_args=())
def selective_scan_bwd(x: Tensor, delta: Tensor, A: Tensor, B: Tensor, C: Tensor, dy: Tensor, D: Optional[Tensor],
                       delta_bias: Optional[Tensor], softplus: bool, state: Optional[Tensor],
                       lengths: Optional[Tensor], d_state: Optional[Tensor]) -> List[Tensor]:
    *grads, d0 = sel.launch_selective_hip_scan_bwd(x, delta, A, B, C, dy, D, delta_bias, softplus, state, lengths,
                                                   d_state, state is not None)
    # separate storages: the three head vectors are rows of one tensor
    out = [g.clone() if i in (2, 5, 6) else g for i, g in enumerate(grads)]
    return out + [x.new_empty((0,), dtype=torch.float32) if d0 is None else d0]


@selective_scan_bwd.register_fake
def _selective_scan_bwd_fake(x, delta, A, B, C, dy, D, delta_bias, softplus, state, lengths, d_state):
    H = x.shape[2]
    heads = [x.new_empty((H,), dtype=torch.float32) for _ in range(3)]
    d0 = x.new_empty((0,) if state is None else state.shape, dtype=torch.float32)
    return [x.new_empty(x.shape), delta.new_empty(delta.shape), heads[0], B.new_empty(B.shape), C.new_empty(C.shape),
            heads[1], heads[2], d0]


def _selective_setup(ctx, inputs, output):
    x, delta, A, B, C, D, delta_bias, softplus, state, lengths = inputs
    ctx.save_for_backward(x, delta, A, B, C, D, delta_bias, state, lengths)
    ctx.softplus = softplus


def _selective_backward(ctx, dy, d_state):
    x, delta, A, B, C, D, delta_bias, state, lengths = ctx.saved_tensors
    dy = torch.zeros_like(x) if dy is None else dy
    dx, dd, dA, dB, dC, dD, dbias, d0 = torch.ops.verace.selective_scan_bwd(
        x, delta, A, B, C, dy, D, delta_bias, ctx.softplus, state, lengths, d_state)
    return (dx, dd, dA.to(A.dtype), dB, dC, None if D is None else dD.to(D.dtype),
            None if delta_bias is None else dbias.to(delta_bias.dtype), None,
            None if state is None else d0.to(state.dtype), None)


selective_scan.register_autograd(_selective_backward, setup_context=_selective_setup)


@torch.library.custom_op("verace::selective_step_", mutates_args=("state",))
def selective_step_(x: Tensor, delta: Tensor, A: Tensor, B: Tensor, C: Tensor, state: Tensor, D: Optional[Tensor],
                    delta_bias: Optional[Tensor], softplus: bool, active_mask: Optional[Tensor]) -> Tensor:
    return sel._launch_selective_step(x, delta, A, B, C, state, D, delta_bias, softplus, active_mask)


@selective_step_.register_fake
def _selective_step_fake(x, delta, A, B, C, state, D, delta_bias, softplus, active_mask):
    b, H, P, _ = state.shape
    return x.new_empty((b, 1, H, P))


@torch.library.custom_op("verace::short_conv", mutates_args=())
def short_conv(x: Tensor, weight: Tensor, bias: Optional[Tensor], state: Optional[Tensor], lengths: Optional[Tensor],
               activation: Optional[str]) -> Tuple[Tensor, Tensor]:
    lengths, state = sel._conv_args(x, weight, bias, state, lengths, activation)
    return sel._launch_conv(x, weight, bias, state, lengths, sel._ACT[activation])


@short_conv.register_fake
def _short_conv_fake(x, weight, bias, state, lengths, activation):
    B, _, C = x.shape
    return x.new_empty(x.shape), x.new_empty((B, weight.shape[1] - 1, C))


def _or_empty(like: Tensor, grads) -> List[Tensor]:
    return [like.new_empty((0,)) if g is None else g for g in grads]


def _new_like(like: Tensor, tensors) -> List[Tensor]:
    return _or_empty(like, [None if t is None else t.new_empty(t.shape) for t in tensors])


@torch.library.custom_op("verace::short_conv_bwd", mutates_args=())
def short_conv_bwd(x: Tensor, weight: Tensor, bias: Optional[Tensor], state: Optional[Tensor],
                   lengths: Optional[Tensor], activation: Optional[str], dy: Optional[Tensor],
                   d_last: Optional[Tensor]) -> List[Tensor]:
    lengths, state = sel._conv_args(x, weight, bias, state, lengths, activation)
    return _or_empty(x, sel._launch_conv_bwd(x, weight, bias, state, lengths, sel._ACT[activation], dy, d_last, (True,) * 4))


@short_conv_bwd.register_fake
def _short_conv_bwd_fake(x, weight, bias, state, lengths, activation, dy, d_last):
    return _new_like(x, (x, weight, bias, state))


def _conv_setup(ctx, inputs, output):
    x, weight, bias, state, lengths, ctx.activation = inputs
    ctx.save_for_backward(x, weight, bias, state, lengths)


def _conv_backward(ctx, dy, d_last):
    x, weight, bias, state, lengths = ctx.saved_tensors
    dx, dw, db, ds = torch.ops.verace.short_conv_bwd(x, weight, bias, state, lengths, ctx.activation, dy, d_last)
    return dx, dw, None if bias is None else db, None if state is None else ds, None, None


short_conv.register_autograd(_conv_backward, setup_context=_conv_setup)


@torch.library.custom_op("verace::short_conv_step_", mutates_args=("state",))
def short_conv_step_(x: Tensor, weight: Tensor, bias: Optional[Tensor], state: Tensor, activation: Optional[str],
                     active_mask: Optional[Tensor]) -> Tensor:
    return sel._launch_conv_step(x, weight, bias, state, activation, active_mask)


@short_conv_step_.register_fake
def _short_conv_step_fake(x, weight, bias, state, activation, active_mask):
    return x.new_empty((state.shape[0], 1, state.shape[2]))


@torch.library.custom_op("verace::gated_norm", mutates_args=())
def gated_norm(y: Tensor, residual: Tensor, gate: Optional[Tensor], w1: Optional[Tensor], scale: Optional[Tensor],
               w2: Optional[Tensor], eps: float, next_eps: float, activation: str) -> Tuple[Tensor, Tensor, Tensor]:
    args = bn._checked(y, residual, gate, w1, scale, w2, activation)
    s, n, stats = bn._launch(*args, eps, next_eps, bn._ACT[activation], True)
    for row, w in zip(stats, (w1, w2)):  # not written without that norm
        if w is None:
            row.zero_()
    return s, y.new_empty((0,)) if n is None else n, stats


@gated_norm.register_fake
def _gated_norm_fake(y, residual, gate, w1, scale, w2, eps, next_eps, activation):
    rows = y.numel() // y.shape[-1]
    return (y.new_empty(y.shape), y.new_empty((0,) if w2 is None else y.shape),
            y.new_empty((2, rows), dtype=torch.float32))


@torch.library.custom_op("verace::gated_norm_bwd", mutates_args=())
def gated_norm_bwd(y: Tensor, residual: Tensor, gate: Optional[Tensor], w1: Optional[Tensor], scale: Optional[Tensor],
                   w2: Optional[Tensor], stats: Tensor, activation: str, ds: Optional[Tensor],
                   dn: Optional[Tensor]) -> List[Tensor]:
    args = bn._checked(y, residual, gate, w1, scale, w2, activation)
    return _or_empty(y, bn._launch_bwd(*args, stats, bn._ACT[activation], ds, dn, (True,) * 6))


@gated_norm_bwd.register_fake
def _gated_norm_bwd_fake(y, residual, gate, w1, scale, w2, stats, activation, ds, dn):
    return _new_like(y, (y, residual, gate, w1, scale, w2))


def _norm_setup(ctx, inputs, output):
    y, residual, gate, w1, scale, w2, _, _, ctx.activation = inputs
    ctx.save_for_backward(y, residual, gate, w1, scale, w2, output[2])


def _norm_backward(ctx, ds, dn, _):
    y, residual, gate, w1, scale, w2, stats = ctx.saved_tensors
    given = (y, residual, gate, w1, scale, w2)
    grads = torch.ops.verace.gated_norm_bwd(*given, stats, ctx.activation, ds, None if w2 is None else dn)
    return (*(None if t is None else g for t, g in zip(given, grads)), None, None, None)


gated_norm.register_autograd(_norm_backward, setup_context=_norm_setup)
