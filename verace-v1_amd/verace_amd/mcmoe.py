"""The layer's third sub-block, M-CMoE: library GEMMs with the steps between them (activation,
routing coefficients, norm and adds) on the fused kernels of :mod:`verace_amd.layer_ops` in
inference, as torch ops otherwise.

``SiTUGLU`` restates ``verace_v1/modules/activations.py:8-31`` and
``ManifoldContinuousMoE`` restates ``verace_v1/modules/mcmoe.py:20-120`` with the same
parameter names and creation order (so seeded construction and ``state_dict`` loading
match the reference).  The sparse top-K sum
``sum_k w_k U_{j_k} (sigma_{j_k} * (V_{j_k} x))`` (the reference's loop at :101-117, which
gathers a [tokens, hidden, rank] basis copy per k) is evaluated as two dense GEMMs over all
components with the non-selected components' coefficients set to zero: the same sum, with
no per-token gathers.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from .feed_forward import gated_linear, linear_add, quantize_rows
from .hip_kernels import traced
from .layer_ops import mcmoe_coef, norm_add, plain, situ_glu


def _weight_alone(linear) -> bool:
    """A projection that is no more than its weight."""
    return plain(linear, nn.Linear) and linear.bias is None


def _marks(linears) -> tuple:
    """Of each weight what tells a change: where its data lies, its version and its type."""
    return tuple((w.data_ptr(), -1 if w.is_inference() else w._version, w.dtype) for w in (m.weight for m in linears))


class SiTUGLU(nn.Module):
    """``[b1 tanh(W_g x / b1) sigmoid(W_g x)] * [b2 tanh(W_u x / b2)]`` (activations.py:8-31).

    ``fuse_products = True`` takes both projections, the activations and their product as one kernel, in training too
    (:func:`~verace_amd.gated_linear`); the projections are then not rounded in between, so results differ from the separate
    ops' by their rounding.  Under autocast, and where a projection is more than its weight (another class, a bias, hooks), the
    separate ops run all the same."""

    fuse_products = False

    def __init__(self, in_features: int, hidden_features: int, beta1: float = 4.0,
                 beta2: float = 25.0):
        super().__init__()
        self.in_features = in_features
        self.hidden_features = hidden_features
        self.beta1 = beta1
        self.beta2 = beta2
        self.w_gate = nn.Linear(in_features, hidden_features, bias=False)
        self.w_up = nn.Linear(in_features, hidden_features, bias=False)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if (self.fuse_products and not torch.is_autocast_enabled("cuda") and _weight_alone(self.w_gate)
                and _weight_alone(self.w_up)):
            return gated_linear(x, self.w_gate.weight, self.w_up.weight, beta1=self.beta1, beta2=self.beta2)
        g = self.w_gate(x)
        u = self.w_up(x)
        return situ_glu(g, u, self.beta1, self.beta2)


class ManifoldContinuousMoE(nn.Module):
    _base8 = None        # the held weights: (q, scale) of the gate's, the up and the down projection
    _base8_of = None     # what the weights were then (_marks)
    _in_8_bits = False   # whether the base path takes them

    def __init__(self, hidden_dim: int = 16384, rank: int = 32, num_components: int = 64,
                 top_k_components: int = 8, beta1: float = 4.0, beta2: float = 25.0):
        super().__init__()
        self.hidden_dim = hidden_dim
        self.rank = rank
        self.num_components = num_components
        self.top_k_components = top_k_components
        self.base_situ_glu = SiTUGLU(hidden_dim, hidden_dim * 2, beta1=beta1, beta2=beta2)
        self.base_w_down = nn.Linear(hidden_dim * 2, hidden_dim, bias=False)
        self.u_basis = nn.Parameter(torch.randn(num_components, hidden_dim, rank) * 0.02)
        self.v_basis = nn.Parameter(torch.randn(num_components, rank, hidden_dim) * 0.02)
        self.router = nn.Linear(hidden_dim, num_components, bias=False)
        self.hyper_sigma = nn.Linear(hidden_dim, num_components * rank, bias=False)
        self.norm = nn.RMSNorm(hidden_dim)

    def _base_linears(self):
        """The base path's three projections, for the path in 8 bits."""
        glu = self.base_situ_glu
        if plain(glu, SiTUGLU):
            linears = glu.w_gate, glu.w_up, self.base_w_down
            if all(_weight_alone(m) for m in linears):
                return linears
        raise RuntimeError("verace_amd.ManifoldContinuousMoE: the base path in 8 bits takes plain modules (SiTUGLU and nn.Linear, no "
                           "bias, no hooks); call quantize_base_(False) to run others")

    def quantize_base_(self, on: bool = True) -> "ManifoldContinuousMoE":
        """Holds the base path's three weights in 8 bits with a scale for each output channel and runs the path on rows in 8 bits, for
        inference (``on=False``: no longer).  The weights themselves stay, and a call that finds them changed in place, replaced or
        moved holds them anew.  A change through ``.data`` or in inference mode leaves no trace, and a captured graph or a traced call
        runs no check: after one, this is called again, outside a capture.  What is held keeps its place, while the path is off too,
        so that a graph captured on the 8-bit weights replays with the ones held last (until a move or a change of shape).  Not part of
        the ``state_dict``.  The path takes the weights alone: modules of another class, with a bias or with hooks are refused, here and
        where it runs."""
        if on:
            self._hold_base()
        self._in_8_bits = on
        return self

    def _hold_base(self) -> None:
        if torch.cuda.is_current_stream_capturing():  # which would run nothing now
            raise RuntimeError("verace_amd.ManifoldContinuousMoE: the weights are new or have changed; call quantize_base_() before the "
                               "capture")
        old, linears = self._base8, self._base_linears()
        with torch.inference_mode(False), torch.no_grad():  # tensors made in inference mode cannot be renewed outside it
            new = tuple(quantize_rows(m.weight.detach()) for m in linears)
            if old and all(o.shape == n.shape and o.device == n.device for (o, _), (n, _) in zip(old, new)):
                for pair, fresh in zip(old, new):
                    for t, n in zip(pair, fresh):
                        t.copy_(n)
                new = old
        # calls on other streams wait for the weights' change at most, not for this
        torch.cuda.current_stream(linears[0].weight.device).synchronize()
        self._base8, self._base8_of = new, _marks(linears)

    def _base_in_8_bits(self, xf: torch.Tensor) -> torch.Tensor:
        if torch.is_grad_enabled():
            raise RuntimeError("verace_amd.ManifoldContinuousMoE: the base path in 8 bits has no gradients; run under "
                               "torch.no_grad(), or call quantize_base_(False)")
        linears = self._base_linears()
        if not traced(xf) and _marks(linears) != self._base8_of:
            self._hold_base()
        (wg, sg), (wu, su), (wd, sd) = self._base8
        glu = self.base_situ_glu
        out = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else xf.dtype
        x, xs = quantize_rows(xf)
        h, hs = quantize_rows(gated_linear(x, wg, wu, xs, sg, su, beta1=glu.beta1, beta2=glu.beta2, out_dtype=out))
        return linear_add(h, wd, x_scale=hs, weight_scale=sd, out_dtype=out)

    def parts(self, x: torch.Tensor):
        """The base path and the manifold path before its norm, both [tokens, hidden]."""
        b, s, d = x.shape
        C, r = self.num_components, self.rank
        xf = x.reshape(b * s, d)
        base_out = self.base_w_down(self.base_situ_glu(xf)) if not self._in_8_bits else self._base_in_8_bits(xf)
        # v_proj[n, j, :] = V_j x_n for every component, then the selected ones' coefficients
        vproj = xf @ self.v_basis.reshape(C * r, d).t()
        coef = mcmoe_coef(self.router(xf), self.hyper_sigma(xf), vproj, min(self.top_k_components, C), C)
        return base_out, coef @ self.u_basis.permute(0, 2, 1).reshape(C * r, d)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        b, s, d = x.shape
        base_out, adapt = self.parts(x)
        return norm_add(adapt, self.norm, base_out)[0].view(b, s, d)
