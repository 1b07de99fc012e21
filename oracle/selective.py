"""The selective state space layer's operators from their definitions, in 64 bits and token by token:
differentiable torch code on any device, for small sizes."""
import torch


def _d(t):
    return None if t is None else t.double()


def _on(B, T, lengths, device):
    if lengths is None:
        return torch.ones(B, T, dtype=torch.bool, device=device)
    return torch.arange(T, device=device) < lengths.to(device).view(B, 1)


def selective_scan(x, delta, A, B, C, D=None, delta_bias=None, softplus=True, initial_state=None, lengths=None,
                   magnitude=False):
    """d = softplus(delta + bias), S = exp(d A) S + d x B^T, y = S C + D x; (y, S).  With ``magnitude`` the
    sums of the terms' absolute values: what rounding errors of the products scale with."""
    x, delta, A, B, C, D, delta_bias, S = (_d(t) for t in (x, delta, A, B, C, D, delta_bias, initial_state))
    b, T, H, P = x.shape
    delta = delta.reshape(b, T, H)
    r = H // B.shape[2]
    on = _on(b, T, lengths, x.device)
    z = delta if delta_bias is None else delta + delta_bias
    d = torch.logaddexp(z, torch.zeros_like(z)) if softplus else z
    if magnitude:
        x, B, C = x.abs(), B.abs(), C.abs()
        D = None if D is None else D.abs()
        S = None if S is None else S.abs()
    S = x.new_zeros(b, H, P, B.shape[-1]) if S is None else S
    B, C = B.repeat_interleave(r, 2), C.repeat_interleave(r, 2)
    ys = []
    for t in range(T):
        live = on[:, t].view(b, 1, 1, 1)
        dt, xt = d[:, t, :, None, None], x[:, t].unsqueeze(-1)
        w = dt.abs() if magnitude else dt
        new = torch.exp(dt * A[:, None, None]) * S + w * xt * B[:, t].unsqueeze(2)
        S = torch.where(live, new, S)
        y = (S * C[:, t].unsqueeze(2)).sum(-1)
        if D is not None:
            y = y + D[:, None] * x[:, t]
        ys.append(torch.where(live[..., 0], y, torch.zeros_like(y)))
    y = torch.stack(ys, 1) if ys else x.new_zeros(b, 0, H, P)
    return y, S


def short_conv(x, weight, bias=None, initial_state=None, lengths=None, activation="silu", magnitude=False):
    """(y, the last K - 1 counted rows)."""
    x, w, bias, state = (_d(t) for t in (x, weight, bias, initial_state))
    B, T, C = x.shape
    K = w.shape[1]
    on = _on(B, T, lengths, x.device).unsqueeze(-1)
    x = torch.where(on, x, torch.zeros_like(x))
    rows = torch.cat([x.new_zeros(B, K - 1, C) if state is None else state, x], 1)
    if magnitude:
        return sum(rows[:, j:j + T].abs() * w[:, j].abs() for j in range(K)) + (0 if bias is None else bias.abs())
    z = sum(rows[:, j:j + T] * w[:, j] for j in range(K))
    z = z if bias is None else z + bias
    y = z * torch.sigmoid(z) if activation == "silu" else z
    n = [T] * B if lengths is None else [max(0, min(T, int(v))) for v in lengths]
    last = torch.stack([rows[i, n[i]:n[i] + K - 1] for i in range(B)]) if B else rows[:, :K - 1]
    return torch.where(on, y, torch.zeros_like(y)), last


def gated_norm_add(y, residual, norm_weight=None, gate=None, scale=None, next_weight=None, eps=1e-6, next_eps=None,
                   activation="silu"):
    """(s, n)."""
    y, residual, norm_weight, gate, scale, next_weight = (
        _d(t) for t in (y, residual, norm_weight, gate, scale, next_weight))
    r = y
    if norm_weight is not None:
        r = y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + eps) * norm_weight
    if gate is not None:
        r = r * torch.sigmoid(gate) * (gate if activation == "silu" else 1.0)
    s = residual + (r if scale is None else scale * r)
    if next_weight is None:
        return s, None
    return s, s * torch.rsqrt(s.pow(2).mean(-1, keepdim=True) + (eps if next_eps is None else next_eps)) * next_weight
