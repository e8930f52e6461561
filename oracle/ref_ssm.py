"""The state-space sequence operators from their definitions, token by token, in 64 bits on the CPU (differentiable): what
vit_amd/ssm.py is tested against."""
import torch


def _live(lengths, B, T):
    n = torch.full((B,), T) if lengths is None else lengths.cpu().long().clamp(0, T)
    return n, torch.arange(T)[None] < n[:, None]


def causal_conv(x, weight, bias=None, *, silu=False, state=None, lengths=None):
    """-> (y, last K-1 inputs before each sample's end)"""
    B, T, C = x.shape
    K = weight.shape[1]
    n, live = _live(lengths, B, T)
    x = torch.where(live[..., None], x, torch.zeros((), dtype=x.dtype))
    full = torch.cat([x.new_zeros(B, K - 1, C) if state is None else state, x], 1)
    u = sum(weight[:, k] * full[:, k:k + T] for k in range(K))
    if bias is not None:
        u = u + bias
    y = u * torch.sigmoid(u) if silu else u
    y = torch.where(live[..., None], y, torch.zeros((), dtype=x.dtype))
    return y, torch.stack([full[b, int(n[b]):int(n[b]) + K - 1] for b in range(B)])


def selective_scan(x, dt, A, Bm, Cm, *, D=None, z=None, dt_bias=None, state=None, lengths=None):
    """-> (y, state behind each sample's last token)"""
    B, T, H, P = x.shape
    G, N = Bm.shape[2:]
    heads = torch.arange(H) // (H // G)
    n, live = _live(lengths, B, T)
    zero = torch.zeros((), dtype=x.dtype)
    mask = lambda v: None if v is None else torch.where(live.reshape(B, T, *[1] * (v.dim() - 2)), v, zero)  # noqa: E731
    x, dt, Bm, Cm, z = (mask(v) for v in (x, dt, Bm, Cm, z))
    raw = dt if dt_bias is None else dt + dt_bias
    d = torch.logaddexp(raw, torch.zeros_like(raw))      # softplus, for any argument
    S = x.new_zeros(B, H, P, N) if state is None else state
    ys = []
    for t in range(T):
        new = torch.exp(d[:, t] * A)[..., None, None] * S + (d[:, t, :, None] * x[:, t])[..., None] * Bm[:, t, heads][:, :, None]
        S = torch.where(live[:, t, None, None, None], new, S)
        v = (S * Cm[:, t, heads][:, :, None]).sum(-1)
        if D is not None:
            v = v + D[:, None] * x[:, t]
        if z is not None:
            v = v * z[:, t] * torch.sigmoid(z[:, t])
        ys.append(torch.where(live[:, t, None, None], v, zero))
    return torch.stack(ys, 1) if ys else torch.zeros_like(x), S


def norm(v, weight, bias, kind, eps):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps) * weight
    return v if bias is None else v + bias


def sandwich_norm(residual, y, post_weight, post_bias, pre_weight, pre_bias, *, gate=None, scale=1.0, kind="layer", eps=1e-5):
    u = norm(y, post_weight, post_bias, kind, eps)
    if gate is not None:
        u = u * (gate[:, None] if gate.dim() == 2 and y.dim() == 3 else gate)
    h = residual + scale * u
    return h, norm(h, pre_weight, pre_bias, kind, eps)
