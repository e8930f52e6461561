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
    """-> (y, state behind each sample's last token).  A, D, dt_bias: [H], or spread out over [B,T,H,P,N] / [B,T,H,P] (D), so
    that their gradients are the terms whose sums are a head's gradients."""
    B, T, H, P = x.shape
    G, N = Bm.shape[2:]
    heads = torch.arange(H) // (H // G)
    n, live = _live(lengths, B, T)
    zero = torch.zeros((), dtype=x.dtype)
    mask = lambda v: None if v is None else torch.where(live.reshape(B, T, *[1] * (v.dim() - 2)), v, zero)  # noqa: E731
    x, dt, Bm, Cm, z = (mask(v) for v in (x, dt, Bm, Cm, z))
    at = lambda v, t: v[:, t] if v.dim() == 5 else v[:, None, None]  # noqa: E731
    S = x.new_zeros(B, H, P, N) if state is None else state
    ys = []
    for t in range(T):
        raw = dt[:, t, :, None, None]
        if dt_bias is not None:
            raw = raw + at(dt_bias, t)
        d = torch.logaddexp(raw, torch.zeros_like(raw))      # softplus, for any argument
        new = torch.exp(d * at(A, t)) * S + d * x[:, t, ..., None] * Bm[:, t, heads][:, :, None]
        S = torch.where(live[:, t, None, None, None], new, S)
        v = (S * Cm[:, t, heads][:, :, None]).sum(-1)
        if D is not None:
            v = v + (D[:, t] if D.dim() == 4 else D[:, None]) * x[:, t]
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


def ssm_stack(p, x, layers, inner, states, head=64, spread=None):
    """The temporal encoder's model_type='ssm' (vit_amd/sequence.py SSMStack) on a dict of its parameters: [B,T,In] -> [B,T,hidden].
    `spread` (a dict): gets A, D and dt_bias of every layer spread out over their terms (selective_scan)."""
    heads = inner // head
    h = x @ p["weight_embed"].t() + p["bias_embed"]
    n = norm(h, p["pre_weight_l0"], p["pre_bias_l0"], "layer", 1e-5)
    for k in range(layers):
        g = lambda name: p[f"{name}_l{k}"]  # noqa: B023,E731
        xbc, z, dt = torch.split(n @ g("in_proj").t(), [inner + 2 * states, inner, heads], dim=-1)
        u, _ = causal_conv(xbc, g("conv_weight"), g("conv_bias"), silu=True)
        xs, Bm, Cm = torch.split(u, [inner, states, states], dim=-1)
        per = {"A_log": g("A_log"), "D": g("D"), "dt_bias": g("dt_bias")}
        if spread is not None:
            B, T = x.shape[:2]
            for name in per:
                v = per[name][:, None, None].expand(B, T, heads, head, states) if name != "D" else per[name][:, None].expand(B, T, heads, head)
                spread[f"{name}_l{k}"] = per[name] = v.detach().clone().requires_grad_()
        y, _ = selective_scan(xs.unflatten(-1, (heads, head)), dt, -torch.exp(per["A_log"]), Bm.unsqueeze(2), Cm.unsqueeze(2), D=per["D"],
                              z=z.unflatten(-1, (heads, head)), dt_bias=per["dt_bias"])
        h, n = sandwich_norm(h, y.flatten(2) @ g("out_proj").t(), g("post_weight"), g("post_bias"), p[f"pre_weight_l{k + 1}"],
                             p[f"pre_bias_l{k + 1}"], gate=g("gate"))
    return n
