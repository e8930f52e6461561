"""State-space sequence operators with autograd: the short causal convolution, the selective scan (whole sequences and one
token at a time) and the norms around a block, on librvit (csrc/ssm_conv.hip, ssm_scan.hip, ssm_scan_bwd.hip, sandwich.hip).
The temporal encoder's `model_type='ssm'` (vit_amd/sequence.py) is built of them.

Tensors live on one GPU; launches go to the current stream of that GPU.  Activations are bf16 or fp32, per-channel and
per-head parameters and kept scan states fp32.  Sums, states and statistics are fp32 or wider whatever the inputs.  Results do
not depend on the order in which workgroups run.  There is no CPU path."""
from __future__ import annotations

import contextlib
from typing import Optional

import torch

from . import ops

F32 = torch.float32
_same = contextlib.nullcontext()


def _on(t: torch.Tensor):
    """The launch goes to the current device's stream: make t's device current where it is not."""
    return _same if not t.is_cuda or t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


def _packed(t: Optional[torch.Tensor], inner: int) -> Optional[torch.Tensor]:
    """t with its last `inner` dimensions packed (a copy only where they are not)."""
    if t is None:
        return None
    step = 1
    for d in range(1, inner + 1):
        if t.shape[-d] != 1 and t.stride(-d) != step:
            return t.contiguous()
        step *= t.shape[-d]
    return t


def _wants_grad(*ts: Optional[torch.Tensor]) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def _c(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return None if t is None else t.contiguous()


# ---- short causal convolution -------------------------------------------------------------------------------------------
def _conv_fwd(x, weight, bias, silu, state, lengths, want_state):
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    after = None
    if want_state:
        after = torch.empty(x.shape[0], max(weight.shape[-1] - 1, 0), x.shape[-1], dtype=x.dtype, device=x.device)
    if x.dim() == 3 and x.shape[1] == 0:     # no tokens: nothing runs, the kept inputs stay
        if want_state:
            after.zero_() if state is None else after.copy_(state)
        return y, after
    ops.ssm_conv(x, weight, bias, y, silu=silu, state=state, state_out=after, lengths=lengths)
    return y, after


class _Conv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, silu, state, lengths, want_state):
        with _on(x):
            y, after = _conv_fwd(x, weight, bias, silu, state, lengths, want_state)
        ctx.save_for_backward(x, weight, bias, state, lengths)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        return y, after

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dafter):
        x, weight, bias, state, lengths = ctx.saved_tensors
        with _on(x):
            dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            dw, db = torch.empty_like(weight), None if bias is None else torch.empty_like(bias)
            ds = None if state is None else torch.empty_like(state)
            dy = torch.zeros_like(dx) if dy is None else _packed(dy, 1)
            if x.shape[1] == 0:
                dw.zero_()
                if db is not None:
                    db.zero_()
                if ds is not None:
                    ds.zero_() if dafter is None else ds.copy_(dafter)
            else:
                ops.ssm_conv_bwd(x, weight, bias, dy, dx, dw, db, silu=ctx.silu, state=state, lengths=lengths, dstate_out=_c(dafter),
                                 dstate=ds)
        return dx, dw, db, None, ds, None, None


def _silu(activation) -> bool:
    if activation not in (None, "silu"):
        raise ValueError(f"causal_conv: activation {activation!r} (None or 'silu')")
    return activation == "silu"


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, activation: Optional[str] = None,
                state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None, return_state: bool = False):
    """act(bias + sum_k weight[:, k] x[:, t - K + 1 + k]) for every token t: x bf16 / fp32 [B,T,C], weight fp32 [C,K] (K: 2..6),
    bias fp32 [C], activation None or 'silu'.  `state` [B,K-1,C] (x's dtype): the inputs before the first token (default: zero).
    `lengths` int32 [B]: sample b ends after lengths[b] tokens; behind it y is zero and nothing of x counts.
    return_state=True also returns the last K-1 inputs before each sample's end (what causal_conv_step goes on from)."""
    silu = _silu(activation)
    x, weight, state = _packed(x, 1), _c(weight), _c(state)
    if _wants_grad(x, weight, bias, state):
        y, after = _Conv.apply(x, weight, bias, silu, state, lengths, return_state)
    else:
        with _on(x):
            y, after = _conv_fwd(x, weight, bias, silu, state, lengths, return_state)
    return (y, after) if return_state else y


@torch.no_grad()
def causal_conv_step(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], state: torch.Tensor, *,
                     activation: Optional[str] = None) -> torch.Tensor:
    """causal_conv for one token: x [B,C], state [B,K-1,C] (advances in place); returns [B,C].  No gradient."""
    with _on(x):
        x = _packed(x, 1)
        return ops.ssm_conv_step(x, weight, bias, state, torch.empty(x.shape, dtype=x.dtype, device=x.device), silu=_silu(activation))


# ---- selective scan -----------------------------------------------------------------------------------------------------
def _scan_fwd(x, dt, A, Bm, Cm, D, z, dt_bias, state, lengths, want_state, train):
    ops._scan_shapes("selective_scan", x, dt, A, Bm, Cm, D, z, dt_bias, False)
    B, T, H, P = x.shape
    G, N = Bm.shape[-2:]
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    after = torch.empty(B, H, P, N, dtype=F32, device=x.device) if want_state else None
    v = torch.empty_like(y) if train and z is not None else None
    states = torch.empty(ops.ssm_scan_plan(B, T, H, P, G, N)[1], dtype=F32, device=x.device) if train else None
    ops.ssm_scan(x, dt, A, Bm, Cm, D, z, dt_bias, y, state=state, state_out=after, lengths=lengths, v=v, states=states)
    return y, after, v, states


class _Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, Bm, Cm, D, z, dt_bias, state, lengths, want_state):
        with _on(x):
            y, after, v, states = _scan_fwd(x, dt, A, Bm, Cm, D, z, dt_bias, state, lengths, want_state, True)
        ctx.save_for_backward(x, dt, A, Bm, Cm, D, z, dt_bias, lengths, v, states)
        ctx.had_state = state is not None
        ctx.set_materialize_grads(False)
        return y, after

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dafter):
        x, dt, A, Bm, Cm, D, z, dt_bias, lengths, v, states = ctx.saved_tensors
        with _on(x):
            new = lambda t: None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device)  # noqa: E731
            dx, ddt, dA, dB, dC, dD, dz, dbias = (new(t) for t in (x, dt, A, Bm, Cm, D, z, dt_bias))
            B, T, H, P = x.shape
            ds = torch.empty(B, H, P, Bm.shape[-1], dtype=F32, device=x.device) if ctx.had_state else None
            if T == 0:
                for t in (dA, dD, dbias):
                    if t is not None:
                        t.zero_()
                if ds is not None:
                    ds.zero_() if dafter is None else ds.copy_(dafter)
            else:
                dy = torch.zeros_like(dx) if dy is None else _packed(dy, 2)
                ops.ssm_scan_bwd(x, dt, A, Bm, Cm, D, z, dt_bias, v, states, dy, dx, ddt, dA, dB, dC, dD, dz, dbias, lengths=lengths,
                                 dstate_out=_c(dafter), dstate=ds)
        return dx, ddt, dA, dB, dC, dD, dz, dbias, ds, None, None


def selective_scan(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, Bm: torch.Tensor, Cm: torch.Tensor, *,
                   D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None,
                   state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None, return_state: bool = False):
    """Selective state-space scan over the tokens of each sample, per head h (its group's Bm, Cm):
        d = softplus(dt + dt_bias);  S_t = exp(d_t A) S_{t-1} + d_t x_t Bm_t^T;  y_t = (S_t Cm_t + D x_t) * silu(z_t)
    x, z bf16 / fp32 [B,T,H,P]; dt [B,T,H]; Bm, Cm [B,T,G,N], H a multiple of G, N <= 128 (one dtype; slices of wider tensors
    are taken as they are where a token's heads and channels are packed); A, D, dt_bias fp32 [H]; state fp32 [B,H,P,N] (default:
    zero).  `lengths` int32 [B]: sample b ends after lengths[b] tokens; behind it y is zero and nothing of the inputs counts.
    return_state=True also returns the state behind each sample's last token, fp32 (what selective_scan_step goes on from).
    A non-finite input may reach every output of its chunk of 64 tokens and everything behind it."""
    x, z, Bm, Cm, dt = _packed(x, 2), _packed(z, 2), _packed(Bm, 2), _packed(Cm, 2), _packed(dt, 1)
    state = _c(state)
    if _wants_grad(x, dt, A, Bm, Cm, D, z, dt_bias, state):
        y, after = _Scan.apply(x, dt, A, Bm, Cm, D, z, dt_bias, state, lengths, return_state)
    else:
        with _on(x):
            y, after, _, _ = _scan_fwd(x, dt, A, Bm, Cm, D, z, dt_bias, state, lengths, return_state, False)
    return (y, after) if return_state else y


@torch.no_grad()
def selective_scan_step(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, Bm: torch.Tensor, Cm: torch.Tensor, state: torch.Tensor, *,
                        D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                        dt_bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """selective_scan for one token: x, z [B,H,P], dt [B,H], Bm, Cm [B,G,N], state fp32 [B,H,P,N] (advances in place); returns
    [B,H,P].  No gradient."""
    with _on(x):
        x, z, Bm, Cm, dt = _packed(x, 2), _packed(z, 2), _packed(Bm, 2), _packed(Cm, 2), _packed(dt, 1)
        return ops.ssm_scan_step(x, dt, A, Bm, Cm, D, z, dt_bias, state, torch.empty(x.shape, dtype=x.dtype, device=x.device))


# ---- norms around a block -----------------------------------------------------------------------------------------------
def _sandwich_fwd(residual, y, pw, pb, nw, nb, gate, scale, rms, eps, train):
    h = torch.empty(residual.shape, dtype=residual.dtype, device=residual.device)
    n = torch.empty(y.shape, dtype=y.dtype, device=y.device)
    stats = torch.empty(y.numel() // max(y.shape[-1], 1), 4, dtype=F32, device=y.device) if train else None
    if y.numel():
        ops.sandwich_norm(residual, y, pw, pb, nw, nb, h, n, gate=gate, scale=scale, rms=rms, eps=eps, stats=stats)
    return h, n, stats


class _Sandwich(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, y, pw, pb, nw, nb, gate, scale, rms, eps):
        with _on(y):
            h, n, stats = _sandwich_fwd(residual, y, pw, pb, nw, nb, gate, scale, rms, eps, True)
        ctx.save_for_backward(residual, y, pw, pb, nw, nb, gate, stats)
        ctx.consts = (scale, rms, eps)
        return h, n

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dn):
        residual, y, pw, pb, nw, nb, gate, stats = ctx.saved_tensors
        scale, rms, eps = ctx.consts
        with _on(y):
            new = lambda t: None if t is None else torch.empty_like(t)  # noqa: E731
            dres, dy, dpw, dpb, dnw, dnb, dg = (new(t) for t in (residual, y, pw, pb, nw, nb, gate))
            if y.numel():
                ops.sandwich_norm_bwd(residual, y, pw, pb, nw, nb, stats, dh.contiguous(), dn.contiguous(), dres, dy, dpw, dpb, dnw, dnb,
                                      gate=gate, dgate=dg, scale=scale, rms=rms, eps=eps)
            else:
                for t in (dpw, dpb, dnw, dnb, dg):
                    if t is not None:
                        t.zero_()
        return dres, dy, dpw, dpb, dnw, dnb, dg, None, None, None


def sandwich_norm(residual: torch.Tensor, y: torch.Tensor, post_weight: torch.Tensor, post_bias: Optional[torch.Tensor],
                  pre_weight: torch.Tensor, pre_bias: Optional[torch.Tensor], *, gate: Optional[torch.Tensor] = None, scale: float = 1.0,
                  kind: str = "layer", eps: float = 1e-5):
    """The norm behind a block, its gate, the residual connection and the norm before the next block, in one pass:
        h = residual + scale * gate * norm_post(y);   n = norm_pre(h);   returns (h, n)
    residual and y bf16 / fp32 [..., E] (E <= 4096; h has residual's dtype, n has y's; n is taken from h before its rounding);
    weights and biases fp32 [E]; kind 'layer' (LayerNorm) or 'rms' (no centring, no biases); gate None, [E], [B,E] (with y
    [B,T,E]: one per sample) or like y, fp32 or y's dtype; scale a number."""
    if kind not in ("layer", "rms"):
        raise ValueError(f"sandwich_norm: kind {kind!r} ('layer' or 'rms')")
    if kind == "rms" and (post_bias is not None or pre_bias is not None):
        raise ValueError("sandwich_norm: kind 'rms' has no biases")
    args = (_c(residual), _c(y), post_weight, post_bias, pre_weight, pre_bias, _c(gate), float(scale), kind == "rms", float(eps))
    ops._sandwich_shapes("sandwich_norm", args[0], args[1], args[6], *args[2:6])
    if _wants_grad(*args[:7]):
        return _Sandwich.apply(*args)
    with _on(y):
        return _sandwich_fwd(*args, False)[:2]
