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
    dev = t.get_device()
    return _same if dev < 0 or dev == ops._raw_device() else torch.cuda.device(dev)


def _packed(t: Optional[torch.Tensor], inner: int) -> Optional[torch.Tensor]:
    """t with its last `inner` dimensions packed (a copy only where they are not)."""
    if t is None:
        return None
    step = 1
    for d in range(1, min(inner, t.dim()) + 1):
        if t.shape[-d] != 1 and t.stride(-d) != step:
            return t.contiguous()
        step *= t.shape[-d]
    return t


def _wants_grad(*ts: Optional[torch.Tensor]) -> bool:
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


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
                ops._ssm_conv_bwd(x, weight, bias, dy, dx, dw, db, ctx.silu, state, lengths, _c(dafter), ds)
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


def causal_conv_step(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], state: torch.Tensor, *,
                     activation: Optional[str] = None) -> torch.Tensor:
    """causal_conv for one token: x [B,C], state [B,K-1,C] (advances in place); returns [B,C].  No gradient."""
    silu = _silu(activation)
    sig = ops._sig("ssm_conv_step", x, weight, bias, state)
    if sig not in ops._SEEN:
        x, sig = _packed(x, 1), None
    with _on(x):
        return ops.ssm_conv_step(x, weight, bias, state, silu=silu, sig=sig)


# ---- selective scan -----------------------------------------------------------------------------------------------------
def _scan_fwd(x, dt, A, Bm, Cm, D, z, dt_bias, state, lengths, want_state, train, sig=None):
    after = v = states = None
    if want_state or train:
        ops._scan_shapes("selective_scan", x, dt, A, Bm, Cm, D, z, dt_bias, False) if sig is None else None
        B, T, H, P = x.shape
        G, N = Bm.shape[-2:]
        if want_state:
            after = torch.empty((B, H, P, N), dtype=F32, device=x.device)
        if train:
            v = None if z is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
            states = torch.empty(ops.ssm_scan_plan(B, T, H, P, G, N)[1], dtype=F32, device=x.device)
    y = ops.ssm_scan(x, dt, A, Bm, Cm, D, z, dt_bias, state=state, state_out=after, lengths=lengths, v=v, states=states, sig=sig)
    return y, after, v, states


class _Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, Bm, Cm, D, z, dt_bias, state, lengths, want_state, sig):
        with _on(x):
            y, after, v, states = _scan_fwd(x, dt, A, Bm, Cm, D, z, dt_bias, state, lengths, want_state, True, sig)
        ctx.save_for_backward(x, dt, A, Bm, Cm, D, z, dt_bias, lengths, v, states)
        ctx.had_state = state is not None
        ctx.set_materialize_grads(False)
        return y, after

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dafter):
        x, dt, A, Bm, Cm, D, z, dt_bias, lengths, v, states = ctx.saved_tensors
        with _on(x):
            T, kind, dev = x.shape[1], x.dtype, x.device
            dx, ddt = torch.empty(x.shape, dtype=kind, device=dev), torch.empty(dt.shape, dtype=kind, device=dev)
            dB, dC = torch.empty(Bm.shape, dtype=kind, device=dev), torch.empty(Cm.shape, dtype=kind, device=dev)
            dz = None if z is None else torch.empty(x.shape, dtype=kind, device=dev)
            dA = torch.empty_like(A)
            dD, dbias = None if D is None else torch.empty_like(D), None if dt_bias is None else torch.empty_like(dt_bias)
            ds = torch.empty((x.shape[0], *x.shape[2:], Bm.shape[-1]), dtype=F32, device=dev) if ctx.had_state else None
            if T == 0:
                for t in (dA, dD, dbias):
                    if t is not None:
                        t.zero_()
                if ds is not None:
                    ds.zero_() if dafter is None else ds.copy_(dafter)
            else:
                dy = torch.zeros_like(dx) if dy is None else _packed(dy, 2)
                ops._ssm_scan_bwd(x, dt, A, Bm, Cm, D, z, dt_bias, v, states, dy, dx, ddt, dA, dB, dC, dD, dz, dbias, lengths, _c(dafter), ds)
        return dx, ddt, dA, dB, dC, dD, dz, dbias, ds, None, None, None


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
    sig = ops._sig("ssm_scan", x, dt, A, Bm, Cm, D, z, dt_bias, state, lengths)
    if sig not in ops._SEEN:
        x, z, Bm, Cm, dt, state = _packed(x, 2), _packed(z, 2), _packed(Bm, 2), _packed(Cm, 2), _packed(dt, 1), _c(state)
        sig = None
    if _wants_grad(x, dt, A, Bm, Cm, D, z, dt_bias, state):
        y, after = _Scan.apply(x, dt, A, Bm, Cm, D, z, dt_bias, state, lengths, return_state, sig)
    else:
        with _on(x):
            y, after, _, _ = _scan_fwd(x, dt, A, Bm, Cm, D, z, dt_bias, state, lengths, return_state, False, sig)
    return (y, after) if return_state else y


def selective_scan_step(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, Bm: torch.Tensor, Cm: torch.Tensor, state: torch.Tensor, *,
                        D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                        dt_bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """selective_scan for one token: x, z [B,H,P], dt [B,H], Bm, Cm [B,G,N], state fp32 [B,H,P,N] (advances in place); returns
    [B,H,P].  No gradient."""
    sig = ops._sig("ssm_scan_step", x, dt, A, Bm, Cm, D, z, dt_bias, state)
    if sig not in ops._SEEN:
        x, z, Bm, Cm, dt, sig = _packed(x, 2), _packed(z, 2), _packed(Bm, 2), _packed(Cm, 2), _packed(dt, 1), None
    with _on(x):
        return ops.ssm_scan_step(x, dt, A, Bm, Cm, D, z, dt_bias, state, sig=sig)


# ---- norms around a block -----------------------------------------------------------------------------------------------
def _sandwich_fwd(residual, y, pw, pb, nw, nb, gate, scale, rms, eps, kind, train):
    stats = None
    if train:
        stats = torch.empty((y.numel() // max(y.shape[-1], 1), 4), dtype=F32, device=y.device)
    if y.numel() == 0:
        return torch.empty_like(residual), torch.empty_like(y), stats
    return (*ops.sandwich_norm(residual, y, pw, pb, nw, nb, gate=gate, scale=scale, rms=rms, eps=eps, stats=stats, kind=kind), stats)


class _Sandwich(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, y, pw, pb, nw, nb, gate, scale, rms, eps, kind):
        with _on(y):
            h, n, stats = _sandwich_fwd(residual, y, pw, pb, nw, nb, gate, scale, rms, eps, kind, True)
        ctx.save_for_backward(residual, y, pw, pb, nw, nb, gate, stats)
        ctx.consts = (scale, rms, eps, kind)
        return h, n

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dn):
        residual, y, pw, pb, nw, nb, gate, stats = ctx.saved_tensors
        with _on(y):
            dres, dy, dpw, dnw = torch.empty_like(residual), torch.empty_like(y), torch.empty_like(pw), torch.empty_like(nw)
            dpb, dnb = None if pb is None else torch.empty_like(pb), None if nb is None else torch.empty_like(nb)
            dg = None if gate is None else torch.empty_like(gate)
            if y.numel():
                ops._sandwich_norm_bwd(residual, y, pw, pb, nw, nb, stats, dh.contiguous(), dn.contiguous(), dres, dy, dpw, dpb, dnw, dnb, gate, dg,
                                       *ctx.consts)
            else:
                for t in (dpw, dpb, dnw, dnb, dg):
                    if t is not None:
                        t.zero_()
        return dres, dy, dpw, dpb, dnw, dnb, dg, None, None, None, None


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
    residual, y, gate = residual.contiguous(), y.contiguous(), _c(gate)
    gate_kind = ops._sandwich_kind("sandwich_norm", residual, y, gate, post_weight, post_bias, pre_weight, pre_bias)
    args = (residual, y, post_weight, post_bias, pre_weight, pre_bias, gate, float(scale), kind == "rms", float(eps), gate_kind)
    if _wants_grad(residual, y, post_weight, post_bias, pre_weight, pre_bias, gate):
        return _Sandwich.apply(*args)
    with _on(y):
        return _sandwich_fwd(*args, False)[:2]
