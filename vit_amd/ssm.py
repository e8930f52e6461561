"""State-space sequence operators with autograd: the short causal convolution, the selective scan (whole sequences and one
token at a time) and the norms around a block, on librvit (csrc/ssm_conv.hip, ssm_scan.hip, ssm_scan_bwd.hip, sandwich.hip)
through the torch binding csrc/ssm_torch.cpp.  The temporal encoder's `model_type='ssm'` (vit_amd/sequence.py) is built of them.

Tensors live on one GPU; launches go to the current stream of that GPU.  Activations are bf16 or fp32, per-channel and per-
head parameters and kept scan states fp32.  Sums, states and statistics are fp32 or wider whatever the inputs.  Results do
not depend on the order in which workgroups run.  First derivatives in reverse mode only: dual tensors (forward mode) and
create_graph=True raise RuntimeError, as does torch.jit.trace.  Wrong shapes, types and devices raise ValueError, a CPU
tensor RuntimeError: there is no CPU path.  An empty batch, or no tokens, gives empty results and leaves states as they are.
Calls can be captured into graphs, training steps with their backward passes too (these only while no eager autograd graph of
the same leaves is alive, as for every torch operation)."""
from __future__ import annotations

import os
from typing import Optional

import torch

from . import _lib, ops

_ext = None


def _load():
    """The binding, loaded once; loud when it is absent or of another library."""
    global _ext
    _lib.load()
    try:
        from . import _ssm
    except ImportError as e:
        raise ImportError(f"vit_amd/_ssm.so ({os.path.dirname(__file__)}): {e}. Build it with `python -c 'import __graft_entry__ as g; "
                          "g.build()'` or `make -C vit_amd/csrc`. vit_amd has no fallback path.") from e
    if _ssm.abi() != _lib.ABI_VERSION:
        raise ImportError(f"_ssm.so is of ABI version {_ssm.abi()}, {_lib.ABI_VERSION} expected; rebuild the library")
    _ext = _ssm
    return _ssm


def _profiled(name: str, flops: int, tensors, fn, *args):
    """Under ops.set_profiler: a span around the call's launches (a backward pass has none)."""
    with ops._Span(name, flops, sum(t.numel() * t.element_size() for t in tensors if t is not None)):
        return fn(*args)


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, activation: Optional[str] = None,
                state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None, return_state: bool = False):
    """act(bias + sum_k weight[:, k] x[:, t - K + 1 + k]) for every token t: x bf16 / fp32 [B,T,C], weight fp32 [C,K] (K: 2..6),
    bias fp32 [C], activation None or 'silu'.  `state` [B,K-1,C] (x's dtype): the inputs before the first token (default: zero).
    `lengths` int32 [B]: sample b ends after lengths[b] tokens (held to 0..T); behind it y is zero and nothing of x counts.
    return_state=True also returns the last K-1 inputs before each sample's end (what causal_conv_step goes on from)."""
    args = (x, weight, bias, _silu(activation), state, lengths, return_state)
    fn = (_ext or _load()).conv
    y, after = fn(*args) if ops._PROF is None else _profiled("ssm_conv_fwd", 2 * x.numel() * weight.shape[1], (x, x), fn, *args)
    return (y, after) if return_state else y


def causal_conv_step(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], state: torch.Tensor, *,
                     activation: Optional[str] = None) -> torch.Tensor:
    """causal_conv for one token: x [B,C], state [B,K-1,C] (advances in place); returns [B,C].  No gradient: in grad
    mode an input that requires one raises RuntimeError."""
    args = (x, weight, bias, state, _silu(activation))
    fn = (_ext or _load()).conv_step
    return fn(*args) if ops._PROF is None else _profiled("ssm_conv_step", 2 * x.numel() * weight.shape[1], (x, x, state, state), fn, *args)


def _silu(activation) -> bool:
    if activation is None:
        return False
    if activation != "silu":
        raise ValueError(f"causal_conv: activation {activation!r} (None or 'silu')")
    return True


def selective_scan(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, Bm: torch.Tensor, Cm: torch.Tensor, *,
                   D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None,
                   state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None, return_state: bool = False):
    """Selective state-space scan over the tokens of each sample, per head h (its group's Bm, Cm):
        d = softplus(dt + dt_bias);  S_t = exp(d_t A) S_{t-1} + d_t x_t Bm_t^T;  y_t = (S_t Cm_t + D x_t) * silu(z_t)
    x, z bf16 / fp32 [B,T,H,P]; dt [B,T,H]; Bm, Cm [B,T,G,N], H a multiple of G, N <= 128 (one dtype; slices of wider tensors
    are taken as they are where a token's heads and channels are packed, and copied otherwise); A, D, dt_bias fp32 [H]; state
    fp32 [B,H,P,N] (default: zero).  `lengths` int32 [B]: sample b ends after lengths[b] tokens (held to 0..T); behind it y is
    zero and nothing of the inputs counts.  return_state=True also returns the state behind each sample's last token, fp32
    (what selective_scan_step goes on from).  A non-finite input may reach every output of its chunk of 64 tokens and
    everything behind it."""
    args = (x, dt, A, Bm, Cm, D, z, dt_bias, state, lengths, return_state)
    fn = (_ext or _load()).scan
    y, after = fn(*args) if ops._PROF is None else _profiled("ssm_scan_fwd", x.numel() * (5 * Bm.shape[-1] + 6), (x, dt, Bm, Cm, z, x, state),
                                                             fn, *args)
    return (y, after) if return_state else y


def selective_scan_step(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, Bm: torch.Tensor, Cm: torch.Tensor, state: torch.Tensor, *,
                        D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                        dt_bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """selective_scan for one token: x, z [B,H,P], dt [B,H], Bm, Cm [B,G,N], state fp32 [B,H,P,N] (advances in place); returns
    [B,H,P].  No gradient: in grad mode an input that requires one raises RuntimeError."""
    args = (x, dt, A, Bm, Cm, state, D, z, dt_bias)
    fn = (_ext or _load()).scan_step
    return fn(*args) if ops._PROF is None else _profiled("ssm_scan_step", x.numel() * (5 * Bm.shape[-1] + 6), (x, dt, Bm, Cm, z, x, state, state),
                                                         fn, *args)


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
    if isinstance(scale, torch.Tensor):
        raise ValueError("sandwich_norm: scale must be a number (a tensor's gradient would be lost: a learned scale belongs into the gate)")
    rms = kind == "rms"
    if rms and (post_bias is not None or pre_bias is not None):
        raise ValueError("sandwich_norm: kind 'rms' has no biases")
    args = (residual, y, post_weight, post_bias, pre_weight, pre_bias, gate, scale, rms, eps)
    fn = (_ext or _load()).sandwich
    return fn(*args) if ops._PROF is None else _profiled("sandwich_norm_fwd", 20 * y.numel(), (residual, y, residual, y), fn, *args)
