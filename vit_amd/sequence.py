"""Sequence model of the reference: CNN-ViT per frame + bidirectional LSTM across frames +
classifier, with the streaming wrapper -- `TemporalEncoder` / `CNNViTSequence` (train_vit.py:188-318,
infer.py:186-265) and `StreamingClassifier` (infer.py:479-630) -- on librvit.

The modules only HOLD parameters, under the reference's state_dict names (`spatial_encoder.*`,
`temporal_encoder.rnn.weight_ih_l0[_reverse]` ..., `classifier.0/.3.*`), so a `cnn_vit_lstm_radar.pt` checkpoint
loads unchanged.  Arithmetic:
  * frames -> features: `CNNViTHybrid.forward_features` (engine / training engine of this package);
  * LSTM / GRU: one fused HIP launch per time step for both directions (csrc/lstm.hip, fp32 straight from the fp32
    parameters), the step's backward likewise; weight / bias / input gradients from the saved gate gradients
    with the package's GEMM kernels;
  * classifier: the same fused GEMM epilogues as the single-frame head.
Both `model_type='lstm'` (the reference default, train_vit.py:267) and 'gru' are built.  `model_type='ssm'` is this package's
own third form: a stack of state-space layers (vit_amd/ssm.py), which trains over the frames of a window in parallel and, in
streaming, goes on from a kept state of fixed size, one frame at a time, instead of running the window again.
There is no CPU path.
"""
from __future__ import annotations

import math
import time
from collections import deque
from dataclasses import dataclass
from typing import Dict, List, Optional, Tuple

import numpy as np
import torch
import torch.nn as nn

from . import _lib, ops, ssm
from .model import CNNViTHybrid, _Linear
from .ops import _ptr, _stream, check

BF16 = torch.bfloat16
F32 = torch.float32
_M64 = (1 << 64) - 1


class _LSTMParams(nn.Module):
    """Parameter holder with nn.LSTM's / nn.GRU's names, shapes and default init (uniform +-1/sqrt(hidden));
    `gates` = 4 (LSTM: i,f,g,o) or 3 (GRU: r,z,n)."""

    def __init__(self, input_dim: int, hidden: int, num_layers: int, bidirectional: bool, gates: int = 4):
        super().__init__()
        self.input_size, self.hidden_size, self.num_layers, self.bidirectional = input_dim, hidden, num_layers, bidirectional
        self.gates = gates
        k = 1.0 / math.sqrt(hidden)
        ndir = 2 if bidirectional else 1
        for layer in range(num_layers):
            fin = input_dim if layer == 0 else hidden * ndir
            for sfx in ("", "_reverse")[:ndir]:
                for name, shape in ((f"weight_ih_l{layer}{sfx}", (gates * hidden, fin)),
                                    (f"weight_hh_l{layer}{sfx}", (gates * hidden, hidden)),
                                    (f"bias_ih_l{layer}{sfx}", (gates * hidden,)), (f"bias_hh_l{layer}{sfx}", (gates * hidden,))):
                    self.register_parameter(name, nn.Parameter(torch.empty(shape).uniform_(-k, k)))

    def direction(self, layer: int, rev: bool):
        s = "_reverse" if rev else ""
        return tuple(getattr(self, f"{n}_l{layer}{s}") for n in ("weight_ih", "weight_hh", "bias_ih", "bias_hh"))


class _Linear16(torch.autograd.Function):
    """y = x @ w.T (+ bias) on bf16 operands (fp32 accumulation, bf16 result): x [rows,K] bf16, w fp32 [N,K]."""

    @staticmethod
    def forward(ctx, x, w, bias):
        N, K = w.shape
        Np = 8 * ((N + 7) // 8)                 # the weight-gradient kernel takes whole groups of 8 rows
        w16 = w.detach().to(BF16)
        if Np != N:
            w16 = torch.cat([w16, w16.new_zeros(Np - N, K)])
        y = torch.empty(x.shape[0], Np, dtype=BF16, device=x.device)
        b = bias if bias is None or Np == N else torch.cat([bias.detach(), bias.new_zeros(Np - N)])
        ops.gemm(x, w16, y, bias=None if b is None else b.detach())
        ctx.save_for_backward(x, w16)
        ctx.n, ctx.has_bias = N, bias is not None
        return y if Np == N else y[:, :N]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w16 = ctx.saved_tensors
        N, (Np, K) = ctx.n, w16.shape
        with torch.cuda.device(x.device):
            if Np != N:
                dyp = dy.new_zeros(dy.shape[0], Np)
                dyp[:, :N] = dy
                dy = dyp
            dy = dy.contiguous()
            dx = torch.empty_like(x)
            ops.gemm(dy, w16.t().contiguous(), dx)
            dw = torch.zeros(N, K, dtype=F32, device=x.device)
            ops.wgrad(dy, x, dw, n_store=N)
            db = None
            if ctx.has_bias:
                db = torch.zeros(Np, dtype=F32, device=x.device)
                ops.colsum(dy, db)
                db = db[:N].contiguous()
        return dx, dw, db


class _Norm16(torch.autograd.Function):
    """LayerNorm of fp32 rows to bf16 (the norm before the first layer, which has no block in front of it)."""

    @staticmethod
    def forward(ctx, x, weight, bias):
        rows = x.shape[0]
        y = torch.empty(x.shape, dtype=BF16, device=x.device)
        mean, rstd = (torch.empty(rows, dtype=F32, device=x.device) for _ in range(2))
        ops.layernorm(x, weight.detach(), bias.detach(), y, mean=mean, rstd=rstd)
        ctx.save_for_backward(x, weight, mean, rstd)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        with torch.cuda.device(x.device):
            dx = torch.empty_like(x)
            dw, db = torch.zeros_like(weight), torch.zeros_like(weight)
            ops.layernorm_bwd(dy.contiguous(), x, mean, rstd, weight, dx, dw, db, accumulate=False)
        return dx, dw, db


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed):
        ctx.p, ctx.seed = p, seed
        return ops.dropout_apply(x, torch.empty_like(x), p, seed)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        with torch.cuda.device(dy.device):
            dy = dy.contiguous()
            return ops.dropout_apply(dy, torch.empty_like(dy), ctx.p, ctx.seed), None, None


class SSMStack(nn.Module):
    """Layers of n -> in_proj -> short causal convolution (SiLU) of x, B, C -> selective scan, gated -> out_proj, each followed
    by the norm behind it, its gate, the residual connection and the norm before the next in one pass (ssm.sandwich_norm).
    Inner width 2 x hidden in heads of 64 channels, one group of B and C.  The residual stream is fp32, activations bf16,
    parameters fp32."""

    HEAD, WINDOW = 64, 4

    def __init__(self, input_dim: int, hidden: int, num_layers: int, states: int = 64):
        super().__init__()
        self.input_size, self.hidden_size, self.num_layers, self.states = input_dim, hidden, num_layers, states
        self.inner = 2 * hidden
        self.heads = self.inner // self.HEAD
        self.conv_width = self.inner + 2 * states
        self.proj_width = self.conv_width + self.inner + self.heads
        lin = lambda fout, fin: torch.empty(fout, fin).uniform_(-1 / math.sqrt(fin), 1 / math.sqrt(fin))  # noqa: E731
        reg = lambda n, v: self.register_parameter(n, nn.Parameter(v))  # noqa: E731
        reg("weight_embed", lin(hidden, input_dim))
        reg("bias_embed", torch.zeros(hidden))
        for k in range(num_layers + 1):          # norm k stands before layer k; the last one ends the stack
            reg(f"pre_weight_l{k}", torch.ones(hidden))
            reg(f"pre_bias_l{k}", torch.zeros(hidden))
        for k in range(num_layers):
            reg(f"in_proj_l{k}", lin(self.proj_width, hidden))
            reg(f"conv_weight_l{k}", torch.empty(self.conv_width, self.WINDOW).uniform_(-0.5, 0.5))
            reg(f"conv_bias_l{k}", torch.zeros(self.conv_width))
            reg(f"A_log_l{k}", torch.empty(self.heads).uniform_(0.0, math.log(16.0)))
            reg(f"D_l{k}", torch.ones(self.heads))
            d = torch.exp(torch.empty(self.heads).uniform_(math.log(1e-3), math.log(1e-1)))
            reg(f"dt_bias_l{k}", d + torch.log(-torch.expm1(-d)))       # softplus of it is d
            reg(f"out_proj_l{k}", lin(hidden, self.inner))
            reg(f"post_weight_l{k}", torch.ones(hidden))
            reg(f"post_bias_l{k}", torch.zeros(hidden))
            reg(f"gate_l{k}", torch.full((hidden,), 0.5))

    def _p(self, name: str, k: int) -> torch.Tensor:
        return getattr(self, f"{name}_l{k}")

    def _split(self, u: torch.Tensor):
        x, Bm, Cm = torch.split(u, [self.inner, self.states, self.states], dim=-1)
        return x.unflatten(-1, (self.heads, self.HEAD)), Bm.unsqueeze(-2), Cm.unsqueeze(-2)

    def _start(self, x2d: torch.Tensor):
        h = _Linear16.apply(x2d.to(BF16).contiguous(), self.weight_embed, self.bias_embed).float()
        return h, _Norm16.apply(h, self.pre_weight_l0, self.pre_bias_l0)

    def _join(self, k: int, h, y):
        return ssm.sandwich_norm(h, y, self._p("post_weight", k), self._p("post_bias", k), self._p("pre_weight", k + 1),
                                 self._p("pre_bias", k + 1), gate=self._p("gate", k))

    def run(self, x: torch.Tensor, lengths=None, p_drop: float = 0.0, base_seed: int = 0, cache=None) -> torch.Tensor:
        """x [B,T,input] -> the normalised stream [B,T,hidden] bf16.  `cache` (a list): goes on from it, and leaves the states
        behind each sample's last frame in it."""
        B, T, _ = x.shape
        h, n = self._start(x.reshape(B * T, -1))
        h, n = h.view(B, T, -1), n.view(B, T, -1)
        widths = [self.conv_width, self.inner, self.heads]
        before, behind = list(cache) if cache else [(None, None)] * self.num_layers, []
        for k in range(self.num_layers):
            proj = _Linear16.apply(n.reshape(B * T, -1), self._p("in_proj", k), None).view(B, T, -1)
            xbc, z, dt = torch.split(proj, widths, dim=-1)
            conv0, scan0 = before[k]
            u, conv1 = ssm.causal_conv(xbc, self._p("conv_weight", k), self._p("conv_bias", k), activation="silu", state=conv0,
                                       lengths=lengths, return_state=True)
            xs, Bm, Cm = self._split(u)
            y, scan1 = ssm.selective_scan(xs, dt, -torch.exp(self._p("A_log", k)), Bm, Cm, D=self._p("D", k),
                                          z=z.unflatten(-1, (self.heads, self.HEAD)), dt_bias=self._p("dt_bias", k), state=scan0,
                                          lengths=lengths, return_state=True)
            behind.append((conv1, scan1))
            o = _Linear16.apply(y.reshape(B * T, self.inner), self._p("out_proj", k), None)
            if p_drop > 0.0 and k < self.num_layers - 1:     # as nn.LSTM: between layers only
                o = _Dropout.apply(o, p_drop, _site_seed(base_seed, 100 + k))
            h, n = self._join(k, h, o.view(B, T, -1))
        if cache is not None:
            cache[:] = behind
        return n

    def new_cache(self, B: int, device) -> list:
        """The states before any frame."""
        return [(torch.zeros(B, self.WINDOW - 1, self.conv_width, dtype=BF16, device=device),
                 torch.zeros(B, self.heads, self.HEAD, self.states, dtype=F32, device=device)) for _ in range(self.num_layers)]

    @torch.no_grad()
    def step(self, x: torch.Tensor, cache: list) -> torch.Tensor:
        """One frame: x [B,input] -> [B,hidden] bf16; the cache's states advance in place."""
        h, n = self._start(x)
        widths = [self.conv_width, self.inner, self.heads]
        for k in range(self.num_layers):
            xbc, z, dt = torch.split(_Linear16.apply(n, self._p("in_proj", k), None), widths, dim=-1)
            conv, scan = cache[k]
            xs, Bm, Cm = self._split(ssm.causal_conv_step(xbc, self._p("conv_weight", k), self._p("conv_bias", k), conv, activation="silu"))
            y = ssm.selective_scan_step(xs, dt, -torch.exp(self._p("A_log", k)), Bm, Cm, scan, D=self._p("D", k),
                                        z=z.unflatten(-1, (self.heads, self.HEAD)), dt_bias=self._p("dt_bias", k))
            h, n = self._join(k, h, _Linear16.apply(y.reshape(-1, self.inner), self._p("out_proj", k), None))
        return n


class TemporalEncoder(nn.Module):
    """train_vit.py:188-229: (bi)LSTM over frame features; returns [forward h at t = T-1 | backward h at t = 0].
    model_type='ssm': a stack of state-space layers (causal: bidirectional=False); returns its output at t = T-1."""

    def __init__(self, input_dim, hidden_dim=256, num_layers=2, dropout=0.3, bidirectional=True, model_type="lstm"):
        super().__init__()
        if model_type not in ("lstm", "gru", "ssm"):
            raise ValueError(f"Unknown model_type: {model_type}")
        if model_type == "ssm":
            if bidirectional:
                raise ValueError("model_type='ssm' is causal: bidirectional=False")
            if hidden_dim % 32 or input_dim % 8 or not 0 < hidden_dim <= 2048 or num_layers < 1:
                raise NotImplementedError("the state-space layers need hidden_dim % 32 == 0 (at most 2048) and input_dim % 8 == 0")
            self.model_type, self.bidirectional, self.hidden_dim, self.num_layers = model_type, False, hidden_dim, num_layers
            self.dropout = float(dropout) if num_layers > 1 else 0.0
            self.rnn = SSMStack(input_dim, hidden_dim, num_layers)
            self.output_dim = hidden_dim
            return
        if hidden_dim % 8 or input_dim % 4:
            raise NotImplementedError("the recurrent kernels need hidden_dim % 8 == 0 and input_dim % 4 == 0")
        self.model_type, self.bidirectional, self.hidden_dim = model_type, bidirectional, hidden_dim
        self.num_layers = num_layers
        self.dropout = float(dropout) if num_layers > 1 else 0.0
        self.rnn = _LSTMParams(input_dim, hidden_dim, num_layers, bidirectional, gates=4 if model_type == "lstm" else 3)
        self.output_dim = hidden_dim * (2 if bidirectional else 1)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if self.model_type == "ssm":
            return self.ssm_features(x)[0]
        return _TemporalFunction.apply(x, self, None, self.training and torch.is_grad_enabled(), *self.parameters())

    def ssm_features(self, x: torch.Tensor, lengths: Optional[torch.Tensor] = None, cache: Optional[list] = None):
        """-> (feature [B,hidden] fp32 of each sample's last frame, seed of this pass's dropout sites).  `lengths` int32 [B]: sample b
        ends after lengths[b] frames (held to 0..T), and what x holds behind counts nowhere; without a frame its feature is zero."""
        if not x.is_cuda:
            raise RuntimeError("the temporal encoder runs on the GPU through librvit only; there is no CPU fallback")
        if x.dim() != 3 or x.shape[2] != self.rnn.input_size or x.shape[0] < 1 or x.shape[1] < 1:
            raise ValueError(f"expected features [B,T,{self.rnn.input_size}], got {tuple(x.shape)}")
        if lengths is not None and (lengths.dtype != torch.int32 or lengths.shape != x.shape[:1] or lengths.device != x.device):
            raise ValueError(f"lengths must be int32 [{x.shape[0]}] on {x.device}, got {lengths.dtype} {tuple(lengths.shape)} on {lengths.device}")
        train = self.training and torch.is_grad_enabled()
        base = int(torch.randint(0, 2 ** 62, (1,)).item()) if train else 0
        with torch.cuda.device(x.device):
            if lengths is not None:      # zero, not only unread: the weights' gradients are products with every row
                ends = lengths.long().clamp(0, x.shape[1])[:, None]
                x = torch.where((torch.arange(x.shape[1], device=x.device) < ends)[..., None], x, x.new_zeros(()))
            n = self.rnn.run(x, lengths, self.dropout if train else 0.0, base, cache)
            if lengths is None:
                last = n[:, -1]
            else:
                last = n.gather(1, (ends - 1).clamp(min=0)[..., None].expand(-1, 1, n.shape[2]))[:, 0]
                last = torch.where(ends > 0, last, last.new_zeros(()))
            return last.float(), base


def _site_seed(base: int, site: int) -> int:
    z = (base + 0x9E3779B97F4A7C15 * (site + 1)) & _M64
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & _M64
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & _M64
    return z ^ (z >> 31)


def _lstm_forward(enc: TemporalEncoder, x: torch.Tensor, train: bool, base_seed: int):
    """x [B,T,In] fp32 -> (top-layer output [B,T,ndir*H], saved tensors per layer)."""
    lib = _lib.load()
    B, T, _ = x.shape
    H, ndir = enc.hidden_dim, 2 if enc.bidirectional else 1
    saved = []
    cur = x.contiguous()
    for layer in range(enc.num_layers):
        In = cur.shape[2]
        out = torch.empty(B, T, ndir * H, dtype=F32, device=x.device)
        lstm = enc.model_type == "lstm"
        c = torch.empty(ndir, B, H, dtype=F32, device=x.device) if lstm else None
        gates = torch.empty(B, T, ndir, 4 * H, dtype=F32, device=x.device) if train else None   # GRU: (r, z, n, hn)
        cseq = torch.empty(B, T, ndir, H, dtype=F32, device=x.device) if train and lstm else None
        wf = [p.detach() for p in enc.rnn.direction(layer, False)]
        wr = [p.detach() for p in enc.rnn.direction(layer, True)] if ndir == 2 else [None] * 4
        with ops._Span("rnn_fwd", 2 * B * T * ndir * enc.rnn.gates * H * (In + H), 0):
            for s in range(T):
                if lstm:
                    check(lib.rvit_lstm_step_fwd(_ptr(cur), *[_ptr(w) for w in wf], *[_ptr(w) for w in wr], _ptr(out),
                                                 _ptr(c), _ptr(gates), _ptr(cseq), B, T, In, H, s, _stream()),
                          "rvit_lstm_step_fwd")
                else:
                    check(lib.rvit_gru_step_fwd(_ptr(cur), *[_ptr(w) for w in wf], *[_ptr(w) for w in wr], _ptr(out),
                                                _ptr(gates), B, T, In, H, s, _stream()), "rvit_gru_step_fwd")
        nxt = out
        seed = 0
        if train and enc.dropout > 0 and layer < enc.num_layers - 1:   # nn.LSTM: dropout on every layer's output but the last
            seed = _site_seed(base_seed, 100 + layer)
            nxt = torch.empty_like(out)
            ops.dropout_apply(out.view(B * T, ndir * H), nxt.view(B * T, ndir * H), enc.dropout, seed)
        saved.append(dict(x=cur, out=out, gates=gates, cseq=cseq, seed=seed))
        cur = nxt
    return cur, saved


def _lstm_backward(enc: TemporalEncoder, saved, dtop: torch.Tensor) -> Tuple[torch.Tensor, Dict[str, torch.Tensor]]:
    """dtop [B,T,ndir*H] -> (dx of layer 0 [B,T,In], {parameter name: gradient})."""
    lib = _lib.load()
    H, ndir = enc.hidden_dim, 2 if enc.bidirectional else 1
    grads: Dict[str, torch.Tensor] = {}
    dout = dtop.contiguous()
    for layer in reversed(range(enc.num_layers)):
        sv = saved[layer]
        x, out = sv["x"], sv["out"]
        B, T, In = x.shape
        dev = x.device
        lstm = enc.model_type == "lstm"
        G = enc.rnn.gates * H                         # gate rows: 4H (LSTM) or 3H (GRU)
        # LSTM: one set of pre-activation gradients; GRU: input-side then hidden-side (they differ in the n gate)
        dG = torch.empty(B, T, ndir, G if lstm else 2 * G, dtype=F32, device=dev)
        carry = torch.empty(ndir, B, H, dtype=F32, device=dev)
        whh_t = [enc.rnn.direction(layer, d == 1)[1].detach().t().contiguous() for d in range(ndir)]
        with ops._Span("rnn_bwd", 2 * B * T * ndir * G * H, 0):
            for s in reversed(range(T)):
                if lstm:
                    check(lib.rvit_lstm_step_bwd(_ptr(dout), _ptr(whh_t[0]), _ptr(whh_t[1]) if ndir == 2 else None,
                                                 _ptr(sv["gates"]), _ptr(sv["cseq"]), _ptr(dG), _ptr(carry), B, T, H, s,
                                                 _stream()), "rvit_lstm_step_bwd")
                else:
                    check(lib.rvit_gru_step_bwd(_ptr(dout), _ptr(whh_t[0]), _ptr(whh_t[1]) if ndir == 2 else None,
                                                _ptr(sv["gates"]), _ptr(out), _ptr(dG), _ptr(carry), B, T, H, s,
                                                _stream()), "rvit_gru_step_bwd")
        x16 = x.reshape(B * T, In).to(BF16)
        dx = torch.empty(B * T, In, dtype=F32, device=dev)
        for d in range(ndir):
            sfx = "_reverse" if d else ""
            w_ih = enc.rnn.direction(layer, d == 1)[0].detach()
            dGd = dG[:, :, d, :G].reshape(B * T, G)                       # fp32, contiguous copy of this direction
            dGh = dGd if lstm else dG[:, :, d, G:].reshape(B * T, G)      # hidden-side gradients (GRU)
            dG16 = dGd.to(BF16)
            dGh16 = dG16 if lstm else dGh.to(BF16)
            hprev = torch.zeros(B, T, H, dtype=BF16, device=dev)          # h of the previous step of this direction
            if T > 1:
                if d == 0:
                    hprev[:, 1:] = out[:, :-1, :H]
                else:
                    hprev[:, :-1] = out[:, 1:, H:]
            g_ih = torch.zeros(G, In, dtype=F32, device=dev)
            g_hh = torch.zeros(G, H, dtype=F32, device=dev)
            g_b = torch.zeros(G, dtype=F32, device=dev)
            ops.wgrad(dG16, x16, g_ih)
            ops.wgrad(dGh16, hprev.view(B * T, H), g_hh)
            ops.batch_sum(dGd, g_b)
            if lstm:
                g_bh = g_b.clone()
            else:
                g_bh = torch.zeros(G, dtype=F32, device=dev)
                ops.batch_sum(dGh, g_bh)
            grads[f"weight_ih_l{layer}{sfx}"], grads[f"weight_hh_l{layer}{sfx}"] = g_ih, g_hh
            grads[f"bias_ih_l{layer}{sfx}"], grads[f"bias_hh_l{layer}{sfx}"] = g_b, g_bh
            # dx (+)= dG_d @ W_ih: gemm computes a @ w.T with w [N=In, K=4H]
            ops.gemm(dG16, w_ih.t().contiguous().to(BF16), dx, residual=dx if d else None)
        dx = dx.view(B, T, In)
        if layer > 0:
            seed = saved[layer - 1]["seed"]
            if seed:
                dd = torch.empty_like(dx)
                ops.dropout_apply(dx.view(B * T, In), dd.view(B * T, In), enc.dropout, seed)
                dx = dd
        dout = dx
    return dout, grads


def _select_last(enc: TemporalEncoder, top: torch.Tensor) -> torch.Tensor:
    H = enc.hidden_dim
    if enc.bidirectional:     # train_vit.py:225-228
        return torch.cat([top[:, -1, :H], top[:, 0, H:]], dim=1)
    return top[:, -1, :].contiguous()


def _scatter_last(enc: TemporalEncoder, dtf: torch.Tensor, B: int, T: int) -> torch.Tensor:
    H = enc.hidden_dim
    ndir = 2 if enc.bidirectional else 1
    dtop = torch.zeros(B, T, ndir * H, dtype=F32, device=dtf.device)
    dtop[:, -1, :H] = dtf[:, :H]
    if enc.bidirectional:
        dtop[:, 0, H:] = dtf[:, H:]
    return dtop


def _cls_forward(cls, tf: torch.Tensor, train: bool, base: int):
    """temporal feature fp32 [B,D] -> (logits fp32 [B,classes], what the backward needs)."""
    B, D = tf.shape
    l0, l3 = cls["0"], cls["3"]
    C = l3.weight.shape[0]
    tf16 = tf.to(BF16)
    h = torch.empty(B, D // 2, dtype=BF16, device=tf.device)
    u0 = torch.empty(B, D // 2, dtype=BF16, device=tf.device) if train else None
    p = cls.drop_p if train else 0.0
    seed = _site_seed(base, 1) if p > 0 else 0
    ops.gemm(tf16, l0.weight.detach().to(BF16), h, bias=l0.bias.detach(), act="gelu", preact=u0,
             drop=("post_act", p, seed) if p > 0 else None)
    logits = torch.empty(B, C, dtype=F32, device=tf.device)
    ops.gemm(h, l3.weight.detach().to(BF16), logits, bias=l3.bias.detach())
    return logits, (tf16, h, u0, p, seed)


def _cls_backward(cls, saved, dout: torch.Tensor):
    """-> (gradient of the temporal feature, [gradients of the classifier's parameters])."""
    tf16, h, u0, p, seed = saved
    B, dev = tf16.shape[0], dout.device
    l0, l3 = cls["0"], cls["3"]
    C, Dh = l3.weight.shape
    Cp = 16 * ((C + 15) // 16)
    dl16 = torch.zeros(B, Cp, dtype=BF16, device=dev)
    dl16[:, :C] = dout
    g3 = torch.zeros(C, Dh, dtype=F32, device=dev)
    ops.wgrad(dl16, h, g3, n_store=C)
    b3 = torch.zeros(Cp, dtype=F32, device=dev)
    ops.colsum(dl16, b3)
    w3t = torch.zeros(Dh, Cp, dtype=BF16, device=dev)
    w3t[:, :C] = l3.weight.detach().t().to(BF16)
    dh = torch.empty(B, Dh, dtype=BF16, device=dev)
    ops.gemm(dl16, w3t, dh, gate=u0, gate_mode="gelu_grad", drop=("post_act", p, seed) if p > 0 else None)
    g0 = torch.zeros(Dh, tf16.shape[1], dtype=F32, device=dev)
    ops.wgrad(dh, tf16, g0)
    b0 = torch.zeros(Dh, dtype=F32, device=dev)
    ops.colsum(dh, b0)
    dtf = torch.empty(B, tf16.shape[1], dtype=F32, device=dev)
    ops.gemm(dh, l0.weight.detach().t().contiguous().to(BF16), dtf)
    return dtf, [g0, b0, g3, b3[:C].contiguous()]


class _ClassifierFunction(torch.autograd.Function):
    """temporal feature [B,D] -> logits, behind an encoder whose own backward is autograd's (model_type='ssm')."""

    @staticmethod
    def forward(ctx, tf, cls, train: bool, base: int, *params):
        with torch.cuda.device(tf.device):
            logits, ctx.cls_saved = _cls_forward(cls, tf.detach(), train, base)
        ctx.cls, ctx.trained = cls, train
        return logits

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        if not ctx.trained:
            raise RuntimeError("backward through a forward that ran in eval mode / without grad")
        with torch.cuda.device(dout.device):
            dtf, grads = _cls_backward(ctx.cls, ctx.cls_saved, dout)
        return (dtf, None, None, None, *grads)


class _TemporalFunction(torch.autograd.Function):
    """features [B,T,E] -> temporal feature [B,out_dim] (classifier=None) or logits [B,classes]."""

    @staticmethod
    def forward(ctx, feats, enc: TemporalEncoder, cls, train: bool, *params):
        if not feats.is_cuda:
            raise RuntimeError("the temporal encoder runs on the GPU through librvit only; there is no CPU fallback")
        with torch.cuda.device(feats.device):   # librvit launches on the current device's stream
            return _TemporalFunction._forward(ctx, feats, enc, cls, train)

    @staticmethod
    def _forward(ctx, feats, enc: TemporalEncoder, cls, train: bool):
        if feats.dim() != 3 or feats.shape[2] != enc.rnn.input_size:
            raise ValueError(f"expected features [B,T,{enc.rnn.input_size}], got {tuple(feats.shape)}")
        base = int(torch.randint(0, 2 ** 62, (1,)).item()) if train else 0
        top, saved = _lstm_forward(enc, feats.detach().float(), train, base)
        tf = _select_last(enc, top)
        ctx.enc, ctx.cls, ctx.saved, ctx.shape = enc, cls, saved, tuple(feats.shape)
        if cls is None:
            return tf
        logits, ctx.cls_saved = _cls_forward(cls, tf, train, base)
        return logits

    @staticmethod
    def backward(ctx, dout):
        with torch.cuda.device(dout.device):
            return _TemporalFunction._backward(ctx, dout)

    @staticmethod
    def _backward(ctx, dout):
        enc, cls, saved = ctx.enc, ctx.cls, ctx.saved
        if saved[0]["gates"] is None:
            raise RuntimeError("backward through a forward that ran in eval mode / without grad")
        B, T, _ = ctx.shape
        dev = dout.device
        cls_grads: List[torch.Tensor] = []
        if cls is None:
            dtf = dout.contiguous().float()
        else:
            dtf, cls_grads = _cls_backward(cls, ctx.cls_saved, dout)
        dfeats, g = _lstm_backward(enc, saved, _scatter_last(enc, dtf, B, T))
        enc_grads = [g[n] for n, _ in enc.rnn.named_parameters()]
        return (dfeats, None, None, None, *enc_grads, *cls_grads)


class _Classifier(nn.ModuleDict):
    """nn.Sequential(Linear, GELU, Dropout, Linear) parameter holder with the Sequential's key names."""

    def __init__(self, dim: int, num_classes: int, drop_p: float):
        super().__init__({"0": _Linear(dim, dim // 2), "3": _Linear(dim // 2, num_classes)})
        self.drop_p = float(drop_p)


class CNNViTSequence(nn.Module):
    """train_vit.py:232-318 / infer.py:230-265: [B,T,3,224,224] -> logits [B,num_classes]."""

    def __init__(self, num_classes, config):
        super().__init__()
        self.spatial_encoder = CNNViTHybrid(num_classes=num_classes, backbone=config["backbone"], embed_dim=config["embed_dim"],
                                            num_heads=config["num_heads"], num_layers=config["num_layers"],
                                            dropout=config["dropout"], pretrained_backbone=False)
        self.temporal_encoder = TemporalEncoder(input_dim=config["embed_dim"], hidden_dim=config.get("temporal_hidden", 256),
                                                num_layers=config.get("temporal_layers", 2),
                                                dropout=config.get("temporal_dropout", 0.3),
                                                bidirectional=config.get("temporal_bidirectional", config.get("temporal_model", "lstm") != "ssm"),
                                                model_type=config.get("temporal_model", "lstm"))
        d = self.temporal_encoder.output_dim
        if (d // 2) % 8:
            raise NotImplementedError("classifier width must be a multiple of 8 for the GEMM kernels")
        self.classifier = _Classifier(d, num_classes, config.get("classifier_dropout", 0.4))
        self.config = config
        self.embed_dim = config["embed_dim"]

    def forward(self, x):
        if x.dim() != 5:
            raise ValueError(f"expected [B,T,3,224,224], got {tuple(x.shape)}")
        B, T = x.shape[:2]
        feats = self.spatial_encoder.forward_features(x.reshape(B * T, *x.shape[2:]))
        return self.forward_temporal_only(feats.view(B, T, -1))

    def forward_spatial_only(self, x):
        """Single frames -> spatial features (streaming)."""
        return self.spatial_encoder.forward_features(x)

    def forward_temporal_only(self, spatial_features):
        """[B,T,E] features -> logits (streaming)."""
        enc = self.temporal_encoder
        if enc.model_type == "ssm":
            tf, base = enc.ssm_features(spatial_features)
            return _ClassifierFunction.apply(tf, self.classifier, self.training and torch.is_grad_enabled(), base,
                                             *self.classifier.parameters())
        return _TemporalFunction.apply(spatial_features, enc, self.classifier, self.training and torch.is_grad_enabled(),
                                       *enc.parameters(), *self.classifier.parameters())

    @torch.no_grad()
    def forward_temporal_step(self, spatial_features, cache: Optional[list] = None):
        """temporal_model='ssm': one frame's features [B,E] -> (logits, cache).  The cache (None: before any frame) holds every
        layer's states and advances in place: the cost of a frame does not grow with the number of frames behind it."""
        enc = self.temporal_encoder
        if enc.model_type != "ssm":
            raise ValueError(f"temporal_model={enc.model_type!r} keeps no state between frames: use forward_temporal_only on a window")
        if not spatial_features.is_cuda:
            raise RuntimeError("the temporal encoder runs on the GPU through librvit only; there is no CPU fallback")
        if spatial_features.dim() != 2 or spatial_features.shape[1] != self.embed_dim:
            raise ValueError(f"expected features [B,{self.embed_dim}], got {tuple(spatial_features.shape)}")
        with torch.cuda.device(spatial_features.device):
            if cache is None:
                cache = enc.rnn.new_cache(spatial_features.shape[0], spatial_features.device)
            tf = enc.rnn.step(spatial_features, cache).float()
            return _cls_forward(self.classifier, tf, False, 0)[0], cache

    def freeze_backbone(self):
        for p in self.spatial_encoder.cnn_backbone.parameters():
            p.requires_grad = False

    def unfreeze_backbone(self):
        for p in self.spatial_encoder.cnn_backbone.parameters():
            p.requires_grad = True


@dataclass
class StreamPrediction:   # infer.py:58-66
    prediction: str
    confidence: float
    is_reliable: bool
    all_probs: List[Tuple[str, float]]
    frame_count: int
    latency_ms: float


class StreamingClassifier:
    """infer.py:479-630: sliding window of per-frame features; a prediction once `sequence_length` frames are in,
    smoothed over the last `smoothing_window` predictions.  Accepts a checkpoint path (reference layout, read with
    weights_only=True) or a ready (model, classes, config) triple."""

    def __init__(self, model_path=None, device: str = "auto", smoothing_window: int = 3, *, model=None, classes=None,
                 config=None, confidence_threshold: float = 0.5, device_preprocess: bool = False, carry_state: bool = False):
        # device_preprocess: uint8 frames given as arrays are resized / normalised on the GPU (vit_amd.pipeline, the
        # same arithmetic as the host transform, bit for bit) instead of by Pillow on the host
        # carry_state (temporal_model='ssm'): every frame goes on from the states the frames before it left, back to the last
        # reset(), instead of running the last `sequence_length` frames again
        self.device_preprocess = bool(device_preprocess)
        self._pre = {}
        self.device = torch.device("cuda" if device == "auto" else device)
        if self.device.type != "cuda":
            raise RuntimeError("StreamingClassifier runs on the GPU through librvit only")
        if model is None:
            from torch.torch_version import TorchVersion
            with torch.serialization.safe_globals([TorchVersion]):
                ckpt = torch.load(model_path, map_location="cpu", weights_only=True)
            classes = ckpt["classes"]
            config = ckpt.get("model_config", {})
            confidence_threshold = ckpt.get("metadata", {}).get("confidence_threshold", 0.5)
            if config.get("mode", "single") == "sequence":
                model = CNNViTSequence(num_classes=len(classes), config=config)
            else:
                model = CNNViTHybrid(num_classes=len(classes), backbone=config.get("backbone", "resnet18"),
                                     embed_dim=config.get("embed_dim", 256), num_heads=config.get("num_heads", 4),
                                     num_layers=config.get("num_layers", 4), dropout=config.get("dropout", 0.1))
            model.load_state_dict(ckpt["model"])
        self.classes, self.config = list(classes), dict(config or {})
        self.mode = "sequence" if isinstance(model, CNNViTSequence) else "single"
        self.sequence_length = self.config.get("sequence_length", 8) if self.mode == "sequence" else 1
        self.confidence_threshold = confidence_threshold
        self.model = model.to(self.device).eval()
        self.carry_state = bool(carry_state)
        if self.carry_state and (self.mode != "sequence" or self.model.temporal_encoder.model_type != "ssm"):
            raise ValueError("carry_state needs a sequence model with temporal_model='ssm'")
        self._cache = None
        self.feature_buffer = deque(maxlen=self.sequence_length)
        self.prediction_history = deque(maxlen=smoothing_window)
        self.frame_count = 0

    def _preprocess(self, image_input) -> torch.Tensor:
        from .infer import preprocess
        if isinstance(image_input, torch.Tensor):
            return image_input
        if isinstance(image_input, np.ndarray):
            if self.device_preprocess and image_input.dtype == np.uint8 and image_input.ndim in (2, 3):
                from .pipeline import DevicePreprocessor
                hw = tuple(image_input.shape[:2])
                pre = self._pre.get(hw)
                if pre is None:
                    pre = self._pre[hw] = DevicePreprocessor(hw, train=False, device=self.device)
                frame = torch.from_numpy(np.ascontiguousarray(image_input))[None].to(self.device, non_blocking=True)
                return pre(frame)[0]
            if image_input.ndim == 2:
                image_input = np.stack([image_input] * 3, axis=-1)
            from PIL import Image
            return preprocess(Image.fromarray(image_input.astype(np.uint8)))
        if isinstance(image_input, (str, bytes)) or hasattr(image_input, "__fspath__"):
            from PIL import Image
            return preprocess(Image.open(image_input).convert("RGB"))
        if hasattr(image_input, "convert"):
            return preprocess(image_input)
        raise TypeError(f"Unsupported input type: {type(image_input)}")

    @torch.no_grad()
    def update(self, frame) -> Optional[StreamPrediction]:
        start = time.perf_counter()
        tensor = self._preprocess(frame).unsqueeze(0).to(self.device)
        self.frame_count += 1
        if self.carry_state:
            logits, self._cache = self.model.forward_temporal_step(self.model.forward_spatial_only(tensor).view(1, -1), self._cache)
            if self.frame_count < self.sequence_length:
                return None
        elif self.mode == "sequence":
            self.feature_buffer.append(self.model.forward_spatial_only(tensor))
            if len(self.feature_buffer) < self.sequence_length:
                return None
            logits = self.model.forward_temporal_only(torch.cat(list(self.feature_buffer), dim=0).unsqueeze(0))
        else:
            logits = self.model(tensor)
        probs = torch.softmax(logits.float(), dim=1)[0].cpu()
        self.prediction_history.append(probs)
        avg = torch.stack(list(self.prediction_history)).mean(dim=0) if len(self.prediction_history) > 1 else probs
        conf, idx = avg.max(0)
        conf, idx = conf.item(), idx.item()
        all_probs = sorted(((self.classes[i], avg[i].item()) for i in range(len(self.classes))), key=lambda v: v[1], reverse=True)
        return StreamPrediction(prediction=self.classes[idx], confidence=conf, is_reliable=conf >= self.confidence_threshold,
                                all_probs=all_probs, frame_count=self.frame_count,
                                latency_ms=(time.perf_counter() - start) * 1000)

    def reset(self):
        self._cache = None
        self.feature_buffer.clear()
        self.prediction_history.clear()
        self.frame_count = 0

    def benchmark(self, n_frames: int = 100) -> dict:
        dummy = (np.random.default_rng(0).random((224, 224, 3)) * 255).astype(np.uint8)
        self.reset()
        for _ in range(self.sequence_length + 5):
            self.update(dummy)
        self.reset()
        lat = [r.latency_ms for r in (self.update(dummy) for _ in range(n_frames)) if r]
        return {"mean_latency_ms": float(np.mean(lat)) if lat else 0, "std_latency_ms": float(np.std(lat)) if lat else 0,
                "fps": 1000 / float(np.mean(lat)) if lat else 0, "sequence_length": self.sequence_length, "mode": self.mode,
                "device": str(self.device)}
