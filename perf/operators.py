"""What the state-space sequence operators of vit_amd cost, and what they compute: the cases, their inputs, the
operators in plain torch (`own` false) or as a user calls them (`own` true), and the same results from their definitions
in 64 bits.

  conv   y[t] = silu(bias + sum_k weight[:, k] x[t - K + 1 + k]) over the tokens of a sequence, a short window per channel
  scan   S[t] = exp(d[t] A) S[t-1] + d[t] x[t] B[t]^T,  y[t] = (S[t] C[t] + D x[t]) * silu(z[t]),  d = softplus(dt + dt_bias)
  norm   h = residual + scale * gate * norm_post(y),  n = norm_pre(h): behind one block and before the next
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
CHUNK = 64


# ---- the cases ----------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one frame of 64 live streams through the window of a layer of inner width 2048 (states of 128)
        {"name": "conv step", "op": "conv", "mode": "step", "dtype": "bf16", "B": 64, "C": 2304, "K": 4},
        # a training batch of long recordings, inner width 1536
        {"name": "conv train", "op": "conv", "mode": "train", "dtype": "bf16", "B": 8, "T": 2048, "C": 1792, "K": 4, "ragged": False},
        # one frame of one live stream: width 256, expanded by two
        {"name": "scan step one", "op": "scan", "mode": "step", "dtype": "bf16", "B": 1, "H": 8, "P": 64, "G": 1, "N": 64},
        # one frame of 256 streams through a wide layer
        {"name": "scan step many", "op": "scan", "mode": "step", "dtype": "bf16", "B": 256, "H": 32, "P": 64, "G": 1, "N": 128},
        # a short prompt on top of a kept state
        {"name": "scan prompt short", "op": "scan", "mode": "prompt", "dtype": "bf16", "B": 2, "T": 197, "H": 8, "P": 64, "G": 1, "N": 64, "ragged": False, "start": True},
        # one long recording
        {"name": "scan prompt long", "op": "scan", "mode": "prompt", "dtype": "bf16", "B": 1, "T": 32768, "H": 16, "P": 64, "G": 1, "N": 128, "ragged": False, "start": False},
        # recordings of unequal lengths in one padded batch, odd sizes, two groups of heads, fp32
        {"name": "scan prompt ragged", "op": "scan", "mode": "prompt", "dtype": "f32", "B": 7, "T": 1021, "H": 6, "P": 48, "G": 2, "N": 40, "ragged": True, "start": True},
        # a training batch of long recordings
        {"name": "scan train", "op": "scan", "mode": "train", "dtype": "bf16", "B": 8, "T": 2048, "H": 24, "P": 64, "G": 1, "N": 128, "ragged": False, "start": False},
        # the sequence model's own training step: windows of 8 frames, fp32
        {"name": "scan train window", "op": "scan", "mode": "train", "dtype": "f32", "B": 64, "T": 8, "H": 8, "P": 64, "G": 1, "N": 64, "ragged": False, "start": False},
        # one frame of one live stream
        {"name": "norm one row", "op": "norm", "mode": "forward", "dtype": "bf16", "residual": "f32", "B": 1, "T": 1, "E": 256, "gate": "channel", "kind": "layer"},
        # the token stream of a ViT-L/16-scale training batch, a learned gate per channel
        {"name": "norm train", "op": "norm", "mode": "train", "dtype": "bf16", "residual": "f32", "B": 128, "T": 197, "E": 1024, "gate": "channel", "kind": "layer"},
        # a gate per sample, no centring, odd sizes, fp32
        {"name": "norm train sample gate", "op": "norm", "mode": "train", "dtype": "f32", "residual": "f32", "B": 37, "T": 51, "E": 387, "gate": "sample", "kind": "rms"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["conv", "scan", "scan", "norm"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "conv":
        mode = rng.choice(["step", "prompt", "train"])
        C = _log_int(rng, 32, 4096)
        case = {"op": op, "mode": mode, "dtype": dtype, "B": _log_int(rng, 1, 512 if mode == "step" else 64), "C": C, "K": rng.randint(2, 6)}
        if mode != "step":
            most = max(1, min(32768, 8 * 2048 * 1792 // (case["B"] * C)))
            case.update(T=_log_int(rng, 1, most), ragged=rng.random() < 0.4)
        return case
    if op == "scan":
        mode = rng.choice(["step", "prompt", "train", "train"])
        G = rng.choice([1, 1, 2, 3])
        case = {"op": op, "mode": mode, "dtype": dtype, "B": _log_int(rng, 1, 256 if mode == "step" else 64), "H": G * _log_int(rng, 1, 12),
                "P": rng.choice([16, 32, 48, 64, 64, 64, 128, rng.randint(9, 100)]), "G": G, "N": rng.choice([16, 32, 64, 64, 128, 128, rng.randint(5, 127)])}
        if mode != "step":
            most = max(1, min(32768, 8 * 2048 * 24 * 64 // (case["B"] * case["H"] * max(case["P"], 16)) // (2 if dtype == "f32" else 1)))
            case.update(T=_log_int(rng, 1, most), ragged=rng.random() < 0.4, start=rng.random() < 0.5)
        return case
    E = rng.choice([256, 512, 768, 1024, 2048, rng.randint(33, 1100)])
    B = _log_int(rng, 1, 128)
    return {"op": op, "mode": rng.choice(["forward", "train", "train"]), "dtype": dtype, "residual": rng.choice(["f32", dtype]), "B": B,
            "T": _log_int(rng, 1, max(1, min(8192, 128 * 197 * 1024 // (B * E)))), "E": E, "gate": rng.choice(["none", "channel", "sample", "token"]),
            "kind": rng.choice(["layer", "rms"])}


# ---- inputs -------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 17)

    def randn(*shape, dtype=torch.float32, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    dt = DTYPES[case["dtype"]]
    B, train = case["B"], case["mode"] == "train"
    s = {"case": case}
    if case["op"] == "conv":
        C, K = case["C"], case["K"]
        s["weight"], s["bias"] = (rand(C, K) * 2 - 1) / math.sqrt(K), (rand(C) * 2 - 1) / math.sqrt(K)
        if case["mode"] == "step":
            # a slice of the block's input projection, as the scan's gate stands beside it
            s["x"] = randn(B, C + 64, dtype=dt)[:, 64:]
            s["state"] = randn(B, K - 1, C, dtype=dt)
            return s
        T = case["T"]
        s["x"] = randn(B, T, C + 64, dtype=dt)[:, :, 64:]
        s["lengths"] = (rand(B) * (T + 1)).to(torch.int32) if case["ragged"] else None
        if train:
            s["dy"] = randn(B, T, C, dtype=dt)
            for k in ("x", "weight", "bias"):
                s[k] = s[k].requires_grad_()
        else:
            s["state"] = randn(B, K - 1, C, dtype=dt)
        return s
    if case["op"] == "scan":
        H, P, G, N = case["H"], case["P"], case["G"], case["N"]
        step = case["mode"] == "step"
        lead = (B,) if step else (B, case["T"])
        # x, B, C are slices of the convolution's output (behind a silu), z and dt slices of the input projection
        inner = randn(*lead, H * P + 2 * G * N, dtype=torch.float32)
        inner = (inner * torch.sigmoid(inner) * 2).to(dt)
        outer = randn(*lead, H * P + H, dtype=dt)
        s["x"] = inner[..., :H * P].unflatten(-1, (H, P))
        s["Bm"] = inner[..., H * P:H * P + G * N].unflatten(-1, (G, N))
        s["Cm"] = inner[..., H * P + G * N:].unflatten(-1, (G, N))
        s["z"] = outer[..., :H * P].unflatten(-1, (H, P))
        s["dt"] = outer[..., H * P:]
        s["A"] = -torch.exp(rand(H) * math.log(16.0))
        s["D"] = randn(H, scale=0.2, shift=1.0)
        d = torch.exp(rand(H) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
        s["dt_bias"] = d + torch.log(-torch.expm1(-d))
        if step:
            s["state"] = randn(B, H, P, N)
            return s
        s["lengths"] = (rand(B) * (case["T"] + 1)).to(torch.int32) if case["ragged"] else None
        s["state"] = randn(B, H, P, N) if case["start"] else None
        if train:
            s["dy"] = randn(B, case["T"], H, P, dtype=dt)
            for k in ("x", "dt", "A", "Bm", "Cm", "D", "z", "dt_bias", "state"):
                s[k] = s[k].requires_grad_() if s[k] is not None else None
        return s
    T, E = case["T"], case["E"]
    rdt = DTYPES[case["residual"]]
    s["residual"], s["y"] = randn(B, T, E, dtype=rdt), randn(B, T, E, dtype=dt, scale=0.7, shift=0.1)
    for k in ("post_weight", "pre_weight"):
        s[k] = randn(E, scale=0.1, shift=1.0)
    for k in ("post_bias", "pre_bias"):
        s[k] = randn(E, scale=0.1) if case["kind"] == "layer" else None
    shape = {"none": None, "channel": (E,), "sample": (B, E), "token": (B, T, E)}[case["gate"]]
    s["gate"] = None if shape is None else randn(*shape, scale=0.3, shift=0.5, dtype=torch.float32 if case["gate"] == "channel" else dt)
    s["scale"] = 0.5
    if train:
        s["dh"], s["dn"] = randn(B, T, E, dtype=rdt), randn(B, T, E, dtype=dt)
        for k in ("residual", "y", "post_weight", "post_bias", "pre_weight", "pre_bias", "gate"):
            s[k] = s[k].requires_grad_() if s[k] is not None else None
    return s


# ---- the operators in plain torch ---------------------------------------------------------------------------------------
def _silu(v):
    return v * torch.sigmoid(v)


def _softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-torch.abs(v)))


def _valid(lengths, B, T, device):
    if lengths is None:
        return torch.ones(B, T, dtype=torch.bool, device=device)
    return torch.arange(T, device=device)[None, :] < lengths[:, None]


def _plain_conv(x, weight, bias, state, lengths):
    B, T, C = x.shape
    K = weight.shape[1]
    before = torch.zeros(B, K - 1, C, device=x.device) if state is None else state.float()
    full = torch.cat([before, x.float()], dim=1)
    u = (full.unfold(1, K, 1) * weight).sum(-1) + bias
    y = torch.where(_valid(lengths, B, T, x.device)[..., None], _silu(u), torch.zeros((), device=x.device))
    ends = torch.full((B,), T, device=x.device) if lengths is None else lengths.long()
    at = ends[:, None] + torch.arange(K - 1, device=x.device)[None, :]
    after = full.gather(1, at[..., None].expand(B, K - 1, C))
    return y.to(x.dtype), after.to(x.dtype)


def _plain_conv_step(x, weight, bias, state):
    full = torch.cat([state.float(), x.float()[:, None]], dim=1)
    y = _silu((full * weight.t()).sum(1) + bias)
    state.copy_(full[:, 1:])
    return y.to(x.dtype)


def _plain_scan(x, dt, A, Bm, Cm, D, z, dt_bias, state, lengths):
    """Chunks of CHUNK tokens: products inside a chunk, the states between chunks as one product with their decays."""
    B, T, H, P = x.shape
    G, N = Bm.shape[2:]
    nc = -(-T // CHUNK)
    pad = nc * CHUNK - T
    grow = lambda v: torch.cat([v, v.new_zeros(B, pad, *v.shape[2:])], dim=1) if pad else v  # noqa: E731
    cut = lambda v: grow(v).unflatten(1, (nc, CHUNK)).transpose(2, 3)  # noqa: E731   [B, nc, H, CHUNK, ..]
    zero = torch.zeros((), device=x.device)
    valid = _valid(lengths, B, T, x.device)[..., None]
    x32 = x.float()
    d = torch.where(valid, _softplus(dt.float() + dt_bias), zero)
    a = cut((d.double() * A.double())[..., None])[..., 0].cumsum(-1)       # sums of log decays: 64 bits
    xs, ds = cut(x32), cut(d[..., None])
    bs, cs = (cut(v.float().repeat_interleave(H // G, dim=2)) for v in (Bm, Cm))
    low = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=x.device).tril()
    decay = torch.exp((a[..., :, None] - a[..., None, :]).masked_fill(~low, -math.inf)).float()
    inside = ((cs @ bs.transpose(-1, -2)) * decay) @ (xs * ds)
    own_state = (xs * (ds * torch.exp(a[..., -1:] - a).float()[..., None])).transpose(-1, -2) @ bs     # [B, nc, H, P, N]
    ends = a[..., -1].cumsum(1).transpose(1, 2)                            # [B, H, nc]: log decay up to a chunk's end
    starts = torch.cat([torch.zeros_like(ends[..., :1]), ends], dim=-1)    # up to a chunk's start; the last: the end of all
    after = torch.ones(nc + 1, nc, dtype=torch.bool, device=x.device).tril(-1)
    carry = torch.exp((starts[..., :, None] - ends[..., None, :]).masked_fill(~after, -math.inf)).float()
    states = (carry @ own_state.transpose(1, 2).flatten(3)).unflatten(-1, (P, N))                      # [B, H, nc + 1, P, N]
    if state is not None:
        states = states + torch.exp(starts).float()[..., None, None] * state.float()[:, :, None]
    across = (cs @ states[:, :, :nc].transpose(1, 2).transpose(-1, -2)) * torch.exp(a).float()[..., None]
    y = (inside + across).transpose(2, 3).flatten(1, 2)[:, :T] + D[:, None] * x32
    y = torch.where(valid[..., None], y * _silu(z.float()), zero)
    return y.to(x.dtype), states[:, :, nc]


def _plain_scan_step(x, dt, A, Bm, Cm, D, z, dt_bias, state):
    r = x.shape[1] // Bm.shape[1]
    d = _softplus(dt.float() + dt_bias)
    b, c = Bm.float().repeat_interleave(r, dim=1), Cm.float().repeat_interleave(r, dim=1)
    new = torch.exp(d * A)[..., None, None] * state + (d[..., None] * x.float())[..., None] * b[:, :, None]
    y = (new * c[:, :, None]).sum(-1) + D[:, None] * x.float()
    state.copy_(new)
    return (y * _silu(z.float())).to(x.dtype)


def _plain_norm(v, weight, bias, kind, eps=1e-5):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + eps) * weight
    return v if bias is None else v + bias


def _plain_sandwich(residual, y, post_weight, post_bias, pre_weight, pre_bias, gate, scale, kind):
    u = _plain_norm(y.float(), post_weight, post_bias, kind)
    if gate is not None:
        u = u * (gate.float()[:, None] if gate.dim() == 2 else gate.float())
    h = residual.float() + scale * u
    return h.to(residual.dtype), _plain_norm(h, pre_weight, pre_bias, kind).to(y.dtype)


# ---- one pass -----------------------------------------------------------------------------------------------------------
def _conv(s):
    if own:
        from vit_amd import ssm
        return ssm.causal_conv(s["x"], s["weight"], s["bias"], activation="silu", state=s.get("state"), lengths=s["lengths"], return_state=True)
    return _plain_conv(s["x"], s["weight"], s["bias"], s.get("state"), s["lengths"])


def _conv_step(s):
    if own:
        from vit_amd import ssm
        return ssm.causal_conv_step(s["x"], s["weight"], s["bias"], s["state"], activation="silu")
    return _plain_conv_step(s["x"], s["weight"], s["bias"], s["state"])


def _scan(s):
    if own:
        from vit_amd import ssm
        return ssm.selective_scan(s["x"], s["dt"], s["A"], s["Bm"], s["Cm"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"], state=s["state"],
                                  lengths=s["lengths"], return_state=True)
    return _plain_scan(s["x"], s["dt"], s["A"], s["Bm"], s["Cm"], s["D"], s["z"], s["dt_bias"], s["state"], s["lengths"])


def _scan_step(s):
    if own:
        from vit_amd import ssm
        return ssm.selective_scan_step(s["x"], s["dt"], s["A"], s["Bm"], s["Cm"], s["state"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"])
    return _plain_scan_step(s["x"], s["dt"], s["A"], s["Bm"], s["Cm"], s["D"], s["z"], s["dt_bias"], s["state"])


def _norm(s):
    if own:
        from vit_amd import ssm
        return ssm.sandwich_norm(s["residual"], s["y"], s["post_weight"], s["post_bias"], s["pre_weight"], s["pre_bias"], gate=s["gate"],
                                 scale=s["scale"], kind=s["case"]["kind"])
    return _plain_sandwich(s["residual"], s["y"], s["post_weight"], s["post_bias"], s["pre_weight"], s["pre_bias"], s["gate"], s["scale"], s["case"]["kind"])


def _gradients(outs, douts, s, names):
    names = [k for k in names if s[k] is not None]
    return dict(zip(("d" + k for k in names), torch.autograd.grad(outs, [s[k] for k in names], douts)))


def run(state):
    s, case = state, state["case"]
    if case["op"] == "conv":
        if case["mode"] == "step":
            return {"y": _conv_step(s), "state": s["state"]}
        y, after = _conv(s)
        if case["mode"] == "train":
            return {"y": y.detach(), **_gradients([y], [s["dy"]], s, ("x", "weight", "bias"))}
        return {"y": y, "state": after}
    if case["op"] == "scan":
        if case["mode"] == "step":
            return {"y": _scan_step(s), "state": s["state"]}
        y, after = _scan(s)
        if case["mode"] == "train":
            return {"y": y.detach(), **_gradients([y], [s["dy"]], s, ("x", "dt", "A", "Bm", "Cm", "D", "z", "dt_bias", "state"))}
        return {"y": y, "state": after}
    h, n = _norm(s)
    if case["mode"] == "train":
        return {"h": h.detach(), "n": n.detach(),
                **_gradients([h, n], [s["dh"], s["dn"]], s, ("residual", "y", "post_weight", "post_bias", "pre_weight", "pre_bias", "gate"))}
    return {"h": h, "n": n}


# ---- what a pass cannot do without --------------------------------------------------------------------------------------
def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    B, T, train = case["B"], case.get("T", 1), case["mode"] == "train"
    if case["op"] == "conv":
        C, K = case["C"], case["K"]
        tokens = B * T * C
        small = C * (K + 1) * 4 * (2 if train else 1) + (0 if train else 2 * B * (K - 1) * C * e)
        # forward: x in, y out; backward: x and dy in, dx out
        return {"bytes": tokens * e * (5 if train else 2) + small, "flops": tokens * (2 * K + 4) * (3 if train else 1)}
    if case["op"] == "scan":
        H, P, G, N = case["H"], case["P"], case["G"], case["N"]
        token = H * P * 2 + H + 2 * G * N                  # x, z, dt, B, C
        held = B * H * P * N * 4
        if case["mode"] == "step":
            return {"bytes": B * (token + H * P) * e + 2 * held + 3 * H * 4, "flops": B * H * P * (5 * N + 6)}
        start = held if case["start"] else 0
        if not train:
            return {"bytes": B * T * (token + H * P) * e + start + held + 3 * H * 4, "flops": B * T * H * P * (5 * N + 6)}
        # forward, then its inputs and dy again and their gradients
        return {"bytes": B * T * e * ((token + H * P) + (token + H * P) + token) + 3 * start + 9 * H * 4, "flops": B * T * H * P * (15 * N + 18)}
    E = case["E"]
    r = 2 if case["residual"] == "bf16" else 4
    n = B * T * E
    ge = {"none": 0, "channel": E * 4, "sample": B * E * e, "token": n * e}[case["gate"]]
    vec = E * 4 * (4 if case["kind"] == "layer" else 2)
    forward = n * (2 * r + 2 * e) + ge + vec
    if not train:
        return {"bytes": forward, "flops": 20 * n}
    # backward: residual, y, gate, dh, dn in; gradients of residual, y and gate out
    return {"bytes": forward + n * (3 * r + 3 * e) + 2 * ge + 2 * vec, "flops": 65 * n}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------
def _exact_conv(case, s):
    x, w, bias = (s[k].detach().double() for k in ("x", "weight", "bias"))
    step = case["mode"] == "step"
    if step:
        x = x[:, None]
    B, T, C = x.shape
    K = w.shape[1]
    st = s.get("state")
    past = x.new_zeros(B, K - 1, C) if st is None else st.detach().double()
    lengths = s.get("lengths")
    lens = [T] * B if lengths is None else lengths.tolist()
    full = torch.cat([past, x], 1)
    u = bias.expand(B, T, C).clone()
    for k in range(K):
        u += w[:, k] * full[:, k:k + T]
    sg = 1 / (1 + torch.exp(-u))
    y = u * sg
    for b, n in enumerate(lens):
        y[b, n:] = 0
    if case["mode"] != "train":
        after = torch.stack([full[b, n:n + K - 1] for b, n in enumerate(lens)])
        return {"y": y[:, 0] if step else y, "state": after}
    du = s["dy"].double() * (sg + u * sg * (1 - sg))
    for b, n in enumerate(lens):
        du[b, n:] = 0
    dfull, dw = torch.zeros_like(full), torch.zeros_like(w)
    for k in range(K):
        dfull[:, k:k + T] += w[:, k] * du
        dw[:, k] = (full[:, k:k + T] * du).sum((0, 1))
    return {"y": y, "dx": dfull[:, K - 1:], "dweight": dw, "dbias": du.sum((0, 1))}


def _exact_scan(case, s):
    step, train = case["mode"] == "step", case["mode"] == "train"
    x, dt, Bm, Cm, z = (s[k].detach().double() for k in ("x", "dt", "Bm", "Cm", "z"))
    A, D, bias = (s[k].detach().double() for k in ("A", "D", "dt_bias"))
    if step:
        x, dt, Bm, Cm, z = (v[:, None] for v in (x, dt, Bm, Cm, z))
    B, T, H, P = x.shape
    G, N = Bm.shape[2:]
    if train and (T * B * H * P * N * 8 > 40e9 or T > 8192):     # kept states beyond 40 GB, or too many steps
        return None
    r = H // G
    raw = dt + bias
    d = torch.logaddexp(raw, torch.zeros_like(raw))
    lengths = s.get("lengths")
    live = torch.ones(B, T, device=x.device, dtype=torch.float64)
    if lengths is not None:
        for b, n in enumerate(lengths.tolist()):
            live[b, n:] = 0
    d = d * live[..., None]
    f = torch.exp(d * A)
    st = s.get("state")
    S = x.new_zeros(B, H, P, N) if st is None else st.detach().double()
    kept = x.new_empty(T + 1, B, H, P, N) if train else None
    if train:
        kept[0] = S
    y = torch.empty_like(x)
    heads = torch.arange(H, device=x.device) // r
    for t in range(T):
        S = f[:, t, :, None, None] * S + (d[:, t, :, None] * x[:, t])[..., None] * Bm[:, t, heads][:, :, None]
        y[:, t] = (S * Cm[:, t, heads][:, :, None]).sum(-1)
        if train:
            kept[t + 1] = S
    v = (y + D[:, None] * x) * live[..., None, None]
    sg = 1 / (1 + torch.exp(-z))
    out = v * z * sg
    if not train:
        return {"y": out[:, 0] if step else out, "state": S}
    dy = s["dy"].double() * live[..., None, None]
    dz = dy * v * (sg + z * sg * (1 - sg))
    dv = dy * z * sg
    dx, dd, dB, dC = D[:, None] * dv, torch.zeros_like(d), torch.zeros_like(Bm), torch.zeros_like(Cm)
    dA = torch.zeros_like(A)
    dS = torch.zeros_like(S)
    for t in reversed(range(T)):
        b, c = Bm[:, t, heads], Cm[:, t, heads]
        dS = dS + dv[:, t][..., None] * c[:, :, None]
        dC[:, t] = (kept[t + 1] * dv[:, t][..., None]).sum(2).unflatten(1, (G, r)).sum(2)
        dSb = (dS * b[:, :, None]).sum(-1)
        dx[:, t] += d[:, t, :, None] * dSb
        dB[:, t] = ((d[:, t, :, None] * x[:, t])[..., None] * dS).sum(2).unflatten(1, (G, r)).sum(2)
        da = (dS * kept[t]).sum((2, 3)) * f[:, t]
        dd[:, t] = (dSb * x[:, t]).sum(-1) + da * A
        dA += (da * d[:, t]).sum(0)
        dS = f[:, t, :, None, None] * dS
    draw_ = dd / (1 + torch.exp(-raw)) * live[..., None]
    got = {"y": out, "dx": dx, "ddt": draw_, "dA": dA, "dBm": dB, "dCm": dC, "dD": (dv * x).sum((0, 1, 3)), "dz": dz, "ddt_bias": draw_.sum((0, 1))}
    if st is not None:
        got["dstate"] = dS
    return got


def _exact_norm(case, s):
    E, layer, eps = case["E"], case["kind"] == "layer", 1e-5
    get = lambda k: s[k].detach().double() if s[k] is not None else None  # noqa: E731
    res, y, w1, b1, w2, b2, gate = (get(k) for k in ("residual", "y", "post_weight", "post_bias", "pre_weight", "pre_bias", "gate"))

    def fwd(v, w, b):
        c = v - v.sum(-1, keepdim=True) / E if layer else v
        rs = 1 / torch.sqrt((c ** 2).sum(-1, keepdim=True) / E + eps)
        hat = c * rs
        return hat, rs, hat * w + (b if b is not None else 0)

    def bwd(dout, hat, rs, w):
        q = dout * w
        q = q - hat * (q * hat).sum(-1, keepdim=True) / E - (q.sum(-1, keepdim=True) / E if layer else 0)
        return q * rs, (dout * hat).sum((0, 1)), dout.sum((0, 1))

    g = torch.ones_like(y) if gate is None else gate[:, None].expand_as(y) if gate.dim() == 2 else gate.expand_as(y)
    hat1, rs1, u = fwd(y, w1, b1)
    h = res + s["scale"] * g * u
    hat2, rs2, n = fwd(h, w2, b2)
    if case["mode"] != "train":
        return {"h": h, "n": n}
    dh, dw2, db2 = bwd(s["dn"].double(), hat2, rs2, w2)
    dh = dh + s["dh"].double()
    dy, dw1, db1 = bwd(s["scale"] * g * dh, hat1, rs1, w1)
    got = {"h": h, "n": n, "dresidual": dh, "dy": dy, "dpost_weight": dw1, "dpre_weight": dw2}
    if layer:
        got.update(dpost_bias=db1, dpre_bias=db2)
    if gate is not None:
        dg = s["scale"] * u * dh
        got["dgate"] = dg if case["gate"] == "token" else dg.sum(1) if case["gate"] == "sample" else dg.sum((0, 1))
    return got


def exact(case, seed):
    s = prepare(case, seed)
    return {"conv": _exact_conv, "scan": _exact_scan, "norm": _exact_norm}[case["op"]](case, s)
