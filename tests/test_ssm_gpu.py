"""State-space sequence operators on the GPU against oracle/ref_ssm.py in 64 bits: values and gradients at the sizes where the
kernels change form (chunks of 64 tokens, 64 channels a block, 32 / 64 / 128 states, segments, vector widths), padding that
holds NaN, strides, in-place steps, streams, captured graphs."""
import pytest
import torch

from oracle import ref_ssm as ref
from tests.ssm_cases import DTYPES, close, leaves64, randn, scan_inputs, to

pytestmark = pytest.mark.gpu

SCAN_NAMES = ("x", "dt", "A", "Bm", "Cm", "D", "z", "dt_bias", "state")


def _call(ssm, s, **kw):
    return ssm.selective_scan(s["x"], s["dt"], s["A"], s["Bm"], s["Cm"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"], state=s["state"], **kw)


# B, T, H, P, G, N
SHAPES = [(1, 1, 1, 1, 1, 1), (2, 3, 4, 8, 2, 16), (1, 63, 2, 64, 1, 64), (2, 64, 2, 32, 1, 32), (1, 65, 3, 16, 3, 33), (2, 130, 4, 64, 1, 128),
          (1, 200, 2, 128, 1, 128), (3, 77, 2, 100, 2, 65), (1, 128, 6, 48, 2, 40), (1, 700, 1, 64, 1, 64), (1, 521, 2, 17, 1, 7), (40, 9, 8, 24, 1, 24)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shape", SHAPES)
def test_scan_forward_and_gradients(dev, shape, dtype):
    from vit_amd import ssm
    B, T, H, P, G, N = shape
    s = scan_inputs(sum(shape), DTYPES[dtype], B, T, H, P, G, N, state=T % 2 == 1)
    g = torch.Generator().manual_seed(9)
    dy, dstate = randn(g, B, T, H, P, dtype=DTYPES[dtype]), randn(g, B, H, P, N)
    want_in = leaves64(s)
    wy, wend = ref.selective_scan(**want_in)
    names = [k for k in SCAN_NAMES if s[k] is not None]
    want = torch.autograd.grad([wy, wend], [want_in[k] for k in names], [dy.double(), dstate.double()])
    d = to(s, dev)
    with torch.no_grad():
        y, end = _call(ssm, d, return_state=True)
    close("y", y, wy)
    close("end", end, wend)
    d = {k: v if v is None else v.requires_grad_() for k, v in d.items()}
    y2, end2 = _call(ssm, d, return_state=True)
    assert torch.equal(y2, y) and torch.equal(end2, end)
    got = torch.autograd.grad([y2, end2], [d[k] for k in names], [dy.to(dev), dstate.to(dev)])
    for k, a, b in zip(names, got, want):
        close("d" + k, a, b)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("drop", [("D",), ("z",), ("dt_bias",), ("D", "z", "dt_bias")])
def test_scan_optional_inputs(dev, drop, dtype):
    from vit_amd import ssm
    s = scan_inputs(5, DTYPES[dtype], 2, 70, 4, 32, 2, 16)
    s.update({k: None for k in drop})
    want_in = leaves64(s)
    wy, _ = ref.selective_scan(**want_in)
    names = [k for k in SCAN_NAMES if s[k] is not None]
    dy = randn(torch.Generator().manual_seed(1), *wy.shape, dtype=DTYPES[dtype])
    want = torch.autograd.grad(wy, [want_in[k] for k in names], dy.double())
    d = {k: v if v is None else v.requires_grad_() for k, v in to(s, dev).items()}
    y = _call(ssm, d)
    close("y", y, wy)
    for k, a, b in zip(names, torch.autograd.grad(y, [d[k] for k in names], dy.to(dev)), want):
        close("d" + k, a, b)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_scan_lengths_and_nan_behind_the_end(dev, dtype):
    """Lengths of zero, inside and at the borders of chunks, above T and below zero (clamped); NaN behind every end."""
    from vit_amd import ssm
    T = 150
    lens = torch.tensor([0, 1, 63, 64, 65, 150, 400, -3], dtype=torch.int32)
    B = len(lens)
    s = scan_inputs(6, DTYPES[dtype], B, T, 4, 24, 2, 20, state=True)
    want_in = leaves64(s)
    wy, wend = ref.selective_scan(**want_in, lengths=lens)
    g = torch.Generator().manual_seed(3)
    dy, dend = randn(g, *wy.shape, dtype=DTYPES[dtype]), randn(g, *wend.shape)
    want = torch.autograd.grad([wy, wend], [want_in[k] for k in SCAN_NAMES], [dy.double(), dend.double()])
    behind = torch.arange(T)[None] >= lens.clamp(0, T)[:, None]
    for k in ("x", "dt", "Bm", "Cm", "z"):
        s[k][behind] = float("nan")
    dy[behind] = float("nan")
    d = {k: v.requires_grad_() for k, v in to(s, dev).items()}
    y, end = _call(ssm, d, lengths=lens.to(dev), return_state=True)
    close("y", y, wy)
    close("end", end, wend)
    assert float(y.detach()[behind.to(dev)].abs().max()) == 0.0
    got = torch.autograd.grad([y, end], [d[k] for k in SCAN_NAMES], [dy.to(dev), dend.to(dev)])
    for k, a, b in zip(SCAN_NAMES, got, want):
        close("d" + k, a, b)
        if k in ("x", "dt", "Bm", "Cm", "z"):
            assert float(a[behind.to(dev)].abs().max()) == 0.0


def test_scan_strong_decay_keeps_precision(dev):
    """A token whose step is in the hundreds forgets everything before it; what follows in its chunk stays exact."""
    from vit_amd import ssm
    s = scan_inputs(7, torch.float32, 1, 128, 2, 16, 1, 16)
    s["dt"][:, 20] = 300.0
    s["dt"][:, 90] = 900.0
    want_in = leaves64(s)
    wy, wend = ref.selective_scan(**want_in)
    y, end = _call(ssm, to(s, dev), return_state=True)
    close("end", end, wend)
    for a, b in ((0, 20), (20, 21), (21, 90), (91, 128)):
        close(f"y {a}..{b}", y[:, a:b], wy[:, a:b])


def test_scan_gradient_against_differences(dev):
    from vit_amd import ssm
    s = scan_inputs(8, torch.float32, 1, 66, 2, 8, 1, 8, state=True)
    g = torch.Generator().manual_seed(4)
    way = {k: randn(g, *s[k].shape).double() for k in SCAN_NAMES}
    cot = randn(g, 1, 66, 2, 8).double()
    f = lambda h: float((ref.selective_scan(**{k: s[k].double() + h * way[k] for k in SCAN_NAMES})[0] * cot).sum())  # noqa: E731
    h = 1e-5
    diff = (f(h) - f(-h)) / (2 * h)
    d = {k: v.requires_grad_() for k, v in to(s, dev).items()}
    got = torch.autograd.grad(_call(ssm, d), [d[k] for k in SCAN_NAMES], cot.float().to(dev))
    terms = [float((a.cpu().double() * way[k]).sum()) for k, a in zip(SCAN_NAMES, got)]
    # differences: h^2 of the third derivative and 2^-52 / h of the value; the gradients' own 2e-5 of each term's norms
    size = sum(float(a.cpu().double().norm() * way[k].norm()) for k, a in zip(SCAN_NAMES, got))
    assert abs(sum(terms) - diff) <= 2e-5 * size + 1e-6 * abs(diff), (sum(terms), diff)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shape", [(1, 8, 64, 1, 64), (3, 4, 24, 2, 20), (5, 2, 100, 1, 128), (2, 3, 1, 3, 1), (17, 2, 7, 1, 5), (2, 2, 64, 1, 96)])
def test_scan_step_is_the_scan_one_token_on(dev, shape, dtype):
    from vit_amd import ssm
    B, H, P, G, N = shape
    s = scan_inputs(11, DTYPES[dtype], B, None, H, P, G, N, state=True)
    one = {k: v[:, None].double() if k in ("x", "dt", "Bm", "Cm", "z") else v.double() for k, v in s.items()}
    wy, wend = ref.selective_scan(**one)
    d = to(s, dev)
    state = d.pop("state")
    y = ssm.selective_scan_step(d["x"], d["dt"], d["A"], d["Bm"], d["Cm"], state, D=d["D"], z=d["z"], dt_bias=d["dt_bias"])
    close("y", y, wy[:, 0])
    close("state", state, wend)
    state = s["state"].to(dev)
    y = ssm.selective_scan_step(d["x"], d["dt"], d["A"], d["Bm"], d["Cm"], state)       # without the optional inputs
    wy, wend = ref.selective_scan(one["x"], one["dt"], one["A"], one["Bm"], one["Cm"], state=one["state"])
    close("y", y, wy[:, 0])
    close("state", state, wend)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_prompt_then_tokens_is_the_whole(dev, dtype):
    """Convolution and scan of a prompt, then token by token on the kept states, against one pass over everything."""
    from vit_amd import ssm
    B, T, T0, H, P, G, N, K = 2, 90, 67, 2, 32, 1, 16, 4
    g = torch.Generator().manual_seed(12)
    W = H * P + 2 * G * N
    raw, w, b = randn(g, B, T, W, dtype=DTYPES[dtype]).to(dev), randn(g, W, K, scale=0.5).to(dev), randn(g, W, scale=0.1).to(dev)
    s = to(scan_inputs(13, DTYPES[dtype], B, T, H, P, G, N), dev)

    def cut(u):
        return u[..., :H * P].unflatten(-1, (H, P)), u[..., H * P:H * P + G * N].unflatten(-1, (G, N)), u[..., H * P + G * N:].unflatten(-1, (G, N))

    x, Bm, Cm = cut(ssm.causal_conv(raw, w, b, activation="silu"))
    kw = dict(D=s["D"], dt_bias=s["dt_bias"])
    whole, end = ssm.selective_scan(x, s["dt"], s["A"], Bm, Cm, z=s["z"], return_state=True, **kw)
    u, conv = ssm.causal_conv(raw[:, :T0], w, b, activation="silu", return_state=True)
    x, Bm, Cm = cut(u)
    part, state = ssm.selective_scan(x, s["dt"][:, :T0], s["A"], Bm, Cm, z=s["z"][:, :T0], return_state=True, **kw)
    ys = [part]
    for t in range(T0, T):
        x, Bm, Cm = cut(ssm.causal_conv_step(raw[:, t], w, b, conv, activation="silu"))
        ys.append(ssm.selective_scan_step(x, s["dt"][:, t], s["A"], Bm, Cm, state, z=s["z"][:, t], **kw)[:, None])
    close("y", torch.cat(ys, 1), whole.double().cpu())
    close("state", state, end.double().cpu())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("B,T,C,K,silu,state,lens", [
    (1, 1, 1, 2, True, False, None), (2, 2, 7, 4, True, True, None), (3, 17, 40, 4, True, True, [0, 5, 17]), (2, 100, 64, 3, False, False, None),
    (1, 300, 24, 6, True, True, None), (2, 64, 130, 5, False, True, [1, 64]), (4, 33, 256, 4, True, False, [33, 2, 1, 3]), (2, 70, 517, 2, True, True, [70, 69])])
def test_conv(dev, B, T, C, K, silu, state, lens, dtype):
    from vit_amd import ssm
    g = torch.Generator().manual_seed(T * C + K)
    dt = DTYPES[dtype]
    x = randn(g, B, T, C + 16, dtype=dt)[:, :, 8:8 + C]
    w, b = randn(g, C, K, scale=0.5), randn(g, C, scale=0.2)
    st = randn(g, B, K - 1, C, dtype=dt) if state else None
    dy, dend = randn(g, B, T, C, dtype=dt), randn(g, B, K - 1, C, dtype=dt)
    lengths = None if lens is None else torch.tensor(lens, dtype=torch.int32)
    leaf = [None if v is None else v.double().requires_grad_() for v in (x, w, b, st)]
    wy, wend = ref.causal_conv(leaf[0], leaf[1], leaf[2], silu=silu, state=leaf[3], lengths=lengths)
    names = ["x", "w", "b"] + (["state"] if state else [])
    want = torch.autograd.grad([wy, wend], [v for v in leaf if v is not None], [dy.double(), dend.double()])
    if lens is not None:
        behind = torch.arange(T)[None] >= lengths[:, None]
        x[behind] = float("nan")
        dy[behind] = float("nan")
    d = to(dict(x=x, w=w, b=b, st=st), dev)
    d = [v if v is None else v.requires_grad_() for v in (d["x"], d["w"], d["b"], d["st"])]
    y, end = ssm.causal_conv(d[0], d[1], d[2], activation="silu" if silu else None, state=d[3], lengths=None if lens is None else lengths.to(dev),
                             return_state=True)
    close("y", y, wy)
    close("end", end, wend)
    for k, a, c in zip(names, torch.autograd.grad([y, end], [v for v in d if v is not None], [dy.to(dev), dend.to(dev)]), want):
        close("d" + k, a, c)
    if T == 2:       # one more token on the kept inputs
        tok = randn(g, B, C, dtype=dt)
        wy, wst = ref.causal_conv(tok[:, None].double(), w.double(), b.double(), silu=silu, state=wend.detach())
        end = end.detach().clone()
        close("step", ssm.causal_conv_step(tok.to(dev), d[1].detach(), d[2].detach(), end, activation="silu" if silu else None), wy[:, 0])
        close("state", end, wst)


@pytest.mark.parametrize("rdt,dt", [("f32", "bf16"), ("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("B,T,E,gate,kind", [(1, 1, 1, None, "rms"), (2, 3, 256, "channel", "layer"), (3, 5, 100, "sample", "rms"), (2, 33, 512, "token", "layer"),
                                             (5, 7, 1024, "sample", "layer"), (1, 9, 387, "channel", "rms"), (2, 2, 2048, "channel", "layer"),
                                             (1, 3, 4096, "token", "layer"), (2, 3, 1025, "sample", "layer"), (1, 700, 64, "channel", "layer")])
def test_sandwich_norm(dev, B, T, E, gate, kind, rdt, dt):
    from vit_amd import ssm
    g = torch.Generator().manual_seed(E + T)
    lay = kind == "layer"
    gdt = torch.float32 if gate == "channel" else DTYPES[dt]
    shape = {None: None, "channel": (E,), "sample": (B, E), "token": (B, T, E)}[gate]
    s = dict(residual=randn(g, B, T, E, dtype=DTYPES[rdt]), y=randn(g, B, T, E, dtype=DTYPES[dt], shift=0.5), post_weight=randn(g, E, shift=1.0, scale=0.2),
             post_bias=randn(g, E) if lay else None, pre_weight=randn(g, E, shift=1.0, scale=0.2), pre_bias=randn(g, E) if lay else None,
             gate=None if gate is None else randn(g, *shape, dtype=gdt))
    dh, dn = randn(g, B, T, E, dtype=DTYPES[rdt]), randn(g, B, T, E, dtype=DTYPES[dt])
    leaf = leaves64(s)
    wh, wn = ref.sandwich_norm(**leaf, scale=0.7, kind=kind, eps=1e-3)
    names = [k for k in s if s[k] is not None]
    want = torch.autograd.grad([wh, wn], [leaf[k] for k in names], [dh.double(), dn.double()])
    d = {k: v if v is None else v.to(dev).requires_grad_() for k, v in s.items()}
    h, n = ssm.sandwich_norm(**d, scale=0.7, kind=kind, eps=1e-3)
    assert h.dtype == DTYPES[rdt] and n.dtype == DTYPES[dt]
    close("h", h, wh)
    close("n", n, wn)
    for k, a, b in zip(names, torch.autograd.grad([h, n], [d[k] for k in names], [dh.to(dev), dn.to(dev)]), want):
        if E == 1 and k != "residual":      # of one column the norm is a constant (or a sign): exact gradients are near zero
            assert float((a.double().cpu() - b).abs().max()) <= 1e-2 * (1 + float(b.abs().max()))
            continue
        close("d" + k, a, b)


def test_runs_of_the_same_call_give_the_same_bits(dev):
    from vit_amd import ssm
    s = {k: v.requires_grad_() for k, v in to(scan_inputs(21, torch.bfloat16, 3, 400, 8, 64, 1, 64, state=True), dev).items()}
    dy = torch.randn(3, 400, 8, 64, device=dev).bfloat16()
    runs = []
    for _ in range(3):
        y = _call(ssm, s)
        runs.append([y.detach()] + list(torch.autograd.grad(y, [s[k] for k in SCAN_NAMES], dy)))
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], r))


def test_no_tokens(dev):
    from vit_amd import ssm
    s = to(scan_inputs(22, torch.float32, 2, 1, 2, 8, 1, 8, state=True), dev)
    s = {k: v[:, :0] if k in ("x", "dt", "Bm", "Cm", "z") else v for k, v in s.items()}
    y, end = _call(ssm, s, return_state=True)
    assert y.shape == (2, 0, 2, 8) and torch.equal(end, s["state"])
    st = torch.randn(2, 3, 5, device=dev)
    y, end = ssm.causal_conv(torch.zeros(2, 0, 5, device=dev), torch.ones(5, 4, device=dev), state=st, return_state=True)
    assert y.shape == (2, 0, 5) and torch.equal(end, st)
    s = {k: v.detach().requires_grad_() for k, v in s.items()}
    y, end = _call(ssm, s, return_state=True)
    g = torch.autograd.grad([y, end], [s["A"], s["state"]], [torch.zeros_like(y), torch.ones_like(end)])
    assert float(g[0].abs().max()) == 0.0 and torch.equal(g[1], torch.ones_like(end))


def test_another_stream_and_order(dev):
    """A call on another stream than the inputs' own, and inputs in another memory order."""
    from vit_amd import ssm
    s = to(scan_inputs(23, torch.bfloat16, 2, 300, 4, 64, 2, 64), dev)
    want = _call(ssm, s)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        got = _call(ssm, s)
    torch.cuda.current_stream().wait_stream(other)
    assert torch.equal(got, want)
    swapped = dict(s, x=s["x"].transpose(0, 1).contiguous().transpose(0, 1), Bm=s["Bm"].transpose(2, 3).contiguous().transpose(2, 3),
                   z=s["z"].transpose(2, 3).contiguous().transpose(2, 3), dt=s["dt"].transpose(1, 2).contiguous().transpose(1, 2))
    assert torch.equal(_call(ssm, swapped), want)
    odd = dict(s, x=torch.empty(2 * 300 * 4 * 64 + 1, dtype=torch.bfloat16, device=dev)[1:].view(2, 300, 4, 64).copy_(s["x"]))   # 2-byte alignment
    assert torch.equal(_call(ssm, odd), want)


def test_captured_steps_replay(dev):
    """A captured token step (convolution and scan in place on kept states) and a captured prompt, replayed with new inputs and
    eager work between, against the eager calls."""
    from vit_amd import ssm
    B, H, P, N, K = 2, 4, 32, 32, 4
    W = H * P + 2 * N
    g = torch.Generator().manual_seed(30)
    w, b = randn(g, W, K).to(dev), randn(g, W).to(dev)
    s = to(scan_inputs(31, torch.bfloat16, B, None, H, P, 1, N, state=True), dev)
    raw = randn(g, B, W, dtype=torch.bfloat16).to(dev)
    conv, state = randn(g, B, K - 1, W, dtype=torch.bfloat16).to(dev), s["state"].clone()

    def token(raw, conv, state):
        u = ssm.causal_conv_step(raw, w, b, conv, activation="silu")
        x, Bm, Cm = u[:, :H * P].unflatten(-1, (H, P)), u[:, H * P:H * P + N, None].transpose(1, 2), u[:, H * P + N:, None].transpose(1, 2)
        return ssm.selective_scan_step(x, s["dt"], s["A"], Bm, Cm, state, D=s["D"], z=s["z"], dt_bias=s["dt_bias"])

    long = to(scan_inputs(32, torch.bfloat16, 1, 600, 1, 64, 1, 64), dev)       # few rows: cut into segments
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        token(raw.clone(), conv.clone(), state.clone())
        _call(ssm, long)
    torch.cuda.current_stream().wait_stream(side)
    c2, s2 = conv.clone(), state.clone()
    graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = token(raw, conv, state)
    with torch.cuda.graph(graph2):
        out2 = _call(ssm, long)
    conv.copy_(c2)
    state.copy_(s2)
    for i in range(4):
        raw.copy_(randn(g, B, W, dtype=torch.bfloat16))
        long["x"].copy_(randn(g, 1, 600, 1, 64, dtype=torch.bfloat16))
        graph.replay()
        graph2.replay()
        want = token(raw, c2, s2)
        assert torch.equal(out, want) and torch.equal(conv, c2) and torch.equal(state, s2)
        assert torch.equal(out2, _call(ssm, long))
        torch.cuda.synchronize()


def _scan_case(seed, dtype, dev, B, T, H, P, G, N, **kw):
    """CPU inputs and their 64-bit outputs and gradients (cotangent: every output), and the device copy as leaves."""
    s = scan_inputs(seed, dtype, B, T, H, P, G, N, **kw)
    names = [k for k in SCAN_NAMES if s[k] is not None]
    dy = randn(torch.Generator().manual_seed(seed), B, T, H, P, dtype=dtype)
    leaf = leaves64(s)
    wy, _ = ref.selective_scan(**leaf)
    want = torch.autograd.grad(wy, [leaf[k] for k in names], dy.double())
    return s, names, dy, wy, dict(zip(names, want)), {k: v if v is None else v.requires_grad_() for k, v in to(s, dev).items()}


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_token_strides_past_32_bits(dev, dtype):
    """Each of x, z, Bm, Cm, dt and dy alone with tokens 2^25 elements apart (70 of them: byte offsets past 2^32)."""
    from vit_amd import ssm
    T, H, P, N = 70, 2, 32, 32
    s, names, dy, wy, want, d = _scan_case(40, DTYPES[dtype], dev, 1, T, H, P, 1, N)
    far = torch.empty((T - 1) * 2 ** 25 + H * P, dtype=DTYPES[dtype], device=dev)

    def spread(v):
        inner = v[0, 0].numel()
        out = far.as_strided((1, T, inner), (far.numel(), 2 ** 25, 1)).unflatten(-1, v.shape[2:])
        return out.copy_(v.detach())

    for k in ("x", "z", "Bm", "Cm", "dt", "dy"):
        c = dict(d)
        if k != "dy":
            c[k] = spread(d[k]).requires_grad_()
        y = _call(ssm, c)
        close("y " + k, y, wy)
        got = torch.autograd.grad(y, [c[n] for n in names], spread(dy.to(dev)) if k == "dy" else dy.to(dev))
        for n, a in zip(names, got):
            close(f"d{n}, {k} far", a, want[n])


def test_expanded_gradient(dev):
    """A sum's gradient is one element spread out: strides of zero."""
    from vit_amd import ssm
    s, names, _, wy, _, d = _scan_case(41, torch.float32, dev, 2, 100, 2, 16, 1, 16)
    leaf = leaves64(s)
    want = torch.autograd.grad(ref.selective_scan(**leaf)[0].sum(), [leaf[k] for k in names])
    for k, a, b in zip(names, torch.autograd.grad(_call(ssm, d).sum(), [d[k] for k in names]), want):
        close("d" + k, a, b)
    x, w = randn(torch.Generator().manual_seed(1), 2, 9, 8), randn(torch.Generator().manual_seed(2), 8, 4)
    lx, lw = x.double().requires_grad_(), w.double().requires_grad_()
    want = torch.autograd.grad(ref.causal_conv(lx, lw)[0].sum(), [lx, lw])
    gx, gw = x.to(dev).requires_grad_(), w.to(dev).requires_grad_()
    for a, b in zip(torch.autograd.grad(ssm.causal_conv(gx, gw).sum(), [gx, gw]), want):
        close("d", a, b)


def test_steps_near_the_types_end(dev):
    """A step of 1e37 (a decay whose logarithm is outside fp32, two in one chunk) forgets what came before, and no more."""
    from vit_amd import ssm
    s = scan_inputs(42, torch.float32, 1, 100, 2, 16, 1, 16, state=True)
    s["A"].fill_(-16.0)
    for t in (30, 40, 80):
        s["dt"][:, t] = 1e37
        s["x"][:, t] *= 1e-34
    leaf = leaves64(s)
    wy, wend = ref.selective_scan(**leaf)
    dy = randn(torch.Generator().manual_seed(5), *wy.shape)
    want = torch.autograd.grad(wy, [leaf[k] for k in ("Bm", "Cm", "z", "state")], dy.double())
    d = {k: v.requires_grad_() for k, v in to(s, dev).items()}
    y, end = _call(ssm, d, return_state=True)
    for a, b in ((0, 30), (30, 31), (31, 40), (40, 41), (41, 60), (60, 80), (80, 100)):
        close(f"y {a}..{b}", y[:, a:b], wy[:, a:b])
    close("end", end, wend)
    for k, a, b in zip(("Bm", "Cm", "z", "state"), torch.autograd.grad(y, [d[k] for k in ("Bm", "Cm", "z", "state")], dy.to(dev)), want):
        close("d" + k, a, b)


def test_second_derivatives_are_refused(dev):
    from vit_amd import ssm
    s = {k: v.requires_grad_() for k, v in to(scan_inputs(43, torch.float32, 1, 5, 1, 4, 1, 4, state=True), dev).items()}
    x, w, e = s["x"].flatten(2), torch.ones(4, 4, device=dev, requires_grad=True), torch.ones(4, device=dev, requires_grad=True)
    for out, leaf in ((_call(ssm, s), s["x"]), (ssm.causal_conv(x, w), w), (ssm.sandwich_norm(x, x, e, None, e, None)[1], e)):
        with pytest.raises(RuntimeError, match="second derivatives"):
            torch.autograd.grad(out.sum(), leaf, create_graph=True)


def test_a_graph_notices_a_state_that_moved_on(dev):
    """The convolution's backward pass reads the kept inputs it started from; a step on them in between is an error, not a wrong
    gradient."""
    from vit_amd import ssm
    x, w, st = torch.randn(2, 5, 8, device=dev), torch.randn(8, 4, device=dev, requires_grad=True), torch.randn(2, 3, 8, device=dev)
    y = ssm.causal_conv(x, w, state=st)
    ssm.causal_conv_step(x[:, 0], w.detach(), None, st)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    s = to(scan_inputs(44, torch.float32, 2, None, 2, 8, 1, 8, state=True), dev)
    before = s["state"]._version
    ssm.selective_scan_step(s["x"], s["dt"], s["A"], s["Bm"], s["Cm"], s["state"])
    assert s["state"]._version == before + 1
    with torch.inference_mode():
        ssm.selective_scan_step(s["x"], s["dt"], s["A"], s["Bm"], s["Cm"], s["state"].clone())


def test_large_batches_of_short_samples(dev):
    """More samples than a grid's second dimension holds, forward and backward."""
    from vit_amd import ssm
    B, T, C, E = 70000, 2, 4, 8
    g = torch.Generator().manual_seed(45)
    x, w, dy = randn(g, B, T, C), randn(g, C, 3), randn(g, B, T, C)
    lx, lw = x.double().requires_grad_(), w.double().requires_grad_()
    wy, _ = ref.causal_conv(lx, lw, silu=True)
    want = torch.autograd.grad(wy, [lx, lw], dy.double())
    gx, gw = x.to(dev).requires_grad_(), w.to(dev).requires_grad_()
    y = ssm.causal_conv(gx, gw, activation="silu")
    close("y", y, wy)
    for a, b in zip(torch.autograd.grad(y, [gx, gw], dy.to(dev)), want):
        close("d", a, b)
    s, names, dy, wy, want, d = _scan_case(46, torch.float32, dev, B, 1, 1, 2, 1, 2, state=True)
    y = _call(ssm, d)
    close("y", y, wy)
    for k, a in zip(names, torch.autograd.grad(y, [d[k] for k in names], dy.to(dev))):
        close("d" + k, a, want[k])
    for T in (1, 2):          # a gate per sample
        s = dict(residual=randn(g, B, T, E), y=randn(g, B, T, E), post_weight=randn(g, E), post_bias=None, pre_weight=randn(g, E), pre_bias=None,
                 gate=randn(g, B, E))
        dn = randn(g, B, T, E)
        leaf = leaves64(s)
        _, wn = ref.sandwich_norm(**leaf)
        names = [k for k in s if s[k] is not None]
        want = torch.autograd.grad(wn, [leaf[k] for k in names], dn.double())
        d = {k: v if v is None else v.to(dev).requires_grad_() for k, v in s.items()}
        n = ssm.sandwich_norm(**d)[1]
        close("n", n, wn)
        for k, a, b in zip(names, torch.autograd.grad(n, [d[k] for k in names], dn.to(dev)), want):
            close("d" + k, a, b)


def test_two_streams_at_once(dev):
    """Two long calls in flight on two streams, forward and backward, each with its own workspace."""
    from vit_amd import ssm
    cases = [to(scan_inputs(50 + i, torch.bfloat16, 2, 2000, 4, 64, 1, 128), dev) for i in range(2)]
    names = [k for k in SCAN_NAMES if cases[0][k] is not None]
    leaves = [{k: v if v is None else v.requires_grad_() for k, v in s.items()} for s in cases]
    dy = torch.randn(2, 2000, 4, 64, device=dev).bfloat16()

    def run(s):
        y = _call(ssm, s)
        return [y.detach()] + list(torch.autograd.grad(y, [s[k] for k in names], dy))

    alone = [run(s) for s in leaves]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in leaves]
    both = []
    for s, st in zip(leaves, streams):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            both.append(run(s))
    torch.cuda.synchronize()
    for a, b in zip(alone, both):
        assert all(torch.equal(u, v) for u, v in zip(a, b))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_captured_training_step_replays(dev, dtype):
    """Convolution, scan (cut into segments) and norms with their backward passes in one captured graph, replayed with new
    inputs and eager work between, against eager calls."""
    from vit_amd import ssm
    B, T, H, P, N = 1, 600, 2, 32, 32
    W = H * P + 2 * N
    dt = DTYPES[dtype]
    g = torch.Generator().manual_seed(60)
    raw = randn(g, B, T, W, dtype=dt).to(dev).requires_grad_()
    rest = to(scan_inputs(61, dt, B, T, H, P, 1, N), dev)
    par = dict(w=randn(g, W, 4, scale=0.5), b=randn(g, W, scale=0.1), pw=randn(g, H * P, shift=1.0), nw=randn(g, H * P, shift=1.0), gate=randn(g, B, H * P))
    par = {k: v.to(dev).requires_grad_() for k, v in par.items()}
    leaves = [raw, *par.values()] + [rest[k].requires_grad_() for k in ("A", "D", "dt_bias")]
    res = randn(g, B, T, H * P).to(dev)
    cot = randn(g, B, T, H * P, dtype=dt).to(dev)

    def step():
        u = ssm.causal_conv(raw, par["w"], par["b"], activation="silu")
        x, Bm, Cm = u[..., :H * P].unflatten(-1, (H, P)), u[..., H * P:H * P + N].unflatten(-1, (1, N)), u[..., H * P + N:].unflatten(-1, (1, N))
        y = ssm.selective_scan(x, rest["dt"], rest["A"], Bm, Cm, D=rest["D"], z=rest["z"], dt_bias=rest["dt_bias"])
        n = ssm.sandwich_norm(res, y.flatten(2), par["pw"], None, par["nw"], None, gate=par["gate"], kind="rms")[1]
        return [n.detach()] + list(torch.autograd.grad(n, leaves, cot))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        with torch.no_grad():
            raw.copy_(randn(g, B, T, W, dtype=dt))
        cot.copy_(randn(g, B, T, H * P, dtype=dt))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_mixed_devices_are_refused(dev):
    from vit_amd import ssm
    s = to(scan_inputs(70, torch.float32, 1, 5, 1, 4, 1, 4), dev)
    for k in ("A", "Bm", "z"):
        with pytest.raises(ValueError, match="cpu"):
            _call(ssm, dict(s, **{k: s[k].cpu()}))
    with pytest.raises(ValueError, match="cpu"):
        ssm.causal_conv(torch.zeros(1, 4, 4, device=dev), torch.zeros(4, 4))
    with pytest.raises(ValueError, match="cpu"):
        ssm.sandwich_norm(torch.zeros(3, 8, device=dev), torch.zeros(3, 8), torch.ones(8, device=dev), None, torch.ones(8, device=dev), None)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_scan_lengths_over_segments(dev, dtype):
    """A sequence that is cut into segments, with samples that end before, inside and at the borders of them."""
    from vit_amd import ssm
    T = 640
    lens = torch.tensor([0, 70, 256, 257, 640, 639], dtype=torch.int32)
    s = scan_inputs(80, DTYPES[dtype], len(lens), T, 2, 24, 1, 20, state=True)
    want_in = leaves64(s)
    wy, wend = ref.selective_scan(**want_in, lengths=lens)
    g = torch.Generator().manual_seed(81)
    dy, dend = randn(g, *wy.shape, dtype=DTYPES[dtype]), randn(g, *wend.shape)
    want = torch.autograd.grad([wy, wend], [want_in[k] for k in SCAN_NAMES], [dy.double(), dend.double()])
    behind = torch.arange(T)[None] >= lens[:, None]
    for k in ("x", "dt", "Bm", "Cm", "z"):
        s[k][behind] = float("nan")
    dy[behind] = float("nan")
    d = {k: v.requires_grad_() for k, v in to(s, dev).items()}
    y, end = _call(ssm, d, lengths=lens.to(dev), return_state=True)
    close("y", y, wy)
    close("end", end, wend)
    for k, a, b in zip(SCAN_NAMES, torch.autograd.grad([y, end], [d[k] for k in SCAN_NAMES], [dy.to(dev), dend.to(dev)]), want):
        close("d" + k, a, b)


def test_kept_states_past_32_bits(dev):
    """4300 chunks of 64 heads x 64 x 128 states: more than 2^31 kept values, inputs past 2^31 bytes.  The end of the sequence against
    the same tokens alone on the state that the first part leaves."""
    from vit_amd import ssm
    T, T0, H, P, N = 4300 * 64 - 7, 4290 * 64, 64, 64, 128
    g = torch.Generator(device=dev).manual_seed(90)
    r = lambda *shape: torch.randn(*shape, generator=g, device=dev, dtype=torch.bfloat16)  # noqa: E731
    s = dict(x=r(1, T, H, P), dt=r(1, T, H), Bm=r(1, T, 1, N), Cm=r(1, T, 1, N), z=r(1, T, H, P), A=-torch.rand(H, generator=g, device=dev) - 0.5,
             D=torch.rand(H, generator=g, device=dev), dt_bias=torch.full((H,), -3.0, device=dev), state=None)
    over = ("x", "dt", "Bm", "Cm", "z")
    leaf = {k: v.requires_grad_() if k in over else v for k, v in s.items()}
    dy = torch.zeros(1, T, H, P, device=dev, dtype=torch.bfloat16)
    dy[:, T0:] = r(1, T - T0, H, P)
    y = _call(ssm, leaf)
    grads = [v[:, T0:].clone() for v in torch.autograd.grad(y, [leaf[k] for k in over], dy)]
    y = y.detach()[:, T0:].clone()
    with torch.no_grad():
        _, state = _call(ssm, {k: v[:, :T0] if k in over else v for k, v in s.items()}, return_state=True)
    tail = {k: v.detach()[:, T0:].clone().requires_grad_() if k in over else v for k, v in s.items()}
    tail["state"] = state
    yt = _call(ssm, tail)
    # (two runs of the same definition: each within the tolerance of it)
    err = float((y.double() - yt.detach().double()).norm() / yt.detach().double().norm())
    assert err <= 2 * (2.0 ** -8 + 2.0 ** -10), err
    for k, a, b in zip(over, grads, torch.autograd.grad(yt, [tail[k] for k in over], dy[:, T0:])):
        err = float((a.double() - b.double()).norm() / b.double().norm())
        assert err <= 2 * (2.0 ** -8 + 2.0 ** -10), (k, err)
    del leaf, s, tail, grads, y, yt, dy, state
    torch.cuda.empty_cache()
