"""State-space operators on the GPU, value by value, against oracle/ref_ssm.py and the formulas in 64 bits: results that are rounded
once, decays and gates at the ends of their range, masks, empty batches, backward passes of one chunk, row counts around the
segments."""
import pytest
import torch

from oracle import ref_ssm as ref
from tests.ssm_cases import DTYPES, close, leaves64, randn, scan_inputs, to

pytestmark = pytest.mark.gpu


def _call(ssm, s, **kw):
    return ssm.selective_scan(s["x"], s["dt"], s["A"], s["Bm"], s["Cm"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"], state=s["state"], **kw)


def _within(name, got, want, bound):
    """Every value within its own bound."""
    off = (got.detach().double().cpu() - want).abs()
    worst = float((off / bound).max())
    assert worst <= 1.0, (name, worst, int((off > bound).sum()), off.numel())


@pytest.mark.parametrize("shape", [(1, 8, 2, 64, 1, 64), (2, 64, 3, 24, 1, 16), (2, 130, 4, 64, 2, 128), (1, 600, 2, 40, 1, 33)])
def test_gate_gradient_is_rounded_once(dev, shape):
    """dz = dy v silu'(z) of bf16 calls: half a step of the value, 2^-8, and what v itself is off by.  v is held in 32 bits: its
    operands of two parts leave 2^-17 of the terms' size, and at most 192 terms a chunk are added with 2^-24 each (2^-16.4),
    so 2^-15 of the sum of the terms' sizes (|x|, |B|, |C|, |D| in the place of x, B, C, D).  silu'(z) = s + z s (1 - s): 2^-21 of
    its two parts' sizes."""
    from vit_amd import ssm
    B, T, H, P, G, N = shape
    s = scan_inputs(sum(shape), torch.bfloat16, B, T, H, P, G, N, state=T == 130)
    dy = randn(torch.Generator().manual_seed(2), B, T, H, P, dtype=torch.bfloat16)
    d = {k: v if v is None else v.double() for k, v in s.items()}
    bare = dict(d, z=None)
    v, _ = ref.selective_scan(**bare)
    size, _ = ref.selective_scan(**{k: t.abs() if t is not None and k in ("x", "Bm", "Cm", "D", "state") else t for k, t in bare.items()})
    sg = torch.sigmoid(d["z"])
    parts = sg + d["z"].abs() * sg * (1 - sg)
    want = dy.double() * v * (sg + d["z"] * sg * (1 - sg))
    bound = 2.0 ** -8 * want.abs() + (1 + 2.0 ** -8) * dy.double().abs() * parts * (2.0 ** -15 * size + 2.0 ** -21 * v.abs())
    leaf = to(s, dev)
    leaf["z"].requires_grad_()
    (dz,) = torch.autograd.grad(_call(ssm, leaf), [leaf["z"]], dy.to(dev))
    _within("dz", dz, want, bound + 1e-30)


def test_function_transforms_are_refused(dev):
    """torch.func's wrappers hold no memory a kernel could read: an error, never a result without its derivative."""
    from vit_amd import ssm
    x, w = torch.randn(2, 5, 8, device=dev), torch.randn(8, 4, device=dev)
    f = lambda v: ssm.causal_conv(v, w)  # noqa: E731
    for call in (lambda: torch.func.jvp(f, (x,), (x,)), lambda: torch.func.grad(lambda v: f(v).sum())(x), lambda: torch.func.vmap(f)(x[None])):
        with pytest.raises(RuntimeError):
            call()
    with torch.autograd.forward_ad.dual_level():       # a tangent that arrives with the gradient
        y = ssm.causal_conv(x.clone().requires_grad_(), w)
        dy = torch.autograd.forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.backward(y, dy)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("low", [float("-inf"), "min"])
def test_tokens_masked_through_dt_do_nothing(dev, low, dtype):
    """dt of -infinity or of the type's lowest value: softplus is zero, the state stays bit for bit, and what starts from nothing
    stays nothing."""
    from vit_amd import ssm
    dt = DTYPES[dtype]
    low = torch.finfo(dt).min if low == "min" else low
    B, T, H, P, G, N = 2, 100, 4, 24, 2, 20
    s = scan_inputs(70, dt, B, T, H, P, G, N)
    s["x"].mul_(64.0)
    s["D"] = s["z"] = None
    s["dt"].fill_(low)
    d = to(s, dev)
    y, end = _call(ssm, d, return_state=True)
    assert float(y.abs().max()) == 0.0 and float(end.abs().max()) == 0.0
    state = torch.randn(B, H, P, N, device=dev)
    _, end = _call(ssm, dict(d, state=state), return_state=True)
    assert torch.equal(end, state)
    for start in (state, torch.zeros_like(state)):
        moved = start.clone()
        ssm.selective_scan_step(d["x"][:, 0], d["dt"][:, 0], d["A"], d["Bm"][:, 0], d["Cm"][:, 0], moved, dt_bias=d["dt_bias"])
        assert torch.equal(moved, start)
    # some of the tokens masked: values and gradients
    s = scan_inputs(71, dt, B, T, H, P, G, N, state=True)
    s["dt"][:, 10:80:3] = low
    s["dt"][1, 64:] = low
    want_in = leaves64(s)
    wy, wend = ref.selective_scan(**want_in)
    names = [k for k in want_in if want_in[k] is not None]
    g = torch.Generator().manual_seed(72)
    dy, dend = randn(g, *wy.shape, dtype=dt), randn(g, *wend.shape)
    want = torch.autograd.grad([wy, wend], [want_in[k] for k in names], [dy.double(), dend.double()])
    leaf = {k: v.requires_grad_() for k, v in to(s, dev).items()}
    y, end = _call(ssm, leaf, return_state=True)
    close("y", y, wy)
    close("end", end, wend)
    for k, a, b in zip(names, torch.autograd.grad([y, end], [leaf[k] for k in names], [dy.to(dev), dend.to(dev)]), want):
        close("d" + k, a, b)
        if k == "dt":
            assert float(a[s["dt"].to(dev) == low].abs().max()) == 0.0


def test_fp32_gates_over_their_range(dev):
    """silu of fp32 values from -85 to 85, value by value: exp(-x) to 1.5 units in the last place (v_exp_f32: one, and its correction's
    rounding), the sum with 1 (0.5), v_rcp_f32 (one) and the product (0.5): 3.5, held to 4 units of 2^-23.  silu'(x) = s + x s (1 - s)
    where x < -2: s to 3 units, twice in its second term, and four roundings: 8 of its parts' sizes, which are within 2.2 of its
    own there and further out within 1.1: 8 of the parts."""
    from vit_amd import ssm
    x = torch.linspace(-85, 85, 4096)
    x64 = x.double()
    sg = torch.sigmoid(x64)
    want = x64 * sg
    w = torch.tensor([0.0, 1.0]).repeat(4096, 1)
    xd = x.to(dev).view(1, 1, -1).requires_grad_()
    y = ssm.causal_conv(xd, w.to(dev), activation="silu")
    tiny = 1e-36      # (below, results have left the normal range's neighbourhood)
    _within("conv", y[0, 0], want, 4 * 2.0 ** -23 * want.abs() + tiny)
    step = ssm.causal_conv_step(xd[0].detach(), w.to(dev), None, torch.zeros(1, 1, 4096, device=dev), activation="silu")
    _within("step", step[0], want, 4 * 2.0 ** -23 * want.abs() + tiny)
    slope, parts = sg + x64 * sg * (1 - sg), sg + x64.abs() * sg * (1 - sg)
    (dx,) = torch.autograd.grad(y.sum(), [xd])
    at = x64 < -2
    _within("conv dx", dx[0, 0].cpu()[at], slope[at], 8 * 2.0 ** -23 * parts[at] + tiny)
    # the scan's gate: B = 0 and D = 1 make v = x = 1
    H, P = 64, 64
    z = x.to(dev).view(1, 1, H, P).requires_grad_()
    one, none = torch.ones(1, 1, H, P, device=dev), torch.zeros(1, 1, 1, 8, device=dev)
    per = lambda v: torch.full((H,), v, device=dev)  # noqa: E731
    y = ssm.selective_scan(one, torch.zeros(1, 1, H, device=dev), per(-1.0), none, none, D=per(1.0), z=z)
    _within("scan", y.reshape(-1), want, 4 * 2.0 ** -23 * want.abs() + tiny)
    (dz,) = torch.autograd.grad(y.sum(), [z])
    _within("scan dz", dz.reshape(-1).cpu()[at], slope[at], 8 * 2.0 ** -23 * parts[at] + tiny)
    step = ssm.selective_scan_step(one[:, 0], torch.zeros(1, H, device=dev), per(-1.0), none[:, 0], none[:, 0], torch.zeros(1, H, P, 8, device=dev), D=per(1.0),
                                   z=z[:, 0].detach())
    _within("scan step", step.reshape(-1), want, 4 * 2.0 ** -23 * want.abs() + tiny)


def test_gates_at_the_ends_of_the_type(dev):
    """Far from zero silu is x or nothing; NaN stays NaN, and nothing else becomes one."""
    from vit_amd import ssm
    w = torch.tensor([[0.0, 1.0]], device=dev)
    for dt in DTYPES.values():
        x = torch.tensor([-3e38, -1e30, -1000.0, -104.0, -89.0, -88.0, 0.0, 89.0, 1000.0, 1e30, 3e38, float("inf"), float("nan")], device=dev, dtype=dt)
        y = torch.cat([ssm.causal_conv(v.view(1, 1, 1), w, activation="silu").view(1) for v in x])
        assert float(y[:6].abs().max()) <= 1e-35 and float(y[6]) == 0.0 and torch.equal(y[7:12], x[7:12]) and bool(torch.isnan(y[12])), y


def test_fp32_decays_keep_their_low_bits(dev):
    """y_t = exp(L_t) of a state of one, L_t the sum of 64 exact log decays down to -45: v_exp_f32 one unit in the last place, the low
    part's correction a half, held to two (2^-22).  (Steps of 30 and more: softplus adds nothing, so the sums are known exactly.)
    A step's factor likewise; the end of five chunks is a product of five such factors and its four roundings."""
    from vit_amd import ssm
    T, H = 64 * 5, 16
    g = torch.Generator().manual_seed(80)
    dt = 30.0 + 4.0 * torch.rand(1, T, H, generator=g)
    A = -0.02 * (1 + 0.1 * torch.rand(H, generator=g))
    L = (dt.double() * A.double()).cumsum(1)
    zero, one = torch.zeros(1, T, H, 1, device=dev), torch.ones(1, T, 1, 1, device=dev)
    for t in (1, 33, 64):
        y, end = ssm.selective_scan(zero[:, :t], dt[:, :t].to(dev), A.to(dev), one[:, :t], one[:, :t], state=torch.ones(1, H, 1, 1, device=dev), return_state=True)
        want = torch.exp(L[:, :t])
        _within("y", y[..., 0], want, 2.0 ** -22 * want)
        _within("end", end[..., 0, 0], want[:, -1], 2.0 ** -22 * want[:, -1])
    # (the head with the slowest decay alone: five chunks stay inside the type)
    slow = A / 8
    L = (dt.double() * slow.double()).cumsum(1)
    _, end = ssm.selective_scan(zero, dt.to(dev), slow.to(dev), one, one, state=torch.ones(1, H, 1, 1, device=dev), return_state=True)
    want = torch.exp(L[:, -1])
    _within("end of five", end[..., 0, 0], want, (5 * 2.0 ** -22 + 4 * 2.0 ** -24) * want)
    # what token 0 of 64 leaves behind: d exp(L_63 - L_0) x B
    x = torch.zeros(1, 64, H, 1, device=dev)
    x[:, 0] = 1.0
    L = (dt[:, :64].double() * A.double()).cumsum(1)
    _, end = ssm.selective_scan(x, dt[:, :64].to(dev), A.to(dev), one[:, :64], one[:, :64], return_state=True)
    want = dt[:, 0].double() * torch.exp(L[:, 63] - L[:, 0])
    _within("left behind", end[..., 0, 0], want, 2.0 ** -22 * want)
    st = torch.ones(1, H, 1, 1, device=dev)
    ssm.selective_scan_step(zero[:, 0], 20 * dt[:, 0].to(dev), A.to(dev), one[:, 0], one[:, 0], st)
    want = torch.exp((20 * dt[:, 0]).double() * A.double())
    _within("step", st[..., 0, 0], want, 2.0 ** -22 * want)


def test_sizes_no_launch_can_take(dev):
    """More threads than a launch has: ValueError, a training call's before anything ran."""
    from vit_amd import ssm
    e = torch.ones(1, device=dev)
    big = torch.zeros(2 ** 26, 1, device=dev, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="sandwich_norm"):
        ssm.sandwich_norm(big, big, e, None, e, None)
    x, w = big[:2 ** 24].unsqueeze(1), torch.ones(1, 2, device=dev, requires_grad=True)
    with pytest.raises(ValueError, match="ssm_conv"):
        ssm.causal_conv(x, w)
    assert ssm.causal_conv(x, w.detach()).shape == x.shape
    pair = big[:2 ** 25].view(2 ** 24, 2, 1)
    with pytest.raises(ValueError, match="sandwich_norm"):
        ssm.sandwich_norm(pair, pair, e.clone().requires_grad_(), None, e, None, gate=big[:2 ** 24])
    one = torch.zeros(2 ** 23, 1, 1, 1, device=dev, dtype=torch.bfloat16)
    a = torch.full((1,), -1.0, device=dev, requires_grad=True)
    with pytest.raises(ValueError, match="backward"):
        ssm.selective_scan(one, one[..., 0], a, one, one)


def test_empty_batch(dev):
    """No samples: empty results, untouched states, gradients of zero; as the norms have it."""
    from vit_amd import ssm
    for T in (0, 5):
        s = to(scan_inputs(90, torch.bfloat16, 2, 5, 4, 8, 2, 16, state=True), dev)
        s = {k: v[:0, :T] if k in ("x", "dt", "Bm", "Cm", "z") else v[:0] if k == "state" else v for k, v in s.items()}
        lens = torch.zeros(0, dtype=torch.int32, device=dev)
        y, end = _call(ssm, s, lengths=lens, return_state=True)
        assert y.shape == (0, T, 4, 8) and end.shape == (0, 4, 8, 16)
        leaf = {k: v.detach().requires_grad_() for k, v in s.items()}
        y, end = _call(ssm, leaf, return_state=True)
        for k, g in zip(leaf, torch.autograd.grad([y, end], list(leaf.values()), [torch.zeros_like(y), torch.zeros_like(end)])):
            assert g.shape == leaf[k].shape and not bool(g.count_nonzero()), k
        x, w, st = torch.zeros(0, T, 8, device=dev), torch.ones(8, 4, device=dev), torch.zeros(0, 3, 8, device=dev)
        y, end = ssm.causal_conv(x, w, state=st, lengths=lens, return_state=True)
        assert y.shape == (0, T, 8) and end.shape == (0, 3, 8)
        w.requires_grad_()
        (dw,) = torch.autograd.grad(ssm.causal_conv(x, w, activation="silu").sum(), [w])
        assert not bool(dw.count_nonzero())
    y = ssm.selective_scan_step(s["x"].new_zeros(0, 4, 8), s["dt"].new_zeros(0, 4), s["A"], s["Bm"].new_zeros(0, 2, 16), s["Cm"].new_zeros(0, 2, 16), s["state"])
    assert y.shape == (0, 4, 8)
    assert ssm.causal_conv_step(torch.zeros(0, 8, device=dev), torch.ones(8, 4, device=dev), None, st).shape == (0, 8)
    e = torch.ones(8, device=dev)
    assert ssm.sandwich_norm(torch.zeros(0, 3, 8, device=dev), torch.zeros(0, 3, 8, device=dev), e, None, e, None)[1].shape == (0, 3, 8)


def test_what_stands_behind_a_samples_last_frame_does_not_count(dev):
    """A padded batch through the encoder: NaN behind the ends gives the features and gradients of any other padding, bit for bit
    (with the ordered reductions: the first norm's weight gradient is a sum of atomics without); a sample of no frames too."""
    from vit_amd import ops
    from vit_amd.sequence import TemporalEncoder
    torch.manual_seed(3)
    enc = TemporalEncoder(128, 64, 2, dropout=0.0, bidirectional=False, model_type="ssm").to(dev).train()
    lens = torch.tensor([9, 1, 4, 0], dtype=torch.int32, device=dev)
    x = torch.randn(4, 9, 128, device=dev)
    behind = torch.arange(9, device=dev)[None] >= lens[:, None]
    cot = torch.randn(4, 64, device=dev)

    def run(fill):
        xs = x.masked_fill(behind[..., None], fill).requires_grad_()
        got, _ = enc.ssm_features(xs, lens)
        return [got.detach()] + list(torch.autograd.grad(got, [p for _, p in enc.named_parameters()] + [xs], cot))

    was = ops.ordered_reductions_enabled(dev)
    ops.enable_ordered_reductions(dev)
    try:
        want = run(0.0)
        assert all(bool(torch.isfinite(v).all()) for v in want) and float(want[-1][behind].abs().max()) == 0.0
        for fill in (float("nan"), float("inf"), 3.0):
            for a, b in zip(run(fill), want):
                assert torch.equal(a, b), fill
    finally:
        ops.enable_ordered_reductions(dev, was)
    with torch.no_grad():
        assert float(enc.ssm_features(x, lens)[0][3].abs().max()) == 0.0      # no frame, no feature
    for bad in (lens.long(), lens[:3], lens.cpu()):
        with pytest.raises(ValueError, match="lengths"):
            enc.ssm_features(x, bad)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T", [1, 8, 63, 64])
@pytest.mark.parametrize("P,N", [(24, 16), (64, 64), (100, 100), (64, 128), (24, 128), (100, 64)])
def test_one_chunk_without_a_state(dev, P, N, T, dtype):
    """The backward pass of one chunk where no gradient of a state comes in or goes out: nothing is swept."""
    from vit_amd import ssm
    s = scan_inputs(T + P + N, DTYPES[dtype], 2, T, 4, P, 2, N)
    leaf = leaves64(s)
    wy, _ = ref.selective_scan(**leaf)
    names = [k for k in s if s[k] is not None]
    dy = randn(torch.Generator().manual_seed(T), *wy.shape, dtype=DTYPES[dtype])
    want = torch.autograd.grad(wy, [leaf[k] for k in names], dy.double())
    d = {k: v if v is None else v.requires_grad_() for k, v in to(s, dev).items()}
    y = _call(ssm, d)
    close("y", y, wy)
    for k, a, b in zip(names, torch.autograd.grad(y, [d[k] for k in names], dy.to(dev)), want):
        if T == 1 and k == "A":      # one token: nothing passes through a decay
            assert float(a.abs().max()) == 0.0
            continue
        close("d" + k, a, b)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("B,H", [(19, 9), (16, 16), (257, 1), (20, 15), (73, 7), (16, 32)])
def test_row_counts_around_the_segments(dev, B, H, dtype):
    """171 to 256 rows of eight chunks are cut in two, 257 and more are one walk: both sides of each step."""
    from vit_amd import ssm
    T, P, N = 513, 4, 4
    s = scan_inputs(B + H, DTYPES[dtype], B, T, H, P, 1, N, state=True)
    leaf = leaves64(s)
    wy, wend = ref.selective_scan(**leaf)
    names = [k for k in s if s[k] is not None]
    g = torch.Generator().manual_seed(B)
    dy, dend = randn(g, *wy.shape, dtype=DTYPES[dtype]), randn(g, *wend.shape)
    want = torch.autograd.grad([wy, wend], [leaf[k] for k in names], [dy.double(), dend.double()])
    d = {k: v.requires_grad_() for k, v in to(s, dev).items()}
    y, end = _call(ssm, d, return_state=True)
    close("y", y, wy)
    close("end", end, wend)
    for k, a, b in zip(names, torch.autograd.grad([y, end], [d[k] for k in names], [dy.to(dev), dend.to(dev)]), want):
        close("d" + k, a, b)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_gradients_through_one_output_only(dev, dtype):
    """A loss on the returned states alone, or on one of the norms' two results."""
    from vit_amd import ssm
    dt = DTYPES[dtype]
    for T in (5, 130):
        s = scan_inputs(100 + T, dt, 2, T, 4, 24, 2, 20, state=True)
        leaf = leaves64(s)
        _, wend = ref.selective_scan(**leaf)
        names = ("x", "dt", "A", "Bm", "dt_bias", "state")
        dend = randn(torch.Generator().manual_seed(T), *wend.shape)
        want = torch.autograd.grad(wend, [leaf[k] for k in names], dend.double())
        d = {k: v.requires_grad_() for k, v in to(s, dev).items()}
        _, end = _call(ssm, d, return_state=True)
        for k, a, b in zip(names, torch.autograd.grad(end, [d[k] for k in names], dend.to(dev)), want):
            close("d" + k, a, b)
        x, w, st = randn(torch.Generator().manual_seed(1), 2, T, 8, dtype=dt), randn(torch.Generator().manual_seed(2), 8, 4), randn(torch.Generator().manual_seed(3), 2, 3, 8, dtype=dt)
        x64, st64 = x.double().requires_grad_(), st.double().requires_grad_()
        _, wend = ref.causal_conv(x64, w.double(), silu=True, state=st64)
        gx, gs = x.to(dev).requires_grad_(), st.to(dev).requires_grad_()
        _, end = ssm.causal_conv(gx, w.to(dev), activation="silu", state=gs, return_state=True)
        cot = torch.ones_like(end)
        for a, b in zip(torch.autograd.grad(end, [gx, gs], cot), torch.autograd.grad(wend, [x64, st64], cot.double().cpu())):
            assert torch.equal(a.double().cpu(), b)      # inputs handed on
    g = torch.Generator().manual_seed(110)
    s = dict(residual=randn(g, 3, 7, 40, dtype=dt), y=randn(g, 3, 7, 40, dtype=dt), post_weight=randn(g, 40, shift=1.0), post_bias=randn(g, 40),
             pre_weight=randn(g, 40, shift=1.0), pre_bias=randn(g, 40), gate=randn(g, 3, 40))
    for which, names in ((0, ("residual", "y", "post_weight", "post_bias", "gate")), (1, tuple(s))):
        leaf = leaves64(s)
        out = ref.sandwich_norm(**leaf)[which]
        cot = randn(g, *out.shape, dtype=dt)
        want = torch.autograd.grad(out, [leaf[k] for k in names], cot.double())
        d = {k: v.to(dev).requires_grad_() for k, v in s.items()}
        got = torch.autograd.grad(ssm.sandwich_norm(**d)[which], [d[k] for k in names], cot.to(dev))
        for k, a, b in zip(names, got, want):
            close("d" + k, a, b)


def test_broadcast_inputs(dev):
    """One B, C, dt and state for all samples, one token for all times: expanded views, their gradients summed."""
    from vit_amd import ssm
    s = scan_inputs(120, torch.float32, 3, 70, 4, 16, 1, 16, state=True, slices=False)
    one = dict(s, Bm=s["Bm"][:1], Cm=s["Cm"][:, :1], dt=s["dt"][:1], state=s["state"][:1], z=s["z"][:1, :1])
    wide = lambda v: {k: t.expand(*s[k].shape) for k, t in v.items()}  # noqa: E731
    leaf = leaves64(one)
    wy, _ = ref.selective_scan(**wide(leaf))
    dy = randn(torch.Generator().manual_seed(4), *wy.shape)
    want = torch.autograd.grad(wy, list(leaf.values()), dy.double())
    d = {k: v.to(dev).requires_grad_() for k, v in one.items()}
    y = _call(ssm, wide(d))
    close("y", y, wy)
    for k, a, b in zip(d, torch.autograd.grad(y, list(d.values()), dy.to(dev)), want):
        close("d" + k, a, b)


def test_captured_calls_read_their_lengths_anew(dev):
    """Two captured graphs (a prompt cut into segments, a convolution with its norms) replayed in turn with other lengths and inputs."""
    from vit_amd import ssm
    s = to(scan_inputs(130, torch.bfloat16, 2, 600, 2, 32, 1, 32, state=True), dev)
    lens = torch.tensor([600, 17], dtype=torch.int32, device=dev)
    x, w, e = torch.randn(2, 600, 64, device=dev), torch.randn(64, 4, device=dev), torch.ones(64, device=dev)

    def scan():
        return _call(ssm, s, lengths=lens, return_state=True)

    def conv():
        u = ssm.causal_conv(x, w, activation="silu", lengths=lens)
        return ssm.sandwich_norm(x, u, e, None, e, None, gate=e)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        scan(), conv()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for f in (scan, conv):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = f()
        graphs.append((f, graph, out))
    for ends in ([600, 17], [0, 600], [513, 512], [1, 64]):
        lens.copy_(torch.tensor(ends, dtype=torch.int32))
        x.normal_()
        for _, graph, _ in graphs:
            graph.replay()
        for f, _, out in graphs:
            for a, b in zip(out, f()):
                assert torch.equal(a, b), ends
        torch.cuda.synchronize()
